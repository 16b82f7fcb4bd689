// Logit processing before a sampler: penalties for repeated tokens, biases, a grammar bit mask and
// the greedy token of the result, in one pass over the logits.
#include <cmath>
#include <cstdio>

#include <cooperative_groups.h>

#include "../../include/mcpm.h"
#include "mcpm_device.cuh"

namespace mcpm {
namespace {

constexpr int LG_CLUSTER = 8;        // CTAs that share a row
constexpr int LG_THREADS = 512;
constexpr int LG_HELD = 8;           // logits a thread holds at once: 40 registers, three CTAs per SM
constexpr int LG_STEP = LG_THREADS * LG_HELD;
constexpr int LG_SLICE = 4 * LG_STEP;   // tokens whose counters a CTA holds at once (one word each)
constexpr int LG_BATCH = 4;          // list entries of a thread in flight
constexpr int LG_COUNT_BITS = 20;    // counter word: times in the history; above: last bias entry + 1
constexpr int LG_MAX_HIST = (1 << LG_COUNT_BITS) - 1, LG_MAX_BIAS = (1 << (32 - LG_COUNT_BITS)) - 2;

struct Best {
    float v;
    int t;
};
// Larger value first, then the lower token; a token above every other stands for "none".
__device__ __forceinline__ void take(Best& a, const Best& b) {
    if (b.v > a.v || (b.v == a.v && b.t < a.t)) a = b;
}

// A cluster of LG_CLUSTER CTAs per row, each with a contiguous share of the vocabulary, LG_SLICE tokens at a
// time.  The slice's logits are on their way to L2 while the history is counted into shared-memory words
// (integer atomics: the order does not matter) and each bias entry leaves its index there (the largest, hence
// the last entry, stays); then the logits stream past the words.  VEC = 4 where all rows are 16-byte aligned,
// else 1.
template <int VEC>
__global__ void __launch_bounds__(LG_THREADS, 3) k_logits(const mcpm_logits_params p) {
    extern __shared__ __align__(16) uint32_t words[];   // [LG_SLICE]
    __shared__ Best warp_best[LG_THREADS / 32], cta_best[LG_CLUSTER];
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    if (p.argmax) cluster.barrier_arrive();   // waited for before the first write to another CTA's memory
    grid_dep_launch();
    grid_dep_wait();
    const int tid = threadIdx.x, rank = cluster.block_rank(), row = blockIdx.x / LG_CLUSTER;
    const int share = ((p.n_vocab + LG_CLUSTER - 1) / LG_CLUSTER + 31) & ~31;   // whole mask words
    const int lo = min(p.n_vocab, rank * share), hi = min(p.n_vocab, lo + share);
    const float* x = p.logits + row * p.logits_stride;
    float* out = p.out + row * p.out_stride;
    const int* hist = p.hist ? p.hist + row * p.hist_stride : nullptr;
    const int n_hist = hist ? (p.hist_len ? min(max(p.hist_len[row], 0), p.hist_max) : p.hist_max) : 0;
    const int* bias_token = p.bias_token ? p.bias_token + row * p.bias_stride : nullptr;
    const int n_bias = bias_token ? (p.bias_len ? min(max(p.bias_len[row], 0), p.bias_max) : p.bias_max) : 0;
    const uint32_t* allow = p.allow ? p.allow + row * p.allow_stride : nullptr;
    const bool lists = n_hist || n_bias;
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    if (n_hist) rep = p.penalties[3 * row], freq = p.penalties[3 * row + 1], pres = p.penalties[3 * row + 2];
    Best best{-INFINITY, 0x7fffffff};
    auto listed = [&](float y, uint32_t w) {
        const uint32_t c = w & LG_MAX_HIST, b = w >> LG_COUNT_BITS;
        if (c) {
            y = y > 0.0f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
            y = __fsub_rn(y, __fadd_rn(__fmul_rn(freq, static_cast<float>(c)), pres));
        }
        if (b) y = __fadd_rn(y, p.bias[row * p.bias_stride + b - 1]);
        return y;
    };
    for (int s0 = lo; s0 < hi; s0 += LG_SLICE) {
        const int n = min(LG_SLICE, hi - s0);
        if (VEC == 4 && tid == 0 && n >= 4) bulk_prefetch_l2(x + s0, (n & ~3) * 4);   // on its way while the lists are counted
        float v[LG_HELD];
        uint32_t bits[LG_HELD / VEC];   // VEC divides 32: a load's tokens share a mask word
        auto load = [&](int c) {
#pragma unroll
            for (int k = 0; k < LG_HELD / VEC; ++k) {
                const int i = c + VEC * (k * LG_THREADS + tid);
                if (VEC == 4 && i + 3 < n)
                    *reinterpret_cast<float4*>(v + VEC * k) = *reinterpret_cast<const float4*>(x + s0 + i);
                else
                    for (int e = 0; e < VEC; ++e) v[VEC * k + e] = i + e < n ? x[s0 + i + e] : 0.0f;
            }
#pragma unroll
            for (int k = 0; k < LG_HELD / VEC; ++k) {
                const int i = c + VEC * (k * LG_THREADS + tid);
                bits[k] = allow && i < n ? allow[(s0 + i) >> 5] >> ((s0 + i) & 31) : 0xffffffffu;
            }
        };
        load(0);
        if (lists) {
            for (int i = tid; i < (n + 3) / 4; i += LG_THREADS) reinterpret_cast<uint4*>(words)[i] = make_uint4(0u, 0u, 0u, 0u);
            __syncthreads();
            for (int i = tid; i < n_bias; i += LG_THREADS) {
                const unsigned t = static_cast<unsigned>(bias_token[i]) - static_cast<unsigned>(s0);
                if (t < static_cast<unsigned>(n)) atomicMax(&words[t], static_cast<uint32_t>(i + 1) << LG_COUNT_BITS);
            }
            if (n_bias) __syncthreads();   // the maximum is taken of whole words: no counts in them yet
            for (int i0 = tid; i0 < n_hist; i0 += LG_BATCH * LG_THREADS) {
                unsigned t[LG_BATCH];
#pragma unroll
                for (int k = 0; k < LG_BATCH; ++k)
                    t[k] = i0 + k * LG_THREADS < n_hist ? static_cast<unsigned>(hist[i0 + k * LG_THREADS]) - static_cast<unsigned>(s0) : ~0u;
#pragma unroll
                for (int k = 0; k < LG_BATCH; ++k)
                    if (t[k] < static_cast<unsigned>(n)) atomicAdd(&words[t[k]], 1u);
            }
            __syncthreads();
        }
        for (int c = 0; c < n; c += LG_STEP) {
            if (c) load(c);
#pragma unroll
            for (int k = 0; k < LG_HELD / VEC; ++k) {
                const int i = c + VEC * (k * LG_THREADS + tid);
                if (i >= n) break;
                float* y = v + VEC * k;
                if (lists) {
                    uint32_t w[VEC], any = 0u;
                    if constexpr (VEC == 4)
                        *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(words + i);
                    else
                        w[0] = words[i];
#pragma unroll
                    for (int e = 0; e < VEC; ++e) any |= w[e];
                    if (any)
#pragma unroll
                        for (int e = 0; e < VEC; ++e)
                            if (w[e]) y[e] = listed(y[e], w[e]);
                }
                float top = -INFINITY;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    if (!(bits[k] >> e & 1u)) y[e] = -INFINITY;
                    if (i + e < n) top = fmaxf(top, y[e]);   // NaN never
                }
                if (top > best.v) {   // seldom; tokens ascend here
#pragma unroll
                    for (int e = VEC - 1; e >= 0; --e)
                        if (i + e < n && y[e] == top) best = Best{top, s0 + i + e};
                }
                if (VEC == 4 && i + 3 < n)
                    *reinterpret_cast<float4*>(out + s0 + i) = *reinterpret_cast<const float4*>(v + VEC * k);
                else
                    for (int e = 0; e < VEC; ++e)
                        if (i + e < n) out[s0 + i + e] = v[VEC * k + e];
            }
        }
        __syncthreads();   // the words are free
    }
    if (!p.argmax) return;   // the whole grid
    for (int o = 16; o >= 1; o >>= 1)
        take(best, Best{__shfl_xor_sync(0xffffffffu, best.v, o), __shfl_xor_sync(0xffffffffu, best.t, o)});
    if ((tid & 31) == 0) warp_best[tid >> 5] = best;
    __syncthreads();
    if (tid == 0)
        for (int w = 1; w < LG_THREADS / 32; ++w) take(best, warp_best[w]);
    cluster.barrier_wait();   // every CTA of the row has started
    if (tid == 0) *cluster.map_shared_rank(&cta_best[rank], 0) = best;
    cluster.sync();
    if (rank == 0 && tid == 0) {
        for (int c = 1; c < LG_CLUSTER; ++c) take(best, cta_best[c]);
        p.argmax[row] = best.t == 0x7fffffff ? -1 : best.t;
    }
}

}  // namespace
}  // namespace mcpm

using namespace mcpm;

extern "C" mcpm_status mcpm_logits_process(const mcpm_logits_params* params, void* stream) {
    if (!params) return MCPM_BAD_ARG;
    mcpm_logits_params p = *params;
    if (p.logits_stride == 0) p.logits_stride = p.n_vocab;
    if (p.out_stride == 0) p.out_stride = p.n_vocab;
    if (p.hist_stride == 0) p.hist_stride = p.hist_max;
    if (p.bias_stride == 0) p.bias_stride = p.bias_max;
    const int mask_words = p.n_vocab > 0 ? (p.n_vocab - 1) / 32 + 1 : 0;
    if (p.allow_stride == 0) p.allow_stride = mask_words;
    if (p.n_seq <= 0 || p.n_vocab <= 0 || p.n_seq > (1 << 20) || p.n_vocab > (1 << 30) || !p.logits || !p.out ||
        p.logits_stride < p.n_vocab || p.out_stride < p.n_vocab ||
        (p.out == p.logits && p.out_stride != p.logits_stride))
        return MCPM_BAD_ARG;
    if (p.hist && (!p.penalties || p.hist_max < 0 || p.hist_max > LG_MAX_HIST || p.hist_stride < p.hist_max)) return MCPM_BAD_ARG;
    if (p.bias_token && (!p.bias || p.bias_max < 0 || p.bias_max > LG_MAX_BIAS || p.bias_stride < p.bias_max)) return MCPM_BAD_ARG;
    if (p.allow && p.allow_stride < mask_words) return MCPM_BAD_ARG;
    auto aligned = [](const float* q, int64_t stride) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0 && stride % 4 == 0; };
    void (*kernel)(mcpm_logits_params) =
        aligned(p.logits, p.logits_stride) && aligned(p.out, p.out_stride) ? k_logits<4> : k_logits<1>;
    const size_t smem = p.hist || p.bias_token ? LG_SLICE * 4 : 0;
    cudaError_t e = smem ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, LG_SLICE * 4) : cudaSuccess;
    if (e == cudaSuccess) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(static_cast<unsigned>(p.n_seq) * LG_CLUSTER);
        cfg.blockDim = dim3(LG_THREADS);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = static_cast<cudaStream_t>(stream);
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = LG_CLUSTER;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // every CTA waits before it reads
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 2;
        e = cudaLaunchKernelEx(&cfg, kernel, p);
    }
    if (e == cudaSuccess) return MCPM_OK;
    std::fprintf(stderr, "[mcpm] mcpm_logits_process: CUDA error: %s\n", cudaGetErrorString(e));
    return MCPM_CUDA_ERROR;
}
