// Logit processing before a sampler: penalties for repeated tokens, biases, a grammar bit mask and
// the greedy token of the result, in one pass over the logits.
#include <cmath>
#include <cstdio>

#include <cooperative_groups.h>

#include "../../include/mcpm.h"
#include "mcpm_cluster.h"
#include "mcpm_device.cuh"
#include "mcpm_paged.cuh"

namespace mcpm {
namespace {

constexpr int LG_CLUSTER_BITS = 3, LG_WIDE_BITS = 4;   // CTAs that share a row: 8, or 16 where few rows leave SMs idle
constexpr int LG_THREADS = 256;
constexpr int LG_CHUNK_BITS = 10, LG_CHUNK = 1 << LG_CHUNK_BITS;   // tokens that go to one CTA in a row, four a thread
constexpr int LG_CHUNKS = 32;        // most chunks whose words a CTA holds at once (places are 16 bits)
constexpr int LG_HELD = 4;           // chunks in registers at once
constexpr int LG_BATCH = 8;          // history entries of a thread in flight
constexpr int LG_QUEUE = 2 * LG_BATCH * LG_THREADS;   // history entries of a CTA in one round
constexpr int LG_LISTED = 1024;      // listed tokens of a slice
constexpr int LG_COUNT_BITS = 20;    // counter: times in the history; above: last bias entry + 1
constexpr int LG_MAX_HIST = (1 << LG_COUNT_BITS) - 1, LG_MAX_BIAS = (1 << (32 - LG_COUNT_BITS)) - 2;
static_assert(LG_CHUNK == 4 * LG_THREADS && LG_CHUNKS * LG_CHUNK <= 65536 && LG_CHUNKS % LG_HELD == 0, "");
// Chunks of a CTA's slice: all of them where they fit, since each slice passes over the history again (39 rows of
// 161648 with histories of 3180: two slices 26 us, one 19 us).
__host__ __device__ inline int slice_chunks(int n_vocab, int bits_cta) {
    const int mine = (((n_vocab - 1) >> LG_CHUNK_BITS) >> bits_cta) + 1;
    return mine < LG_CHUNKS ? mine : LG_CHUNKS;
}
static_assert(LG_LISTED >= LG_CHUNK, "one chunk's tokens fit the list");

struct Best {
    float v;
    int t;
};
// Larger value first, then the lower token; a token above every other stands for "none".
__device__ __forceinline__ void take(Best& a, const Best& b) {
    if (b.v > a.v || (b.v == a.v && b.t < a.t)) a = b;
}

// A cluster of 8 or 16 CTAs per row.  Chunks of the vocabulary go to them in turn: frequent tokens have low
// ids, and with contiguous shares the first CTA had half of a long history (64 rows with 4096 tokens each: 35 us).
// Per slice of a CTA's tokens: every thread passes over a share of the history and queues the entries that are
// this CTA's (an eighth: worked on in place they would keep every warp busy for a few lanes).  The queued tokens
// claim their 16-bit words, the first of each takes a place on a list, and then every entry counts at its
// token's place and every bias entry leaves its index there (integer atomics: the order does not matter; the
// largest index is the last entry).  The streaming pass puts the logits of listed tokens aside, and they are
// computed side by side after it.  A slice with more listed tokens than the list holds is cut in half until
// they fit.  VEC = 4 where all rows are 16-byte aligned, else 1.
// 64 rows of 130560 without lists 13.4 us, 5.0 TB/s (a device copy of them: 16 us); with 4096 tokens of history,
// 64 biases and a mask each 24.8 us, of which 10.7 us are bytes: the lists' round trips come before the logits'.
// One row 6.4 us.
template <int VEC, bool LISTS, bool MASK, int bits_cta>
__global__ void __launch_bounds__(LG_THREADS, 4) k_logits(const mcpm_logits_params p) {
    extern __shared__ __align__(16) uint16_t words[];    // [tokens of a slice] place on the list plus 1; zero: not listed
    __shared__ uint32_t counts[LISTS ? LG_LISTED : 1];   // the counters of the listed tokens
    __shared__ float aside[LISTS ? LG_LISTED : 1];       // their logits
    __shared__ uint16_t list[LISTS ? LG_LISTED : 1];     // their places in the slice
    __shared__ uint16_t queue[LISTS ? LG_QUEUE : 1];
    __shared__ int n_list, n_queue;
    __shared__ Best warp_best[LG_THREADS / 32], cta_best[1 << LG_WIDE_BITS];
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    if (p.argmax) cluster.barrier_arrive();   // waited for before the first write to another CTA's memory
    grid_dep_launch();
    grid_dep_wait();
    constexpr int n_cta = 1 << bits_cta;   // CTAs of the row's cluster
    const int tid = threadIdx.x, rank = cluster.block_rank(), row = blockIdx.x >> bits_cta;
    const int V = p.n_vocab;
    const float* x = p.logits + row * p.logits_stride;
    float* out = p.out + row * p.out_stride;
    const uint32_t* allow = MASK ? p.allow + row * p.allow_stride : nullptr;
    // chunk k of this CTA begins at token base_of(k); a thread's tokens of it are place(0 .. 3) further
    auto base_of = [&](int k) { return (k << bits_cta | rank) << LG_CHUNK_BITS; };
    auto place = [&](int e) { return VEC == 4 ? 4 * tid + e : e * LG_THREADS + tid; };
    const int mine = (((V + LG_CHUNK - 1) >> LG_CHUNK_BITS) - rank + n_cta - 1) >> bits_cta;   // chunks of this CTA
    Best best{-INFINITY, 0x7fffffff};
    float v[LG_HELD][4];
    uint32_t bits[LG_HELD][VEC == 4 ? 1 : 4];   // the mask words of the thread's tokens
    auto load = [&](int k0) {
#pragma unroll
        for (int k = 0; k < LG_HELD; ++k) {
            const int base = base_of(k0 + k);
            if (base + LG_CHUNK <= V) {
                if constexpr (VEC == 4) {
                    *reinterpret_cast<float4*>(v[k]) = *reinterpret_cast<const float4*>(x + base + 4 * tid);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[k][e] = x[base + place(e)];
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[k][e] = base + place(e) < V ? x[base + place(e)] : -INFINITY;
            }
        }
        if constexpr (MASK) {
#pragma unroll
            for (int k = 0; k < LG_HELD; ++k)
#pragma unroll
                for (int e = 0; e < (VEC == 4 ? 1 : 4); ++e) {
                    const int t = base_of(k0 + k) + place(e);
                    bits[k][e] = t < V ? allow[t >> 5] : 0u;
                }
        }
    };
    const int* hist = LISTS && p.hist ? p.hist + row * p.hist_stride : nullptr;
    const int* bias_token = LISTS && p.bias_token ? p.bias_token + row * p.bias_stride : nullptr;
    int n_hist = hist ? p.hist_max : 0, n_bias = bias_token ? p.bias_max : 0;
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    int first_bias = -1;
    if constexpr (LISTS) {
        if (tid < n_bias) first_bias = bias_token[tid];
        if (hist && p.hist_len) n_hist = min(max(p.hist_len[row], 0), p.hist_max);
        if (bias_token && p.bias_len) n_bias = min(max(p.bias_len[row], 0), p.bias_max);
        if (hist) rep = p.penalties[3 * row], freq = p.penalties[3 * row + 1], pres = p.penalties[3 * row + 2];
    }
    auto listed = [&](float y, uint32_t w) {
        const uint32_t c = w & LG_MAX_HIST, b = w >> LG_COUNT_BITS;
        if (c) {
            y = y > 0.0f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
            y = __fsub_rn(y, __fadd_rn(__fmul_rn(freq, static_cast<float>(c)), pres));
        }
        return b ? __fadd_rn(y, p.bias[row * p.bias_stride + b - 1]) : y;
    };
    for (int c0 = 0, c1; c0 < mine; c0 = c1) {
        c1 = min(mine, c0 + slice_chunks(V, bits_cta));
        if constexpr (LISTS) {
            const int lane = tid & 31;
            // the word of a token, if it is in this slice
            auto word_of = [&](int token) -> unsigned {
                const unsigned chunk = static_cast<unsigned>(token) >> LG_CHUNK_BITS, k = (chunk >> bits_cta) - c0;
                const bool here = (chunk & (n_cta - 1)) == static_cast<unsigned>(rank) && k < static_cast<unsigned>(c1 - c0) && token < V;   // a negative token's chunk lies beyond
                return here ? k << LG_CHUNK_BITS | (token & (LG_CHUNK - 1)) : ~0u;
            };
            auto claim = [&](unsigned w) {
                if (words[w] || atomicCAS(&words[w], static_cast<unsigned short>(0), static_cast<unsigned short>(0xffff))) return;
                const int at = atomicAdd(&n_list, 1);
                if (at < LG_LISTED) {
                    list[at] = static_cast<uint16_t>(w);
                    counts[at] = 0u;
                    words[w] = static_cast<uint16_t>(at + 1);   // read after a barrier
                }
            };
            for (bool again = true; again;) {
                if (tid == 0) n_list = n_queue = 0;
                for (int i = tid; i < (c1 - c0) * LG_CHUNK / 8; i += LG_THREADS) reinterpret_cast<uint4*>(words)[i] = make_uint4(0u, 0u, 0u, 0u);
                __syncthreads();
                auto each_bias = [&](auto f) {
                    for (int i = tid; i < n_bias; i += LG_THREADS) {
                        const unsigned w = word_of(i < LG_THREADS ? first_bias : bias_token[i]);
                        if (w != ~0u) f(i, w);
                    }
                };
                each_bias([&](int, unsigned w) { claim(w); });
                again = false;
                for (int r0 = 0; r0 == 0 || (r0 < n_hist && !again); r0 += LG_QUEUE) {   // rounds
                    for (int b0 = r0; b0 < min(n_hist, r0 + LG_QUEUE); b0 += LG_BATCH * LG_THREADS) {
                        unsigned w[LG_BATCH];
                        int before[LG_BATCH], sum = 0;
#pragma unroll
                        for (int k = 0; k < LG_BATCH; ++k) {
                            const int i = b0 + k * LG_THREADS + tid;
                            w[k] = static_cast<unsigned>(i < n_hist ? hist[i] : -1);
                        }
#pragma unroll
                        for (int k = 0; k < LG_BATCH; ++k) {
                            w[k] = word_of(static_cast<int>(w[k]));
                            const unsigned m = __ballot_sync(0xffffffffu, w[k] != ~0u);
                            before[k] = sum + __popc(m & ((1u << lane) - 1u));
                            sum += __popc(m);
                        }
                        int at = 0;
                        if (lane == 0 && sum) at = atomicAdd(&n_queue, sum);
                        at = __shfl_sync(0xffffffffu, at, 0);
#pragma unroll
                        for (int k = 0; k < LG_BATCH; ++k)
                            if (w[k] != ~0u) queue[at + before[k]] = static_cast<uint16_t>(w[k]);
                    }
                    // The logits come to L2 while the entries are counted; asked for earlier, they held the history
                    // up for 5 us.
                    if (VEC == 4 && r0 == 0 && tid < c1 - c0 && base_of(c0 + tid) + LG_CHUNK <= V)
                        bulk_prefetch_l2(x + base_of(c0 + tid), LG_CHUNK * 4);
                    __syncthreads();
                    const int n = n_queue;
                    for (int i = tid; i < n; i += LG_THREADS) claim(queue[i]);
                    __syncthreads();
                    again = n_list > LG_LISTED;
                    if (!again) {
                        for (int i = tid; i < n; i += LG_THREADS) atomicAdd(&counts[words[queue[i]] - 1], 1u);
                        if (r0 == 0)
                            each_bias([&](int i, unsigned w) {   // the largest index, beside a count that others add to
                                uint32_t* c = &counts[words[w] - 1];
                                const uint32_t mark = static_cast<uint32_t>(i + 1);
                                for (uint32_t old = *c; (old >> LG_COUNT_BITS) < mark;) {   // each failure is another's success
                                    const uint32_t seen = atomicCAS(c, old, mark << LG_COUNT_BITS | (old & LG_MAX_HIST));
                                    if (seen == old) break;
                                    old = seen;
                                }
                            });
                    }
                    if (tid == 0) n_queue = 0;
                    __syncthreads();
                }
                if (again) c1 = c0 + (c1 - c0 + 1) / 2;   // ends: a chunk's tokens fit the list
            }
        }
        for (int k0 = c0; k0 < c1; k0 += LG_HELD) {
            load(k0);
#pragma unroll
            for (int k = 0; k < LG_HELD; ++k) {
                if (k0 + k >= c1) break;
                float* y = v[k];
                const int base = base_of(k0 + k);
                if constexpr (MASK) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!(bits[k][VEC == 4 ? 0 : e] >> (place(e) & 31) & 1u)) y[e] = -INFINITY;   // base is a multiple of 32
                }
                if constexpr (LISTS) {
                    const uint16_t* w = words + ((k0 + k - c0) << LG_CHUNK_BITS);
                    uint16_t z[4];
                    if constexpr (VEC == 4) {
                        *reinterpret_cast<uint2*>(z) = reinterpret_cast<const uint2*>(w)[tid];
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) z[e] = w[place(e)];
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (z[e]) aside[z[e] - 1] = y[e];
                        y[e] = z[e] ? -INFINITY : y[e];   // not a candidate yet; its place in out is written again below
                    }
                }
                const float top = fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]));   // NaN never
                if (top > best.v) {   // seldom; a thread's tokens ascend
#pragma unroll
                    for (int e = 3; e >= 0; --e)
                        if (y[e] == top) best = Best{top, base + place(e)};
                }
                if (base + LG_CHUNK <= V) {
                    if constexpr (VEC == 4) {
                        *reinterpret_cast<float4*>(out + base + 4 * tid) = *reinterpret_cast<const float4*>(y);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) out[base + place(e)] = y[e];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (base + place(e) < V) out[base + place(e)] = y[e];
                }
            }
        }
        if constexpr (LISTS) {
            __syncthreads();
            for (int k = tid; k < n_list; k += LG_THREADS) {
                const int i = list[k], t = base_of(c0 + (i >> LG_CHUNK_BITS)) + (i & (LG_CHUNK - 1));
                float y = listed(aside[k], counts[k]);   // the mask's -inf stays -inf, unless it meets an infinite penalty or bias
                if (MASK && y != y && !(allow[t >> 5] >> (t & 31) & 1u)) y = -INFINITY;
                out[t] = y;
                if (y > best.v || (y == best.v && t < best.t && y > -INFINITY)) best = Best{y, t};
            }
            __syncthreads();   // the words are free
        }
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
    cluster.barrier_arrive();
    if (rank) return;         // only the first CTA waits for the others
    cluster.barrier_wait();
    if (tid == 0) {
        for (int c = 1; c < n_cta; ++c) take(best, cta_best[c]);
        p.argmax[row] = best.t == 0x7fffffff ? -1 : best.t;
    }
}

using Kernel = void (*)(mcpm_logits_params);

constexpr size_t LG_SMEM = LG_CHUNKS * LG_CHUNK * sizeof(uint16_t);

// The kernel of a variant, its attributes set once per device (setting them again does no harm); null: the device
// cannot run its cluster.
template <int VEC, int BITS, bool LISTS, bool MASK>
cudaError_t prepared(int dev, Kernel& kernel) {
    static signed char done[64] = {};   // 1: runs, -1: does not
    kernel = k_logits<VEC, LISTS, MASK, BITS>;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!done[dev]) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(LG_SMEM));
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
        const auto active = [&](int width) { return active_clusters(kernel, width, LG_THREADS, LG_SMEM); };
        done[dev] = widest_cluster(1 << BITS, active) == 1 << BITS ? 1 : -1;
    }
    if (done[dev] < 0) kernel = nullptr;
    return cudaSuccess;
}
template <int VEC, int BITS>
cudaError_t pick(bool lists, bool mask, int dev, Kernel& kernel) {
    return lists ? mask ? prepared<VEC, BITS, true, true>(dev, kernel) : prepared<VEC, BITS, true, false>(dev, kernel)
           : mask ? prepared<VEC, BITS, false, true>(dev, kernel) : prepared<VEC, BITS, false, false>(dev, kernel);
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
    auto aligned = [&](const float* q, int64_t stride) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0 && (p.n_seq == 1 || stride % 4 == 0); };
    const bool lists = p.hist || p.bias_token, mask = p.allow != nullptr;
    const bool vec = aligned(p.logits, p.logits_stride) && aligned(p.out, p.out_stride);
    int dev = 0, n_sm = 0;
    Kernel kernel = nullptr;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = sm_count(dev, n_sm);
    int bits_cta = LG_WIDE_BITS;
    if (e == cudaSuccess && static_cast<long long>(p.n_seq) << LG_WIDE_BITS <= cluster_ctas(n_sm))
        e = vec ? pick<4, LG_WIDE_BITS>(lists, mask, dev, kernel) : pick<1, LG_WIDE_BITS>(lists, mask, dev, kernel);
    if (e == cudaSuccess && !kernel) {
        bits_cta = LG_CLUSTER_BITS;
        e = vec ? pick<4, LG_CLUSTER_BITS>(lists, mask, dev, kernel) : pick<1, LG_CLUSTER_BITS>(lists, mask, dev, kernel);
    }
    const size_t smem = lists ? slice_chunks(p.n_vocab, bits_cta) * LG_CHUNK * sizeof(uint16_t) : 0;
    if (e == cudaSuccess) {
        const unsigned cluster = 1u << bits_cta;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(static_cast<unsigned>(p.n_seq) * cluster);
        cfg.blockDim = dim3(LG_THREADS);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = static_cast<cudaStream_t>(stream);
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = cluster;
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
