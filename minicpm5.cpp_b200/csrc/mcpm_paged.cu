// Paged KV cache: append of new tokens (RoPE, rounding, page writes) and eviction of the positions with
// the least attention mass; the attention between them is in mcpm_paged_attention.cu.
#include <algorithm>
#include <cmath>
#include <cstdio>

#include <cooperative_groups.h>

#include "../../include/mcpm.h"
#include "mcpm_cluster.h"
#include "mcpm_device.cuh"
#include "mcpm_paged.cuh"

namespace mcpm {
namespace {

// ---------------------------------------------------------------- append
struct AppendArgs {
    mcpm_paged_tokens t;
    const int* table;
    void *kc, *vc;
    float* mass;
    int n_seq;
};

// A CTA per token; a token's rows are its query heads, its KV heads' K, then their V.  D / 4 lanes to a row, a
// float4 (two rotary pairs, the same ones in every row) a lane, AP_HELD rows of a lane in flight.
// (x0, x1) -> (c x0 - s x1, s x0 + c x1), one fma per output as mcpm_rope_kv_append.
// Bound by the memory: 8192 tokens of 16 + 2 + 2 heads x 128 (fp32 cache) 30.5 us, 5.6 TB/s; 64 tokens 5.3 us, the
// time of a call.
constexpr int AP_WARPS = 4, AP_HELD = 5;
template <typename T, int D>
__global__ void __launch_bounds__(32 * AP_WARPS) k_paged_append(const PagedGeom g, const AppendArgs a) {
    constexpr int LANES = D / 4, AT_ONCE = AP_WARPS * 32 / LANES;   // lanes of a row, rows of the CTA
    grid_dep_launch();
    grid_dep_wait();
    const size_t i = blockIdx.x;
    const int x = threadIdx.x % LANES, first = threadIdx.x / LANES, nq = a.t.q ? g.n_head : 0, nk = g.n_head_kv, rows = nq + 2 * nk;
    const int tok_slot = a.t.tok_slot[i], seq = a.t.tok_seq ? a.t.tok_seq[i] : static_cast<int>(i);
    // Slots of the token's sequence, 0: padding.  The stores alone look at it, so the loads do not wait for it.
    const unsigned slots = tok_slot >= 0 && seq >= 0 && seq < a.n_seq ? static_cast<unsigned>(g.max_pages * g.page_size) : 0u;
    const int pos = a.t.tok_pos ? a.t.tok_pos[i] : tok_slot;
    const float4 cs = a.t.rope ? reinterpret_cast<const float4*>(a.t.rope)[static_cast<size_t>(min(max(pos, 0), a.t.rope_len - 1)) * LANES + x]
                               : make_float4(1.0f, 0.0f, 1.0f, 0.0f);
    int page = -1, slot = 0;
    const bool held = static_cast<unsigned>(tok_slot) < slots && g.locate(a.table + static_cast<size_t>(seq) * g.max_pages, tok_slot, page, slot);
    for (int r0 = first; r0 < rows; r0 += AT_ONCE * AP_HELD) {
        float4 v[AP_HELD];
#pragma unroll
        for (int k = 0; k < AP_HELD; ++k) {
            const int r = r0 + k * AT_ONCE;
            if (r >= rows) break;
            const float* src = r < nq ? a.t.q + i * a.t.q_stride + r * D
                                      : (r < nq + nk ? a.t.k : a.t.v) + i * a.t.kv_stride + (r < nq + nk ? r - nq : r - nq - nk) * D;
            v[k] = reinterpret_cast<const float4*>(src)[x];
        }
#pragma unroll
        for (int k = 0; k < AP_HELD; ++k) {
            const int r = r0 + k * AT_ONCE;
            if (r >= rows) break;
            float4 y = v[k];
            if (a.t.rope && r < nq + nk)
                y = make_float4(__fmaf_rn(cs.x, y.x, -__fmul_rn(cs.y, y.y)), __fmaf_rn(cs.y, y.x, __fmul_rn(cs.x, y.y)),
                                __fmaf_rn(cs.z, y.z, -__fmul_rn(cs.w, y.w)), __fmaf_rn(cs.w, y.z, __fmul_rn(cs.z, y.w)));
            if (r < nq) {
                if (slots) reinterpret_cast<float4*>(a.t.q_out + (i * g.n_head + r) * D)[x] = y;
            } else if (held) {
                const bool is_v = r >= nq + nk;
                const int head = r - nq - (is_v ? nk : 0);
                kv_store4(static_cast<T*>(is_v ? a.vc : a.kc) + g.row(page, slot, head) + 4 * x, y);
                if (!is_v && x == 0 && a.mass) a.mass[g.mass_at(page, slot, head)] = 0.0f;
            }
        }
    }
}

template <typename T>
cudaError_t launch_append(const PagedGeom& g, const AppendArgs& a, cudaStream_t s) {
    return launch_dependent(g.head_dim == 64 ? k_paged_append<T, 64> : k_paged_append<T, 128>, dim3(a.t.n_tok), 32 * AP_WARPS, 0, s, g, a);
}

// ---------------------------------------------------------------- eviction
struct EvictArgs {
    void *kc, *vc;
    float* mass;
    const int *table, *len, *dst;
    int *new_len, *kept;
    int n_keep, n_sink, n_recent;
};

constexpr int EV_MAX_CLUSTER = 16;   // beyond the portable 8, where the device can run it
constexpr int EV_BITS = 11, EV_BINS = 1 << EV_BITS, EV_PASSES = 3;   // digits of 11, 11 and 10 bits, highest first
constexpr int EV_KEYS = 32768;   // keys a CTA holds in shared memory
constexpr int EV_RANKED = 512;   // at most a CTA's threads
constexpr int EV_HELD = 4;       // positions a thread reads at once
constexpr int EV_SMEM = (EV_PASSES * EV_BINS + EV_KEYS) * 4;

// Order-preserving unsigned key of a position: a larger key is kept first.  Absent positions 0, NaN 1
// (lightest), then the floats in order (-0 and +0 alike), then the protected positions.
__device__ __forceinline__ uint32_t mass_key(float m) {
    if (m != m) return 1u;
    const uint32_t u = __float_as_uint(m + 0.0f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;   // -inf is 0x007fffff
}

// A cluster per (KV head, sequence), each CTA with a contiguous share of the positions.  Radix selection of
// the n_keep-th largest key: per digit a histogram in each CTA, summed over the cluster, and the bin in
// which the count from above reaches n_keep.  Then every warp counts its positions above and at the
// threshold, and writes its part of the list in order.  Keys stay in shared memory between the passes.
// 4 bytes a position are nothing to the memory; what counts is the number of dependent steps: 2112 positions in
// one CTA 7 us, 65537 in a cluster of sixteen 15 us (one CTA: 290 us with the copy).
template <int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) k_paged_evict_select(const PagedGeom g, const EvictArgs a) {
    constexpr int WARPS = THREADS / 32;
    extern __shared__ __align__(16) uint32_t ev_smem[];
    __shared__ int groups[EV_PASSES][EV_BINS / 32], warp_gt[32], warp_eq[32], pick[3], n_cand;
    __shared__ int2 cta_sum;
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    grid_dep_wait();
    grid_dep_launch();   // after the wait: see k_paged_evict_copy
    uint32_t* hist = ev_smem;   // [EV_PASSES][EV_BINS]
    uint32_t* keys = ev_smem + EV_PASSES * EV_BINS;
    const int n_cta = cluster.num_blocks(), rank = cluster.block_rank();
    const int kv = blockIdx.x / n_cta, seq = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n = g.clamp_len(a.len[seq]);
    const int share = ((n + n_cta - 1) / n_cta + 31) & ~31;
    const int lo = min(n, rank * share), m = min(n, lo + share) - lo;   // this CTA's positions lo .. lo + m - 1
    const int* row = a.table + static_cast<size_t>(seq) * g.max_pages;
    int* kept = a.kept + (static_cast<size_t>(seq) * g.n_head_kv + kv) * a.n_keep;
    auto read_key = [&](int i) -> uint32_t {
        const int j = lo + i;
        int page, slot;
        if (!g.locate(row, j, page, slot)) return 0u;
        if (j < a.n_sink || j >= n - a.n_recent) return 0xffffffffu;
        return mass_key(a.mass[g.mass_at(page, slot, kv)]);
    };
    auto key = [&](int i) { return i < EV_KEYS ? keys[i] : read_key(i); };
    for (int i = tid; i < EV_PASSES * EV_BINS; i += THREADS) hist[i] = 0u;
    __syncthreads();
    // One count, or one for the whole warp where its keys share a bin (protected positions; equal masses).
    auto count = [&](uint32_t* h, int bin) {   // whole warps; bin -1: none
        const unsigned some = __ballot_sync(0xffffffffu, bin >= 0);
        int same = 0;
        if (some == 0xffffffffu) __match_all_sync(0xffffffffu, bin, &same);
        if (same) {
            if (lane == 0) atomicAdd(&h[bin], 32u);
        } else if (bin >= 0) {
            atomicAdd(&h[bin], 1u);
        }
    };
    for (int i0 = 32 * warp; i0 < m; i0 += EV_HELD * THREADS) {   // EV_HELD positions of a thread in flight
        const int batch = min(EV_HELD, (m - i0 + THREADS - 1) / THREADS);   // of the warp
        int page[EV_HELD], slot[EV_HELD];
        float x[EV_HELD];
        bool present[EV_HELD];
#pragma unroll
        for (int k = 0; k < EV_HELD; ++k)
            if (k < batch) {
                const int i = i0 + lane + k * THREADS;
                present[k] = i < m && g.locate(row, lo + i, page[k], slot[k]);
            }
#pragma unroll
        for (int k = 0; k < EV_HELD; ++k)
            if (k < batch) x[k] = present[k] ? a.mass[g.mass_at(page[k], slot[k], kv)] : 0.0f;
#pragma unroll
        for (int k = 0; k < EV_HELD; ++k)
            if (k < batch) {
                const int i = i0 + lane + k * THREADS, j = lo + i;
                const uint32_t y = !present[k] ? 0u : j < a.n_sink || j >= n - a.n_recent ? 0xffffffffu : mass_key(x[k]);
                if (i < m && i < EV_KEYS) keys[i] = y;
                count(hist, present[k] ? static_cast<int>(y >> (32 - EV_BITS)) : -1);
            }
    }
    __syncthreads();
    // Threshold key and how many positions with exactly that key are kept.  Fewer present positions than
    // n_keep: the scans end in bin 0 with room to spare, the threshold is 0, which absent positions alone have.
    uint32_t prefix = 0u;
    int need = a.n_keep;
    for (int pass = 0; pass < EV_PASSES; ++pass) {
        const int low = pass == 0 ? 32 - EV_BITS : pass == 1 ? 32 - 2 * EV_BITS : 0;   // lowest bit of the digit
        uint32_t* mine = hist + pass * EV_BINS;
        if (pass > 0) {
            const int above = low + (pass == 1 ? EV_BITS : 32 - 2 * EV_BITS);
            for (int i0 = 32 * warp; i0 < m; i0 += THREADS) {
                const uint32_t k = i0 + lane < m ? key(i0 + lane) : 0u;
                count(mine, k && (k >> above) == (prefix >> above) ? static_cast<int>(k >> low & ((1u << (above - low)) - 1u)) : -1);
            }
        }
        __syncthreads();
        for (int q = warp; q < EV_BINS / 32; q += WARPS) {
            const int s = __reduce_add_sync(0xffffffffu, mine[32 * q + lane]);
            if (lane == 0) groups[pass][q] = s;
        }
        if (n_cta > 1)
            cluster.sync();
        else
            __syncthreads();
        // The bin in which the count from above reaches `need`, in two steps of 64 groups of 32 bins, so that a
        // CTA reads 96 words of each of the others' histograms and not all of them.
        auto from_top = [&](int c, int& before, int& all) {   // lane 0 holds the highest
            int s = c;
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += y;
            }
            before = s - c;
            all = __shfl_sync(0xffffffffu, s, 31);
        };
        if (warp == 0) {
            int c[2] = {0, 0}, before[2], all[2];   // groups 63 - lane and 31 - lane
#pragma unroll
            for (int r = 0; r < EV_MAX_CLUSTER; ++r)
                if (r < n_cta) {
                    const int* h = n_cta > 1 ? cluster.map_shared_rank(groups[pass], r) : groups[pass];
                    c[0] += h[63 - lane];
                    c[1] += h[31 - lane];
                }
            from_top(c[0], before[0], all[0]);
            from_top(c[1], before[1], all[1]);
            before[1] += all[0];
            const unsigned hit0 = __ballot_sync(0xffffffffu, before[0] < need && before[0] + c[0] >= need);
            const unsigned hit1 = __ballot_sync(0xffffffffu, before[1] < need && before[1] + c[1] >= need);
            // fewer positions than needed: bin 0 is taken whole
            const int group = hit0 ? 63 - (__ffs(hit0) - 1) : hit1 ? 31 - (__ffs(hit1) - 1) : 0;
            const int above = hit0   ? __shfl_sync(0xffffffffu, before[0], __ffs(hit0) - 1)
                              : hit1 ? __shfl_sync(0xffffffffu, before[1], __ffs(hit1) - 1)
                                     : __shfl_sync(0xffffffffu, before[1], 31);
            int f = 0, fb, fa;
#pragma unroll
            for (int r = 0; r < EV_MAX_CLUSTER; ++r)
                if (r < n_cta) f += static_cast<int>((n_cta > 1 ? cluster.map_shared_rank(mine, r) : mine)[32 * group + 31 - lane]);
            from_top(f, fb, fa);
            fb += above;
            const unsigned hit = __ballot_sync(0xffffffffu, fb < need && fb + f >= need);
            const int at = hit ? __ffs(hit) - 1 : 31;
            if (lane == at) pick[0] = 32 * group + 31 - lane, pick[1] = fb, pick[2] = hit ? f : THREADS + 1;
        }
        __syncthreads();
        prefix |= static_cast<uint32_t>(pick[0]) << low;
        need -= pick[1];
        const int in_bin = pick[2];
        __syncthreads();
        if (in_bin <= EV_RANKED && pass + 1 < EV_PASSES) {
            // Few keys share the threshold's digits (2^-11 of the keys' spread, then 2^-22): the CTAs list theirs
            // and each key is ranked against the others, in place of the remaining passes.
            uint32_t* cand = hist + (pass + 1) * EV_BINS;   // zeroed; this CTA's, then behind EV_RANKED all of them
            if (tid == 0) n_cand = 0;
            __syncthreads();
            for (int i = tid; i < m; i += THREADS) {
                const uint32_t k = key(i);
                if (k && (k >> low) == (prefix >> low)) cand[atomicAdd(&n_cand, 1)] = k;
            }
            const uint32_t* all = cand;
            if (n_cta > 1) {
                cluster.sync();
                if (warp < n_cta && lane == 0) warp_gt[warp] = *cluster.map_shared_rank(&n_cand, warp);
                __syncthreads();
                if (warp < n_cta) {   // a warp per CTA's list; in_bin entries in all
                    const int c = warp_gt[warp], at = __reduce_add_sync(0xffffffffu, lane < warp ? warp_gt[lane] : 0);
                    const uint32_t* theirs = cluster.map_shared_rank(cand, warp);
                    for (int i = lane; i < c; i += 32) cand[EV_RANKED + at + i] = theirs[i];
                }
                all = cand + EV_RANKED;
            }
            __syncthreads();
            if (tid < in_bin) {
                const uint32_t k = all[tid];
                int above = 0, at = 0;
#pragma unroll 4
                for (int i = 0; i < in_bin; i += 4) {   // the list ends in zeros, which are no keys
                    const uint4 x = *reinterpret_cast<const uint4*>(all + i);
                    above += (x.x > k) + (x.y > k) + (x.z > k) + (x.w > k);
                    at += (x.x == k) + (x.y == k) + (x.z == k) + (x.w == k);
                }
                if (above < need && above + at >= need) pick[1] = static_cast<int>(k), pick[2] = need - above;   // equal keys write the same
            }
            __syncthreads();
            prefix = static_cast<uint32_t>(pick[1]);
            need = pick[2];
            break;   // other CTAs may still read this one's list: the next cluster barrier comes before any reuse
        }
    }
    // each warp's contiguous positions: how many are above the threshold, how many at it
    const int per = ((m + WARPS - 1) / WARPS + 31) & ~31;
    const int w0 = min(m, warp * per), w1 = min(m, w0 + per);
    int gt = 0, eq = 0;
    for (int i = w0 + lane; i - lane < w1; i += 32) {
        const uint32_t k = i < w1 ? key(i) : 0u;
        gt += __popc(__ballot_sync(0xffffffffu, k > prefix));
        eq += __popc(__ballot_sync(0xffffffffu, k && k == prefix));
    }
    if (lane == 0) warp_gt[warp] = gt, warp_eq[warp] = eq;
    __syncthreads();
    // before this warp, and in the whole CTA
    const int wg = lane < WARPS ? warp_gt[lane] : 0, we = lane < WARPS ? warp_eq[lane] : 0;
    int g0 = __reduce_add_sync(0xffffffffu, lane < warp ? wg : 0), e0 = __reduce_add_sync(0xffffffffu, lane < warp ? we : 0);
    int g_all = __reduce_add_sync(0xffffffffu, wg), e_all = __reduce_add_sync(0xffffffffu, we);
    if (n_cta > 1) {
        if (tid == 0) cta_sum = make_int2(g_all, e_all);
        cluster.sync();
        if (warp == 0) {
            const int2 s = lane < n_cta ? *cluster.map_shared_rank(&cta_sum, lane) : make_int2(0, 0);
            const int gb = __reduce_add_sync(0xffffffffu, lane < rank ? s.x : 0), eb = __reduce_add_sync(0xffffffffu, lane < rank ? s.y : 0);
            const int ga = __reduce_add_sync(0xffffffffu, s.x), ea = __reduce_add_sync(0xffffffffu, s.y);
            if (lane == 0) pick[0] = gb, pick[1] = eb, pick[2] = ga, n_cand = ea;
        }
        __syncthreads();
        g0 += pick[0], e0 += pick[1];
        g_all = pick[2], e_all = n_cand;
    }
    for (int i = w0 + lane; i - lane < w1; i += 32) {
        const uint32_t k = i < w1 ? key(i) : 0u;
        const bool above = k > prefix, at = k && k == prefix;
        const unsigned mg = __ballot_sync(0xffffffffu, above), me = __ballot_sync(0xffffffffu, at), below = (1u << lane) - 1u;
        const int eq_rank = e0 + __popc(me & below);
        if (above || (at && eq_rank < need)) kept[g0 + __popc(mg & below) + min(eq_rank, need)] = lo + i;
        g0 += __popc(mg);
        e0 += __popc(me);
    }
    const int total = g_all + min(e_all, need);
    for (int i = total + rank * THREADS + tid; i < a.n_keep; i += n_cta * THREADS) kept[i] = -1;
    if (tid == 0 && kv == 0 && rank == 0) a.new_len[seq] = total;
    if (n_cta > 1) cluster.sync();   // no CTA ends while another reads its counts
}

// A warp per EV_ROWS kept rows: K, V (16 bytes a lane, eight loads in flight) and the mass.  Bound by the memory:
// 64 x 2 x 2048 rows of 128 fp16 in 42 us, 6.4 TB/s read and written; a warp per row took 150 us.
constexpr int EV_ROWS = 8, EV_COPY_WARPS = 4;
template <typename T, int D>
__global__ void __launch_bounds__(32 * EV_COPY_WARPS) k_paged_evict_copy(const PagedGeom g, const EvictArgs a) {
    constexpr int CH = D * static_cast<int>(sizeof(T)) / 16, ITEMS = EV_ROWS * 2 * CH / 32;   // chunks of a row; 16-byte copies a lane
    const int i0 = (blockIdx.x * EV_COPY_WARPS + (threadIdx.x >> 5)) * EV_ROWS, kv = blockIdx.y, seq = blockIdx.z;
    const int lane = threadIdx.x & 31, i = i0 + lane;
    int sp, ss, dp = 0, ds = 0;
    // the table is final: the selection before this kernel lets it start only after its own wait
    const bool dst = lane < EV_ROWS && i < a.n_keep && g.locate(a.dst + static_cast<size_t>(seq) * g.max_pages, i, dp, ds);
    grid_dep_wait();
    grid_dep_launch();
    if (i0 >= a.n_keep) return;
    long long from = -1, to = -1;
    if (lane < EV_ROWS && i < a.n_keep) {
        const int j = a.kept[(static_cast<size_t>(seq) * g.n_head_kv + kv) * a.n_keep + i];
        if (j >= 0 && dst && g.locate(a.table + static_cast<size_t>(seq) * g.max_pages, j, sp, ss)) {
            from = g.row(sp, ss, kv);
            to = g.row(dp, ds, kv);
            a.mass[g.mass_at(dp, ds, kv)] = a.mass[g.mass_at(sp, ss, kv)];
        }
    }
    T *kc = static_cast<T*>(a.kc), *vc = static_cast<T*>(a.vc);
#pragma unroll
    for (int b = 0; b < ITEMS; b += 8) {
        uint4 x[8];
#pragma unroll
        for (int k = 0; k < 8 && b + k < ITEMS; ++k) {
            const int at = (b + k) * 32 + lane, r = at / (2 * CH), c = at % (2 * CH);
            const long long o = __shfl_sync(0xffffffffu, from, r);
            if (o >= 0) x[k] = __ldcs(reinterpret_cast<const uint4*>((c < CH ? kc : vc) + o) + c % CH);
        }
#pragma unroll
        for (int k = 0; k < 8 && b + k < ITEMS; ++k) {
            const int at = (b + k) * 32 + lane, r = at / (2 * CH), c = at % (2 * CH);
            const long long o = __shfl_sync(0xffffffffu, to, r);
            if (o >= 0) reinterpret_cast<uint4*>((c < CH ? kc : vc) + o)[c % CH] = x[k];
        }
    }
}

template <typename T>
cudaError_t launch_evict_copy(const PagedGeom& g, const EvictArgs& a, int n_seq, cudaStream_t s) {
    const int per = EV_ROWS * EV_COPY_WARPS;
    const dim3 grid((a.n_keep + per - 1) / per, g.n_head_kv, n_seq);
    return launch_dependent(g.head_dim == 64 ? k_paged_evict_copy<T, 64> : k_paged_evict_copy<T, 128>, grid, 32 * EV_COPY_WARPS, 0, s, g, a);
}

// One CTA for up to 3072 positions, more where the table has room for longer sequences (the lengths are the device's,
// the host does not know them) and SMs are free (8000
// positions: one CTA 16.6 us with the copy, two 15.5, four 13.3; 2112: one 11.4, two 12.3); CTAs of
// 512 threads, two to an SM, where there are more pairs than SMs (200 pairs of 2621 positions: a second wave of
// selections cost 9 us).
template <int THREADS>
cudaError_t prepare_select(int dev, int& widest) {   // per device: a repeated call finds the same again
    static int known[64] = {};
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!known[dev]) {
        auto* kernel = k_paged_evict_select<THREADS>;
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, EV_SMEM);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
        known[dev] = widest_cluster(EV_MAX_CLUSTER, [&](int width) { return active_clusters(kernel, width, THREADS, EV_SMEM); });
    }
    widest = known[dev];
    return cudaSuccess;
}
cudaError_t launch_evict_select(const PagedGeom& g, const EvictArgs& a, int n_seq, cudaStream_t s) {
    int dev = 0, n_sm = 0, widest = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = sm_count(dev, n_sm);
    if (e != cudaSuccess) return e;
    const long long room = static_cast<long long>(g.max_pages) * g.page_size, pairs = static_cast<long long>(n_seq) * g.n_head_kv;
    const bool many = pairs > n_sm;
    e = many ? prepare_select<512>(dev, widest) : prepare_select<1024>(dev, widest);
    if (e != cudaSuccess) return e;
    int cluster = 1;
    while (cluster < widest && cluster * 3072LL < room && pairs * cluster * 2 <= cluster_ctas(n_sm)) cluster *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(g.n_head_kv * cluster, n_seq);
    cfg.blockDim = dim3(many ? 512 : 1024);
    const long long keys = std::min<long long>(EV_KEYS, (room + cluster - 1) / cluster + 32);
    cfg.dynamicSmemBytes = (EV_PASSES * EV_BINS + static_cast<size_t>(keys)) * 4;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, many ? k_paged_evict_select<512> : k_paged_evict_select<1024>, g, a);
}

// ---------------------------------------------------------------- host side
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int kv_bytes(int kv_type) { return kv_type == MCPM_KV_F32 ? 4 : 2; }

// Checks a configuration and fills the kernels' geometry.
mcpm_status geometry(const mcpm_paged_config* c, PagedGeom& g) {
    if (!c) return MCPM_BAD_ARG;
    if (c->kv_type != MCPM_KV_F32 && c->kv_type != MCPM_KV_F16 && c->kv_type != MCPM_KV_BF16) return MCPM_UNSUPPORTED_TYPE;
    if (c->n_head_kv <= 0 || c->n_head <= 0 || c->n_head % c->n_head_kv || c->n_head / c->n_head_kv > PAGED_MAX_GROUP ||
        (c->head_dim != 64 && c->head_dim != 128) || c->page_size <= 0 || c->n_pages <= 0 || c->max_seqs <= 0 ||
        c->max_pages <= 0 || c->n_head > 4096 || c->max_seqs > 65535)
        return MCPM_BAD_ARG;
    constexpr long long most = 1 << 30;   // positions are ints with room for a block's stride
    if (static_cast<long long>(c->n_pages) * c->page_size > most || static_cast<long long>(c->max_pages) * c->page_size > most)
        return MCPM_BAD_ARG;
    g.n_head = c->n_head;
    g.n_head_kv = c->n_head_kv;
    g.head_dim = c->head_dim;
    g.page_size = c->page_size;
    g.n_pages = c->n_pages;
    g.max_pages = c->max_pages;
    g.page_stride = c->page_stride;
    g.row_stride = c->row_stride;
    g.head_stride = c->head_stride;
    if (!c->page_stride && !c->row_stride && !c->head_stride) {
        g.head_stride = c->head_dim;
        g.row_stride = static_cast<long long>(c->n_head_kv) * c->head_dim;
        g.page_stride = g.row_stride * c->page_size;
    }
    const long long per16 = 16 / kv_bytes(c->kv_type);
    if (g.page_stride <= 0 || g.row_stride <= 0 || g.head_stride <= 0 || g.page_stride % per16 || g.row_stride % per16 ||
        g.head_stride % per16)
        return MCPM_BAD_ARG;
    g.by_page.set(static_cast<uint32_t>(c->page_size));
    return MCPM_OK;
}

mcpm_status check_pool(const mcpm_paged_pool* p) {
    return p && p->k && p->v && aligned16(p->k) && aligned16(p->v) ? MCPM_OK : MCPM_BAD_ARG;
}

mcpm_status status(const char* what, cudaError_t e) {
    if (e == cudaSuccess) return MCPM_OK;
    std::fprintf(stderr, "[mcpm] %s: CUDA error: %s\n", what, cudaGetErrorString(e));
    return MCPM_CUDA_ERROR;
}

}  // namespace
}  // namespace mcpm

using namespace mcpm;

extern "C" {

size_t mcpm_paged_workspace_bytes(const mcpm_paged_config* cfg) {
    PagedGeom g;
    return geometry(cfg, g) == MCPM_OK ? paged_attention_workspace(g, cfg->max_seqs) : 0;
}

mcpm_status mcpm_rope_table(float* out, int n_pos, int head_dim, float rope_base) {
    if (!out || n_pos <= 0 || head_dim <= 0 || head_dim % 2 || !(rope_base > 0.0f)) return MCPM_BAD_ARG;
    const float inv = 1.0f / static_cast<float>(head_dim);
    for (int i = 0; i < head_dim; i += 2) {
        const float theta = powf(rope_base, -(static_cast<float>(i) * inv));
        for (int pos = 0; pos < n_pos; ++pos) {
            const float angle = theta * static_cast<float>(pos);
            float* o = out + static_cast<size_t>(pos) * head_dim + i;
            o[0] = cosf(angle);
            o[1] = sinf(angle);
        }
    }
    return MCPM_OK;
}

mcpm_status mcpm_paged_append(const mcpm_paged_config* cfg, const mcpm_paged_pool* pool, const int* table, int n_seq,
                              const mcpm_paged_tokens* tokens, void* stream) {
    PagedGeom g;
    mcpm_status st = geometry(cfg, g);
    if (st == MCPM_OK) st = check_pool(pool);
    if (st != MCPM_OK) return st;
    if (!tokens || !table || n_seq <= 0 || n_seq > cfg->max_seqs) return MCPM_BAD_ARG;
    AppendArgs a{*tokens, table, pool->k, pool->v, pool->mass, n_seq};
    mcpm_paged_tokens& t = a.t;
    const int q_row = g.n_head * g.head_dim, kv_row = g.n_head_kv * g.head_dim;
    if (t.q_stride == 0) t.q_stride = q_row;
    if (t.kv_stride == 0) t.kv_stride = kv_row;
    if (t.n_tok < 0 || !t.tok_slot || !t.k || !t.v || !aligned16(t.k) || !aligned16(t.v) || t.kv_stride < kv_row ||
        t.kv_stride % 4)
        return MCPM_BAD_ARG;
    if (t.q && (!t.q_out || !aligned16(t.q) || !aligned16(t.q_out) || t.q_stride < q_row || t.q_stride % 4 ||
                (t.q_out == t.q && t.q_stride != q_row)))
        return MCPM_BAD_ARG;
    if (t.rope && (t.rope_len <= 0 || !aligned16(t.rope))) return MCPM_BAD_ARG;
    if (t.n_tok == 0) return MCPM_OK;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return status("mcpm_paged_append", cfg->kv_type == MCPM_KV_F32   ? launch_append<float>(g, a, s)
                                       : cfg->kv_type == MCPM_KV_F16 ? launch_append<__half>(g, a, s)
                                                                     : launch_append<__nv_bfloat16>(g, a, s));
}

mcpm_status mcpm_paged_attention(const mcpm_paged_config* cfg, const mcpm_paged_pool* pool, const int* table,
                                 const int* seq_len, int n_seq, const float* q, int64_t q_stride, float* out,
                                 float scale, void* ws, size_t ws_bytes, void* stream) {
    PagedGeom g;
    mcpm_status st = geometry(cfg, g);
    if (st == MCPM_OK) st = check_pool(pool);
    if (st != MCPM_OK) return st;
    if (q_stride == 0) q_stride = static_cast<int64_t>(g.n_head) * g.head_dim;
    if (!table || !seq_len || !q || !out || !ws || n_seq <= 0 || n_seq > cfg->max_seqs || !aligned16(q) || !aligned16(out) ||
        !aligned16(ws) || ws_bytes < paged_attention_workspace(g, cfg->max_seqs) || q_stride < static_cast<int64_t>(g.n_head) * g.head_dim ||
        q_stride % 4 || !(scale >= 0.0f))
        return MCPM_BAD_ARG;
    if (scale == 0.0f) scale = 1.0f / sqrtf(static_cast<float>(g.head_dim));
    return status("mcpm_paged_attention",
                  launch_paged_attention(g, cfg->kv_type, cfg->max_seqs, pool->k, pool->v, pool->mass, table, seq_len, n_seq, q,
                                         q_stride, out, scale, ws, static_cast<cudaStream_t>(stream)));
}

mcpm_status mcpm_paged_evict(const mcpm_paged_config* cfg, const mcpm_paged_pool* pool, const int* table,
                             const int* seq_len, const int* dst_table, int* new_len, int* kept, int n_seq, int n_keep,
                             int n_sink, int n_recent, void* ws, size_t ws_bytes, void* stream) {
    PagedGeom g;
    mcpm_status st = geometry(cfg, g);
    if (st == MCPM_OK) st = check_pool(pool);
    if (st != MCPM_OK) return st;
    if (!pool->mass || !table || !seq_len || !dst_table || dst_table == table || !new_len || !kept || !ws || n_seq <= 0 ||
        n_seq > cfg->max_seqs || n_keep <= 0 || n_sink < 0 || n_recent < 0 || n_sink > n_keep || n_recent > n_keep - n_sink ||
        n_keep > g.max_pages * g.page_size || !aligned16(ws) || ws_bytes < paged_attention_workspace(g, cfg->max_seqs))
        return MCPM_BAD_ARG;
    EvictArgs a{pool->k, pool->v, pool->mass, table, seq_len, dst_table, new_len, kept, n_keep, n_sink, n_recent};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = launch_evict_select(g, a, n_seq, s);
    if (e == cudaSuccess)
        e = cfg->kv_type == MCPM_KV_F32   ? launch_evict_copy<float>(g, a, n_seq, s)
            : cfg->kv_type == MCPM_KV_F16 ? launch_evict_copy<__half>(g, a, n_seq, s)
                                          : launch_evict_copy<__nv_bfloat16>(g, a, n_seq, s);
    return status("mcpm_paged_evict", e);
}

}  // extern "C"
