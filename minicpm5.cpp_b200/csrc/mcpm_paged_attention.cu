// Attention of one query per sequence over a paged KV cache, in one pass over K and V:
//   s_hj = scale q_h . K_j,  m_h = max_j s_hj,  l_h = sum_j exp(s_hj - m_h),
//   out_h = sum_j exp(s_hj - m_h) V_j / l_h
// with a running m, l and unnormalised output per warp, joined at the end of each (sequence, KV head).
//
// The g query heads of a KV head share its rows, so the products are matrix products with g columns:
// S^T (16 positions x 8 heads) = K (16 x D) q^T and O^T (D x 8 heads) += V^T (D x 16) P^T, on warp-level
// tensor-core instructions whose 8-wide N side the heads fill.  The work is bound by the bytes of K and V
// (2 D esz per position and KV head against 4 g D operations), far below the rate at which 128-row
// tensor-memory instructions would pay for their padding of g heads.
//
// fp32 results.  Operands of the cache type are exact; the fp32 operands (q, and the weights P) are split
// into parts of that type, two for fp16 (22 bits), three for bf16 (24 bits); an fp32 cache is itself split
// into two tf32 parts, with the three products that matter.  Accumulators are fp32.
//
// Work is split over the grid in units of 128 positions: the units of all (sequence, KV head) pairs in a
// row, an equal share per CTA.  A pair that spans several CTAs leaves a partial result per CTA, and the
// CTA that arrives last joins them in order of position, so results do not depend on arrival order.
//
// Measured (16 query heads, 2 KV heads, 128 dims): 4 x 131072 positions of fp16 95 us, 5.7 TB/s; of fp32 181 us,
// 5.9 TB/s; bound by the memory (a device copy: 6.46 TB/s).  Short calls are bound by a chain of round trips:
// lengths, page table, K, V, then record, arrival and join where a pair is split: 8193 fp32 positions 13.6 us,
// of which 2.6 us are bytes; 137 positions 8.7 us.  With one KV head, whose 16 heads take two products a tile,
// 4 x 131072 fp16 positions take 65 us, 4.1 TB/s: eight warps an SM carry twice the products.
#include <algorithm>
#include <cmath>

#include "../../include/mcpm.h"
#include "mcpm_device.cuh"
#include "mcpm_paged.cuh"

namespace mcpm {
namespace {

constexpr int WARPS = 8, THREADS = 32 * WARPS;
constexpr int ROWS = 16;            // positions of a warp's tile
constexpr int UNIT = ROWS * WARPS;  // positions of a unit of work
constexpr int FAN = 16, FAN_BITS = 4, LEVELS = 3;   // records joined at a time, FAN^LEVELS >= PAGED_MAX_CTAS
// Shares are equal in steps: a pair's steps are its units and LEAD before them, for what a pair costs beside its
// units (q, the join of the warps, the output).  An end of a share inside a pair of at most WHOLE units, among its
// LEAD steps or within `slack` units of one of its ends moves to that end: the rest would cost more as a record
// with its arrival and join than as work.
constexpr int WHOLE = 2, LEAD = 1;   // LEAD 1, 2, 3: 30.6, 31.6, 32.8 us at 200 sequences of 20 to 900 fp16 positions
constexpr float LOG2E = 1.4426950408889634f;

template <typename T>
constexpr int parts() { return sizeof(T) == 4 || __is_same(T, __half) ? 2 : 3; }
// Powers of two that keep parts and products in range.  fp16 parts have five bits of exponent: weights are multiplied
// by 1024 and q brought to [2^7, 2^8), so that the parts of small ones stay normal, and no product of values up to
// 65504 comes near the end of fp32.  The other parts have fp32's eight bits: weights stay as they are, and q is brought
// to [2^-8, 2^-7), where 128 products with finite values cannot exceed the largest of them.  Undone in the output and
// in the factor of the scores.
template <typename T>
constexpr float p_scale() { return __is_same(T, __half) ? 1024.0f : 1.0f; }
template <typename T>
constexpr int q_exponent() { return __is_same(T, __half) ? 7 : -8; }

template <typename T, int D, int NT>
struct Tile {
    static constexpr int RB = D * static_cast<int>(sizeof(T));   // bytes of a row
    static constexpr int CHUNKS = RB / 16;
    static constexpr int HALF = ROWS * RB;      // a tile's K, or its V: one slot of the warp's ring
    static constexpr int WHERE = 8;             // tiles whose rows' places are remembered
    static constexpr int KSTEPS = sizeof(T) == 4 ? D / 8 : D / 16;
    static constexpr int QWORDS = parts<T>() * 2;   // words of q per lane, k step and 8 heads
    static constexpr int OTHER = WARPS * WHERE * ROWS * 4 + KSTEPS * NT * 32 * QWORDS * 4;
    // Two CTAs per SM where 128 registers hold a thread's part of the output, else one.  The slots take what
    // memory is left: 128 KB of copies in flight per SM.
    static constexpr int CTAS = sizeof(T) == 2 && D == 64 && NT == 1 ? 2 : 1;
    static constexpr int FIT = ((CTAS == 2 ? 109 : 222) * 1024 - OTHER) / (WARPS * HALF);
    static constexpr int SLOTS = FIT < 8 ? FIT : 8;
    static constexpr int SMEM = WARPS * SLOTS * HALF + OTHER;
    static_assert(SLOTS >= 3 && 8 * D * 4 <= HALF, "a slot holds a warp's output for 8 heads");
    static_assert(SLOTS / 2 + 2 <= WHERE, "");
    // The 16-byte chunks of a row are swizzled so that the fragment loads are conflict-free: ldmatrix reads one
    // chunk of 8 rows; the fp32 loads of 16 bytes per lane read, 8 lanes at a time, 4 chunks of 2 rows (K) or
    // 2 chunks of 4 rows (V).
    static __device__ __forceinline__ int k_swz(int r) { return sizeof(T) == 4 ? (r & 1) << 2 : r & 7; }
    static __device__ __forceinline__ int v_swz(int r) { return sizeof(T) == 4 ? (r & 3) << 1 : r & 7; }
};

struct AttArgs {
    const void *kc, *vc;
    const int *table, *len;
    const float* q;
    long long q_stride;
    float* out;
    float scale;
    int n_seq, group;
    unsigned* cnt;     // [LEVELS][slot of the first record] arrivals, zero between calls
    float2* stats;     // [seq][head] (max in units of log2, 1 / sum); mass only
    float* part;       // [2 CTA + which][m[group], l[group], pad to 32, o[group][D]]
    float* scores;     // [page * page_size + slot][n_head] scores in units of log2; mass only
};

__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, bool fill) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(fill ? 0 : 16) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float4 lds_f4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (sizeof(T) == 4)
        asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else if constexpr (__is_same(T, __half))
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// x = hi + lo in tf32.  The instruction drops the 13 lowest bits of an operand, so of a cache element x itself
// serves as hi, and what it drops as lo: two operations.  q and the weights are split with rounding instead, so
// that their lo parts have mean zero and the omitted lo * lo does not add up (rms error of a score of 128 random
// products 2.1e-7, with truncation on both sides 5.1e-7, an fp32 sum 1.5e-7).
__device__ __forceinline__ uint32_t tf32_hi(float x) { return __float_as_uint(x); }
__device__ __forceinline__ uint32_t tf32_lo(float x) {
    return __float_as_uint(x - __uint_as_float(__float_as_uint(x) & 0xffffe000u));
}
__device__ __forceinline__ void tf32_round(float x, uint32_t& hi, uint32_t& lo) {   // |x| well below the largest float
    hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi)) + 0x1000u;
}
// 2^x with 2 ulp, results below 2^-126 zero.
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Part i of a value in 16-bit parts; x becomes what is left.
template <typename T>
__device__ __forceinline__ uint16_t take_part(float& x) {
    if constexpr (__is_same(T, __half)) {
        const __half h = __float2half_rn(x);
        x -= __half2float(h);
        return __half_as_ushort(h);
    } else {
        const __nv_bfloat16 h = __float2bfloat16_rn(x);
        x -= __bfloat162float(h);
        return __bfloat16_as_ushort(h);
    }
}
template <typename T>
__device__ __forceinline__ uint32_t take_parts2(float& x, float& y) {   // x in the lower half
    const uint32_t a = take_part<T>(x);
    return a | static_cast<uint32_t>(take_part<T>(y)) << 16;
}

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

// a / b for 0 <= a, 0 < b: 32-bit where it can be, a fifth of the time.
__device__ __forceinline__ long long quotient(long long a, long long b) {
    return (a | b) <= 0xffffffffLL ? static_cast<long long>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b)) : a / b;
}
// Equal shares of `total` units for n <= total CTAs, the first total % n of them one unit longer.
struct Shares {
    long long per, rem;
    __device__ Shares(long long total, int n) : per(quotient(total, n)), rem(total - per * n) {}
    __device__ long long start(int c) const { return c * per + min(static_cast<long long>(c), rem); }
    __device__ int of(long long unit) const {
        const long long wide = rem * (per + 1);
        return static_cast<int>(unit < wide ? quotient(unit, per + 1) : rem + quotient(unit - wide, per));
    }
};

template <typename T, int D, int NT, bool MASS>
__global__ void __launch_bounds__(THREADS, Tile<T, D, NT>::CTAS) k_paged_attention(const PagedGeom g, const AttArgs a) {
    using L = Tile<T, D, NT>;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ long long s_sum[WARPS], s_at[2];
    __shared__ int s_seq, s_kv, s_u, s_last;
    __shared__ float s_qf[8 * NT];              // scale of a head's scores in units of log2
    __shared__ float s_m[WARPS][8 * NT], s_l[WARPS][8 * NT], s_inv[8 * NT];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gq = lane >> 2, t4 = lane & 3;
    uint8_t* ring = smem + warp * L::SLOTS * L::HALF;   // slot i % SLOTS: K of tile i / 2 (i even) or its V (i odd)
    int* where = reinterpret_cast<int*>(smem + WARPS * L::SLOTS * L::HALF) + warp * L::WHERE * ROWS;   // physical slots, -1: not visible
    uint32_t* qs = reinterpret_cast<uint32_t*>(smem + WARPS * L::SLOTS * L::HALF + WARPS * L::WHERE * ROWS * 4);
    const T *kc = static_cast<const T*>(a.kc), *vc = static_cast<const T*>(a.vc);
    const int group = a.group, hkv = g.n_head_kv;

    grid_dep_launch();
    grid_dep_wait();
    // ---- this CTA's share of the units
    auto units_of = [&](int seq) { return (g.clamp_len(a.len[seq]) + UNIT - 1) / UNIT; };
    auto steps_of = [](int units) { return units ? units + LEAD : 0; };
    const int per = (a.n_seq + THREADS - 1) / THREADS;
    long long mine = 0;
    for (int i = tid * per; i < min(a.n_seq, (tid + 1) * per); ++i) mine += steps_of(units_of(i));
    long long before = mine;   // inclusive scan over the threads
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += x;
    }
    if (lane == 31) s_sum[warp] = before;
    __syncthreads();
    long long total = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        if (w < warp) before += s_sum[w];
        total += s_sum[w];
    }
    before = (before - mine) * hkv;
    total *= hkv;
    const int n_cta = static_cast<int>(min(static_cast<long long>(gridDim.x), total));
    // sequences without positions: zeros
    for (int seq = blockIdx.x; seq < a.n_seq; seq += gridDim.x)
        if (a.len[seq] <= 0)
            for (int i = tid; i < g.n_head * D; i += THREADS) a.out[static_cast<size_t>(seq) * g.n_head * D + i] = 0.0f;
    if (static_cast<int>(blockIdx.x) >= n_cta) return;
    // where this share begins and the next one does
    const Shares shares(total, n_cta);
    const int slack = shares.per >= 8 ? 1 : 0;
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        const long long f = shares.start(blockIdx.x + side);
        long long base = before;
        if (f == total && tid == 0 && side) s_at[1] = total;
        if (f >= base && f < base + mine * hkv)
            for (int i = tid * per;; ++i) {
                const int units = units_of(i), steps = steps_of(units);
                if (f < base + static_cast<long long>(steps) * hkv) {
                    const int kv = static_cast<int>(quotient(f - base, steps));
                    const long long seg0 = base + static_cast<long long>(kv) * steps;
                    const int u = max(static_cast<int>(f - seg0) - LEAD, 0);
                    const bool near = units <= WHOLE || min(u, units - u) <= slack, down = near && u <= units - u, up = near && !down;
                    s_at[side] = up ? seg0 + steps : down ? seg0 : f;   // in steps
                    if (side == 0) s_seq = i, s_kv = kv + up, s_u = near ? 0 : u;
                    break;
                }
                base += static_cast<long long>(steps) * hkv;
            }
    }
    __syncthreads();
    long long at = s_at[0];
    const long long end = s_at[1];   // steps of this CTA; every pair in them begins there or at unit s_u
    if (at >= end) return;
    int seq = s_seq, kv = s_kv, u = s_u;
    if (kv == hkv) {
        kv = 0;
        do ++seq;
        while (units_of(seq) == 0);   // ends: steps follow
    }
    int units = units_of(seq);
    long long seg0 = u ? at - u - LEAD : at;   // first step of the pair
    auto end_of = [&](long long seg, int n_units) { return static_cast<int>(min(static_cast<long long>(n_units), end - seg - LEAD)); };
    int u_end = end_of(seg0, units);   // this CTA has the pair's units u .. u_end - 1

    // ---- copies of K and V, SLOTS - 1 half tiles ahead of the products whatever pair they belong to, so the memory
    // does not idle where one pair ends and the next begins.  Lane & 15 looks one row of the warp's tile up a unit
    // before its copy, all lanes copy.
    struct Ahead {
        int page, slot, kv;
    };
    int p_seq = seq, p_kv = kv, p_u = u, p_units = units, p_end = u_end, p_len = g.clamp_len(a.len[seq]);
    long long p_seg0 = seg0;
    auto look = [&](Ahead& x) {   // past the last unit: no page, hence no copies
        x = Ahead{-1, 0, p_kv};
        if (p_seg0 >= end) return;
        const int j = p_u * UNIT + warp * ROWS + (lane & 15), c = static_cast<int>(g.by_page.div(static_cast<uint32_t>(j)));
        x.slot = j - c * g.page_size;
        if (j < p_len) x.page = __ldg(a.table + static_cast<size_t>(p_seq) * g.max_pages + c);
        if (++p_u == p_end) {
            p_seg0 += p_units + LEAD;
            if (p_seg0 >= end) return;
            p_u = 0;
            if (++p_kv == hkv) {
                p_kv = 0;
                do p_len = g.clamp_len(a.len[++p_seq]);
                while (p_len == 0);   // ends: steps are left
                p_units = (p_len + UNIT - 1) / UNIT;
            }
            p_end = end_of(p_seg0, p_units);
        }
    };
    Ahead next;
    long long off = -1;   // this lane's row of the tile whose K was issued last
    bool some = false;    // that tile has a visible row
    bool plain = false;   // all 16 are visible and lie row_stride apart (one page)
    const int r0 = lane / L::CHUNKS, c0 = lane % L::CHUNKS;
    constexpr int RSTEP = 32 / L::CHUNKS;   // rows of one instruction
    const long long lane_off = r0 * g.row_stride + c0 * (16 / static_cast<int>(sizeof(T))), step_off = RSTEP * g.row_stride;
    auto copy = [&](int slot, const T* pool, bool is_v) {
        const uint32_t dst = smem_u32(ring + slot * L::HALF);
        if (plain) {
            const T* src = pool + __shfl_sync(0xffffffffu, off, 0) + lane_off;
#pragma unroll
            for (int i = 0; i < ROWS / RSTEP; ++i, src += step_off) {
                const int r = i * RSTEP + r0;
                cp_async16(dst + r * L::RB + ((c0 ^ (is_v ? L::v_swz(r) : L::k_swz(r))) << 4), src);
            }
        } else {
#pragma unroll 1
            for (int i = 0; i < ROWS / RSTEP; ++i) {
                const int r = i * RSTEP + r0;
                const long long o = __shfl_sync(0xffffffffu, off, r);
                cp_async16_zfill(dst + r * L::RB + ((c0 ^ (is_v ? L::v_swz(r) : L::k_swz(r))) << 4),
                                 pool + (o < 0 ? 0 : o) + c0 * (16 / sizeof(T)), o < 0);
            }
        }
    };
    auto issue_k = [&](int k, int slot, const Ahead& x) {
        const bool ok = static_cast<unsigned>(x.page) < static_cast<unsigned>(g.n_pages);
        off = ok ? g.row(x.page, x.slot, x.kv) : -1;
        const long long top_row = __shfl_sync(0xffffffffu, off, 0);
        some = __any_sync(0xffffffffu, ok);
        plain = __all_sync(0xffffffffu, ok && off == top_row + (lane & 15) * g.row_stride);
        if (lane < 16) where[k % L::WHERE * ROWS + lane] = ok ? x.page * g.page_size + x.slot : -1;
        if (some) copy(slot, kc, false);
        cp_async_commit();
    };
    auto issue_v = [&](int slot) {
        if (some) copy(slot, vc, true);
        cp_async_commit();
    };
    auto issue = [&](int half, int slot) {   // in order; half's parity is known at compile time
        if (half & 1) {
            issue_v(slot);
        } else {
            issue_k(half / 2, slot, next);
            look(next);
        }
    };
    // q of a pair: heads warp, warp + WARPS, ... of its group
    float qx[NT][D / 32];
    auto load_q = [&](int q_seq, int q_kv) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int h = warp + WARPS * i;
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
                qx[i][d] = h < group ? a.q[q_seq * a.q_stride + static_cast<size_t>(q_kv * group + h) * D + lane + 32 * d] : 0.0f;
        }
    };
    look(next);
    load_q(seq, kv);
#pragma unroll 1
    for (int i = 0; i < L::SLOTS - 1; ++i) issue(i, i);

    // ---- A pair of several CTAs leaves a record (m, l, o) per CTA.  Records are joined FAN at a time, in order
    // of position, by the CTA that arrives last at them; its result is a record of the next level, and the
    // last level's is the output.  One CTA reading all records of a long sequence took 7 us of a 20 us call.
    const int rec = 2 * PAGED_MAX_GROUP + group * D;   // floats of a record
    auto arrive = [&](int level, int slot, int members) {   // thread 0, after the CTA's stores and a barrier
        unsigned* c = a.cnt + level * 2 * PAGED_MAX_CTAS + slot;
        unsigned before;   // release of the CTA's record, acquire of the others'
        asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(c) : "memory");
        const bool last = before == static_cast<unsigned>(members - 1);
        if (last) *c = 0u;
        return last;
    };
    struct Shared {   // a pair of CTAs first .. first + np - 1, this one's record being the k-th
        int seq, kv, first, np, k;
    };
    auto slot_of = [](const Shared& s, int k) { return 2 * (s.first + k) + (k == 0); };   // a CTA begins one pair at most
    auto members_of = [](const Shared& s, int level) {
        const int step = 1 << FAN_BITS * level, at = s.k >> FAN_BITS * (level + 1) << FAN_BITS * (level + 1);
        return min(FAN, (s.np - at + step - 1) >> FAN_BITS * level);
    };
    auto join = [&](Shared s) {   // s_last: whether this CTA arrived last at its first FAN records
        for (int level = 0; s_last; ++level) {
            const int at = s.k >> FAN_BITS * (level + 1) << FAN_BITS * (level + 1), members = members_of(s, level);
            const bool done = s.np <= 1 << FAN_BITS * (level + 1);
            float* to = a.part + static_cast<size_t>(slot_of(s, at)) * rec;
            float* out = a.out + (static_cast<size_t>(s.seq) * g.n_head + s.kv * group) * D;
            for (int i0 = 32 * warp; i0 < group * D / 4; i0 += THREADS) {   // whole warps: a head's items are one warp's
                const int i = min(i0 + lane, group * D / 4 - 1), h = 4 * i / D;
                const bool mine = i == i0 + lane;
                float top = -INFINITY, sum = 0.0f;
                float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                constexpr int TOGETHER = L::CTAS == 1 ? FAN : 8;   // records whose loads are in flight
#pragma unroll 1
                for (int j0 = 0; j0 < members; j0 += TOGETHER) {
                    float mr[TOGETHER], lr[TOGETHER];
                    float4 r[TOGETHER];
#pragma unroll
                    for (int j = 0; j < TOGETHER; ++j) {
                        mr[j] = -INFINITY, lr[j] = 0.0f, r[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        if (j0 + j < members) {
                            const float* p = a.part + static_cast<size_t>(slot_of(s, at + ((j0 + j) << FAN_BITS * level))) * rec;
                            mr[j] = __ldcg(p + h);
                            lr[j] = __ldcg(p + PAGED_MAX_GROUP + h);
                            r[j] = __ldcg(reinterpret_cast<const float4*>(p + 2 * PAGED_MAX_GROUP) + i);
                        }
                    }
                    float to_top = top;
#pragma unroll
                    for (int j = 0; j < TOGETHER; ++j) to_top = fmaxf(to_top, mr[j]);
                    const float keep = top == -INFINITY ? 0.0f : fast_exp2(top - to_top);
                    sum *= keep;
                    x = make_float4(x.x * keep, x.y * keep, x.z * keep, x.w * keep);
                    top = to_top;
#pragma unroll
                    for (int j = 0; j < TOGETHER; ++j) {
                        const float e = mr[j] == -INFINITY ? 0.0f : fast_exp2(mr[j] - top);
                        sum = fmaf(lr[j], e, sum);
                        x = make_float4(fmaf(r[j].x, e, x.x), fmaf(r[j].y, e, x.y), fmaf(r[j].z, e, x.z), fmaf(r[j].w, e, x.w));
                    }
                }
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum, f = done ? inv * (1.0f / p_scale<T>()) : 1.0f;
                const float4 y = make_float4(x.x * f, x.y * f, x.z * f, x.w * f);
                if (done) {
                    if (mine) reinterpret_cast<float4*>(out)[i] = y;
                    if (MASS && mine && 4 * i % D == 0) a.stats[static_cast<size_t>(s.seq) * g.n_head + s.kv * group + h] = make_float2(top, inv);
                } else {
                    __syncwarp();   // the record is joined in place: all lanes have read it
                    if (mine) reinterpret_cast<float4*>(to + 2 * PAGED_MAX_GROUP)[i] = y;
                    if (mine && 4 * i % D == 0) to[h] = top, to[PAGED_MAX_GROUP + h] = sum;
                }
            }
            __syncthreads();
            if (done) break;
            s.k = at;
            if (tid == 0) s_last = arrive(level + 1, slot_of(s, s.k >> FAN_BITS * (level + 2) << FAN_BITS * (level + 2)), members_of(s, level + 1));
            __syncthreads();
        }
    };
    Shared open{-1, 0, 0, 0, 0};   // this CTA's first pair, if other CTAs share it
    bool open_last = false;

    int before_slot, k_slot, v_slot = L::SLOTS - 1;   // slots of the last tile's V and of this tile's K and V
    for (int k = 0; seg0 < end;) {
        // ---- q in fragment order, normalised per head
#pragma unroll
        for (int qi = 0; qi < NT; ++qi) {
            const int h = warp + WARPS * qi;
            const float(&x)[D / 32] = qx[qi];
            float top = 0.0f;
            for (int i = 0; i < D / 32; ++i) top = fmaxf(top, fabsf(x[i]));
            for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const int e = min(max(q_exponent<T>() - (static_cast<int>(__float_as_uint(top) >> 23) - 127), -120), 120);
            const float up = pow2(e);
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                float v = x[i] * up;
                const int d = lane + 32 * i;
                if constexpr (sizeof(T) == 4) {
                    // dims 16 c + 4 t + (0, 1, 2, 3) of lane t: k = t and t + 4 of steps 2c and 2c + 1
                    const int ks = 2 * (d / 16) + ((d >> 1) & 1), t = (d >> 2) & 3, w = d & 1;
                    uint32_t* p = qs + ((ks * NT + (h >> 3)) * 32 + (h & 7) * 4 + t) * 4;
                    tf32_round(v, p[w], p[2 + w]);
                } else {
                    const int ks = d / 16, r = d & 15, t = (r & 7) >> 1, w = r >> 3;
                    uint16_t* p = reinterpret_cast<uint16_t*>(qs + ((ks * NT + (h >> 3)) * 32 + (h & 7) * 4 + t) * L::QWORDS + w) + (r & 1);
#pragma unroll
                    for (int k = 0; k < parts<T>(); ++k) p[4 * k] = take_part<T>(v);
                }
            }
            if (lane == 0) s_qf[h] = a.scale * pow2(-e) * LOG2E;   // in this order: a scale for large K may be subnormal
        }
        __syncthreads();
        float qf[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) qf[nt][0] = s_qf[8 * nt + 2 * t4], qf[nt][1] = s_qf[8 * nt + 2 * t4 + 1];

        float o[NT][D / 16][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.0f;
        }

        for (const int k1 = k + u_end - u; k < k1; ++k) {
            before_slot = v_slot;
            k_slot = v_slot + 1 == L::SLOTS ? 0 : v_slot + 1;
            v_slot = k_slot + 1 == L::SLOTS ? 0 : k_slot + 1;
            cp_async_wait_group<L::SLOTS - 2>();
            __syncwarp();   // K is in shared memory for all lanes, and all are done with the V before it
            issue(2 * k + L::SLOTS - 1, before_slot);
            const int where0 = where[k % L::WHERE * ROWS + gq], where1 = where[k % L::WHERE * ROWS + gq + 8];
            if (!__any_sync(0xffffffffu, where0 >= 0 || where1 >= 0)) {   // nothing visible: beyond the length, absent pages
                cp_async_wait_group<L::SLOTS - 2>();
                __syncwarp();
                issue(2 * k + L::SLOTS, k_slot);
                continue;
            }
            const uint32_t ks = smem_u32(ring + k_slot * L::HALF), vs = smem_u32(ring + v_slot * L::HALF);

            // ---- scores
            // Independent accumulators: the instruction truncates, so short chains lose less, and they overlap.
            constexpr int LO = sizeof(T) == 4 ? 4 : 2 * (parts<T>() - 1);
            float s[NT][4], s_hi[NT][2][4], s_lo[NT][LO][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s_hi[nt][0][i] = s_hi[nt][1][i] = 0.0f;
                    for (int c = 0; c < LO; ++c) s_lo[nt][c][i] = 0.0f;
                }
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int c = 0; c < D / 16; ++c) {
                    const uint32_t at = ks + gq * L::RB + (((4 * c + t4) ^ L::k_swz(gq)) << 4);
                    const float4 r0 = lds_f4(at), r8 = lds_f4(at + 8 * L::RB);
                    uint32_t hi[2][4], lo[2][4];
                    hi[0][0] = tf32_hi(r0.x), lo[0][0] = tf32_lo(r0.x);
                    hi[0][1] = tf32_hi(r8.x), lo[0][1] = tf32_lo(r8.x);
                    hi[0][2] = tf32_hi(r0.y), lo[0][2] = tf32_lo(r0.y);
                    hi[0][3] = tf32_hi(r8.y), lo[0][3] = tf32_lo(r8.y);
                    hi[1][0] = tf32_hi(r0.z), lo[1][0] = tf32_lo(r0.z);
                    hi[1][1] = tf32_hi(r8.z), lo[1][1] = tf32_lo(r8.z);
                    hi[1][2] = tf32_hi(r0.w), lo[1][2] = tf32_lo(r0.w);
                    hi[1][3] = tf32_hi(r8.w), lo[1][3] = tf32_lo(r8.w);
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const uint4 b = *reinterpret_cast<const uint4*>(qs + (((2 * c + k) * NT + nt) * 32 + lane) * 4);
                            mma<T>(s_hi[nt][k], hi[k], b.x, b.y);
                            mma<T>(s_lo[nt][k], hi[k], b.z, b.w);
                            mma<T>(s_lo[nt][2 + k], lo[k], b.x, b.y);
                        }
                }
            } else {
#pragma unroll
                for (int c = 0; c < D / 16; ++c) {
                    uint32_t k[4];
                    ldsm4(k, ks + (lane & 15) * L::RB + (((2 * c + (lane >> 4)) ^ L::k_swz(lane)) << 4));
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const uint2* b = reinterpret_cast<const uint2*>(qs + ((c * NT + nt) * 32 + lane) * L::QWORDS);
                        mma<T>(s_hi[nt][c & 1], k, b[0].x, b[0].y);
#pragma unroll
                        for (int p = 1; p < parts<T>(); ++p) mma<T>(s_lo[nt][2 * (p - 1) + (c & 1)], k, b[p].x, b[p].y);
                    }
                }
            }
            // ---- weights: lane (gq, t4) holds positions gq, gq + 8 of heads 2 t4, 2 t4 + 1
            float keep[NT][2];   // factor of what was summed before this tile
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float lo = s_lo[nt][0][i] + s_lo[nt][1][i];
                    if constexpr (LO == 4) lo += s_lo[nt][2][i] + s_lo[nt][3][i];
                    s[nt][i] = s_hi[nt][0][i] + s_hi[nt][1][i] + lo;
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float x = where0 >= 0 ? s[nt][i] * qf[nt][i] : -INFINITY;
                    const float y = where1 >= 0 ? s[nt][2 + i] * qf[nt][i] : -INFINITY;
                    if constexpr (MASS) {
                        const int h = 8 * nt + 2 * t4 + i;
                        if (h < group && where0 >= 0) a.scores[static_cast<size_t>(where0) * g.n_head + kv * group + h] = x;
                        if (h < group && where1 >= 0) a.scores[static_cast<size_t>(where1) * g.n_head + kv * group + h] = y;
                    }
                    float v = fmaxf(x, y);
                    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
                    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
                    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
                    const float top = fmaxf(m[nt][i], v);
                    keep[nt][i] = m[nt][i] == -INFINITY ? 0.0f : fast_exp2(m[nt][i] - top);
                    l[nt][i] *= keep[nt][i];
                    m[nt][i] = top;
                }
            }
            float p[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float ref = m[nt][i] == -INFINITY ? 0.0f : m[nt][i];
                    // s qf - ref without the product's rounding (at most 2^-17 here), which a pair's weights then share as
                    // a factor.  With it beyond 128: the factor would set the weights apart from the masses, which come
                    // from rounded scores, and from 2^32 on leave fp32.
                    const bool fused = fabsf(ref) < 128.0f;
                    const float x = s[nt][i], y = s[nt][2 + i], f = qf[nt][i];
                    p[nt][i] = where0 >= 0 ? fast_exp2(fused ? __fmaf_rn(x, f, -ref) : __fsub_rn(__fmul_rn(x, f), ref)) : 0.0f;
                    p[nt][2 + i] = where1 >= 0 ? fast_exp2(fused ? __fmaf_rn(y, f, -ref) : __fsub_rn(__fmul_rn(y, f), ref)) : 0.0f;
                    l[nt][i] += p[nt][i] + p[nt][2 + i];
                    p[nt][i] *= p_scale<T>();
                    p[nt][2 + i] *= p_scale<T>();
                }
            cp_async_wait_group<L::SLOTS - 2>();
            __syncwarp();   // V is there, and all lanes are done with K
            issue(2 * k + L::SLOTS, k_slot);
            // ---- O^T += V^T P^T, the tile's product from zero and then added: the instruction truncates its sums
            // (one accumulator over 131072 positions lost three times the error of everything else)
            auto add = [&](int nt, int i, const float (&x)[4]) {
#pragma unroll
                for (int e = 0; e < 4; ++e) o[nt][i][e] = fmaf(o[nt][i][e], keep[nt][e & 1], x[e]);
            };
            if constexpr (sizeof(T) == 4) {
                uint32_t ph[NT][2][2], pl[NT][2][2];   // [8 positions][k = t4, t4 + 4]
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                        for (int w = 0; w < 2; ++w) {
                            const int src = 4 * (t4 + 4 * w) + (gq >> 1);
                            const float x = __shfl_sync(0xffffffffu, p[nt][2 * kk], src);
                            const float y = __shfl_sync(0xffffffffu, p[nt][2 * kk + 1], src);
                            tf32_round(gq & 1 ? y : x, ph[nt][kk][w], pl[nt][kk][w]);
                        }
#pragma unroll
                for (int b = 0; b < D / 32; ++b)
                {
                    float x[2][NT][4] = {};
#pragma unroll
                    for (int kk = 0; kk < 2; ++kk) {
                        const uint32_t at = vs + (8 * kk + t4) * L::RB + (((8 * b + gq) ^ L::v_swz(t4)) << 4);
                        const float4 r0 = lds_f4(at), r4 = lds_f4(at + 4 * L::RB);
                        uint32_t hi[2][4], lo[2][4];
                        hi[0][0] = tf32_hi(r0.x), lo[0][0] = tf32_lo(r0.x);
                        hi[0][1] = tf32_hi(r0.y), lo[0][1] = tf32_lo(r0.y);
                        hi[0][2] = tf32_hi(r4.x), lo[0][2] = tf32_lo(r4.x);
                        hi[0][3] = tf32_hi(r4.y), lo[0][3] = tf32_lo(r4.y);
                        hi[1][0] = tf32_hi(r0.z), lo[1][0] = tf32_lo(r0.z);
                        hi[1][1] = tf32_hi(r0.w), lo[1][1] = tf32_lo(r0.w);
                        hi[1][2] = tf32_hi(r4.z), lo[1][2] = tf32_lo(r4.z);
                        hi[1][3] = tf32_hi(r4.w), lo[1][3] = tf32_lo(r4.w);
#pragma unroll
                        for (int i = 0; i < 2; ++i)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                mma<T>(x[i][nt], hi[i], ph[nt][kk][0], ph[nt][kk][1]);
                                mma<T>(x[i][nt], hi[i], pl[nt][kk][0], pl[nt][kk][1]);
                                mma<T>(x[i][nt], lo[i], ph[nt][kk][0], ph[nt][kk][1]);
                            }
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) add(nt, 2 * b + i, x[i][nt]);
                }
            } else {
                uint32_t pb[NT][parts<T>()][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int k = 0; k < parts<T>(); ++k) {
                        pb[nt][k][0] = transpose8x8(take_parts2<T>(p[nt][0], p[nt][1]));
                        pb[nt][k][1] = transpose8x8(take_parts2<T>(p[nt][2], p[nt][3]));
                    }
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    uint32_t v[4];
                    ldsm4_t(v, vs + ((lane & 7) + (lane >> 4) * 8) * L::RB + (((2 * i + (lane >> 3 & 1)) ^ L::v_swz(lane)) << 4));
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float x[4] = {};
#pragma unroll
                        for (int k = 0; k < parts<T>(); ++k) mma<T>(x, v, pb[nt][k][0], pb[nt][k][1]);
                        add(nt, i, x);
                    }
                }
            }
        }

        // ---- the next pair's q is on its way while this pair's result is put together
        const int at_seq = seq, at_kv = kv, at_units = units;
        const long long at_seg0 = seg0;
        const bool begins = u == 0, whole = begins && u_end == units;
        seg0 += units + LEAD;
        if (seg0 < end) {
            u = 0;
            if (++kv == hkv) {
                kv = 0;
                do units = units_of(++seq);
                while (units == 0);
            }
            u_end = end_of(seg0, units);
            load_q(seq, kv);
        }

        // ---- the CTA's result for this (sequence, KV head): the slot of the last V holds a warp's output, 8 heads at
        // a time
        auto comb = [&](int w) { return reinterpret_cast<float*>(smem + (w * L::SLOTS + v_slot) * L::HALF); };
        auto swizzled = [&](int h, int d) {   // conflict-free stores of the accumulators' layout
            return h * D + (d ^ ((h >> 1 & 3) * (sizeof(T) == 4 ? 1 : 8)));
        };
        __syncwarp();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float x = l[nt][i];
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                if (gq == 0) s_m[warp][8 * nt + 2 * t4 + i] = m[nt][i], s_l[warp][8 * nt + 2 * t4 + i] = x;
            }
        auto put = [&](const float (&x)[D / 16][4]) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int d = sizeof(T) == 4 ? 32 * (i / 2) + 4 * gq + 2 * (i & 1) + (e >> 1) : 16 * i + gq + 8 * (e >> 1);
                    comb(warp)[swizzled(2 * t4 + (e & 1), d)] = x[i][e];
                }
        };
        put(o[0]);
        __syncthreads();
        float* part = a.part + (2 * static_cast<size_t>(blockIdx.x) + begins) * rec;
        if (tid < group) {   // factors of the warps' outputs
            float top = s_m[0][tid], sum = 0.0f;
#pragma unroll
            for (int w = 1; w < WARPS; ++w) top = fmaxf(top, s_m[w][tid]);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float e = s_m[w][tid] == -INFINITY ? 0.0f : fast_exp2(s_m[w][tid] - top);
                sum = fmaf(s_l[w][tid], e, sum);
                s_m[w][tid] = e;
            }
            if (whole) {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                s_inv[tid] = inv * (1.0f / p_scale<T>());
                if (MASS) a.stats[static_cast<size_t>(at_seq) * g.n_head + at_kv * group + tid] = make_float2(top, inv);
            } else {
                s_inv[tid] = 1.0f;
                part[tid] = top;
                part[PAGED_MAX_GROUP + tid] = sum;
            }
        }
        __syncthreads();
        float* to = whole ? a.out + (static_cast<size_t>(at_seq) * g.n_head + at_kv * group) * D : part + 2 * PAGED_MAX_GROUP;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if (nt) {
                __syncthreads();
                put(o[nt]);
                __syncthreads();
            }
            for (int i = tid; i < min(8, group - 8 * nt) * D; i += THREADS) {
                const int h = i / D, d = i % D;
                float x = 0.0f;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) x = fmaf(comb(w)[swizzled(h, d)], s_m[w][8 * nt + h], x);
                to[8 * nt * D + i] = x * s_inv[8 * nt + h];
            }
        }
        if (!whole) {
            // shares whose (moved) ends lie in this pair
            const int first = shares.of(at_seg0 + LEAD + slack), last = shares.of(at_seg0 + LEAD + at_units - 1 - slack);
            const Shared s{at_seq, at_kv, first, last - first + 1, static_cast<int>(blockIdx.x) - first};
            __syncthreads();
            if (seg0 < end) {   // joined after this CTA's other pairs, so the arrival's round trip is not waited for
                open = s;
                if (tid == 0) open_last = arrive(0, slot_of(s, s.k & ~(FAN - 1)), members_of(s, 0));
            } else {
                if (tid == 0) s_last = arrive(0, slot_of(s, s.k & ~(FAN - 1)), members_of(s, 0));
                __syncthreads();
                join(s);
            }
        }
    }
    if (open.seq >= 0) {
        __syncthreads();
        if (tid == 0) s_last = open_last;
        __syncthreads();
        join(open);
    }
}

// mass[position] += sum over the KV head's query heads of exp(s - max) / sum.  A warp per 32 positions of a KV
// head, VEC heads a load; grid.y sequences.  A weight is known only when its pair's maximum and sum are, so the
// scores wait in the workspace (32 bytes against 512 of fp16 K and V) for this pass.  Bound by its own chain of
// loads (length, page, scores): 7 us at 64 x 2000 positions, which is why a warp gets one tile; adding the mass in
// the CTA that finishes a pair made the chain part of the longest CTA (42 -> 52 us).
constexpr int MASS_WARPS = 8;
template <int VEC>
__global__ void __launch_bounds__(32 * MASS_WARPS) k_paged_mass(const PagedGeom g, const AttArgs a, float* __restrict__ mass) {
    grid_dep_launch();
    grid_dep_wait();
    const int seq = blockIdx.y, n = g.clamp_len(a.len[seq]), hkv = g.n_head_kv, lane = threadIdx.x & 31;
    const int* row = a.table + static_cast<size_t>(seq) * g.max_pages;
    const long long items = static_cast<long long>((n + 31) / 32) * hkv;
    for (long long w = static_cast<long long>(blockIdx.x) * MASS_WARPS + (threadIdx.x >> 5); w < items; w += static_cast<long long>(gridDim.x) * MASS_WARPS) {
        const int tile = static_cast<int>(quotient(w, hkv)), kv = static_cast<int>(w - static_cast<long long>(tile) * hkv);
        const int j = 32 * tile + lane;
        int page, slot;
        if (j >= n || !g.locate(row, j, page, slot)) continue;
        const float* s = a.scores + (static_cast<size_t>(page) * g.page_size + slot) * g.n_head + kv * a.group;
        const float2* st = a.stats + static_cast<size_t>(seq) * g.n_head + kv * a.group;
        float* to = mass + g.mass_at(page, slot, kv);
        const float before = *to;
        float x = 0.0f;
        for (int h = 0; h < a.group; h += VEC) {
            float v[VEC];
            if constexpr (VEC == 4)
                *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(s + h);
            else
                v[0] = s[h];
#pragma unroll
            for (int i = 0; i < VEC; ++i) x = fmaf(fast_exp2(v[i] - st[h + i].x), st[h + i].y, x);
        }
        *to = before + x;
    }
}

constexpr size_t up(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }
constexpr size_t COUNTERS = sizeof(unsigned) * LEVELS * 2 * PAGED_MAX_CTAS;
size_t part_floats(const PagedGeom& g) {
    return 2ull * PAGED_MAX_CTAS * (2 * PAGED_MAX_GROUP + g.n_head / g.n_head_kv * g.head_dim);
}

template <typename T, int D, int NT, bool MASS>
cudaError_t run(const PagedGeom& g, const AttArgs& a, float* mass, int dev, int n_sm, cudaStream_t s) {
    using L = Tile<T, D, NT>;
    auto* kernel = k_paged_attention<T, D, NT, MASS>;
    static bool prepared[64] = {};   // per device: a repeated call sets the same value again
    cudaError_t e;
    if (!prepared[dev]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM);
        if (e != cudaSuccess) return e;
        prepared[dev] = true;
    }
    e = launch_dependent(kernel, dim3(std::min(n_sm * L::CTAS, PAGED_MAX_CTAS)), THREADS, L::SMEM, s, g, a);
    if (e != cudaSuccess || !MASS) return e;
    const long long items = (static_cast<long long>(g.max_pages) * g.page_size + 31) / 32 * g.n_head_kv;
    const long long blocks = std::min<long long>((items + MASS_WARPS - 1) / MASS_WARPS, std::max(1, 16 * n_sm / a.n_seq));
    return launch_dependent(a.group % 4 ? k_paged_mass<1> : k_paged_mass<4>, dim3(static_cast<unsigned>(blocks), a.n_seq), 32 * MASS_WARPS, 0,
                            s, g, a, mass);
}

template <typename T>
cudaError_t pick(const PagedGeom& g, const AttArgs& a, float* mass, int dev, int n_sm, cudaStream_t s) {
    const bool two = a.group > 8;   // heads beside the 8 of one instruction
    if (g.head_dim == 64)
        return mass ? (two ? run<T, 64, 2, true>(g, a, mass, dev, n_sm, s) : run<T, 64, 1, true>(g, a, mass, dev, n_sm, s))
                    : (two ? run<T, 64, 2, false>(g, a, mass, dev, n_sm, s) : run<T, 64, 1, false>(g, a, mass, dev, n_sm, s));
    return mass ? (two ? run<T, 128, 2, true>(g, a, mass, dev, n_sm, s) : run<T, 128, 1, true>(g, a, mass, dev, n_sm, s))
                : (two ? run<T, 128, 2, false>(g, a, mass, dev, n_sm, s) : run<T, 128, 1, false>(g, a, mass, dev, n_sm, s));
}

}  // namespace

size_t paged_attention_workspace(const PagedGeom& g, int max_seqs) {
    return up(COUNTERS) + up(sizeof(float2) * max_seqs * g.n_head) + up(sizeof(float) * part_floats(g)) +
           sizeof(float) * static_cast<size_t>(g.n_pages) * g.page_size * g.n_head;
}

cudaError_t launch_paged_attention(const PagedGeom& g, int kv_type, int max_seqs, const void* kc, const void* vc, float* mass,
                                   const int* table, const int* len, int n_seq, const float* q, long long q_stride, float* out,
                                   float scale, void* ws, cudaStream_t s) {
    int dev = 0, n_sm = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = sm_count(dev, n_sm);
    if (e != cudaSuccess) return e;
    uint8_t* w = static_cast<uint8_t*>(ws);
    AttArgs a{kc, vc, table, len, q, q_stride, out, scale, n_seq, g.n_head / g.n_head_kv};
    a.cnt = reinterpret_cast<unsigned*>(w);
    w += up(COUNTERS);
    a.stats = reinterpret_cast<float2*>(w);
    w += up(sizeof(float2) * max_seqs * g.n_head);
    a.part = reinterpret_cast<float*>(w);
    w += up(sizeof(float) * part_floats(g));
    a.scores = reinterpret_cast<float*>(w);
    if (kv_type == MCPM_KV_F32) return pick<float>(g, a, mass, dev, n_sm, s);
    if (kv_type == MCPM_KV_F16) return pick<__half>(g, a, mass, dev, n_sm, s);
    return pick<__nv_bfloat16>(g, a, mass, dev, n_sm, s);
}

}  // namespace mcpm
