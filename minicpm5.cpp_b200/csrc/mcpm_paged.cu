// Paged KV cache: append of new tokens (RoPE, rounding, page writes), attention of one new token
// per sequence over its pages, and eviction of the positions with the least attention mass.
#include <cmath>
#include <cstdio>

#include "../../include/mcpm.h"
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
    int n_seq, items;   // items: float4s of one token's q, k and v rows
};

// One float4 (two rotary pairs) per thread; a token's items are its query heads, its KV heads' K,
// then their V.  (x0, x1) -> (c x0 - s x1, s x0 + c x1), one fma per output as mcpm_rope_kv_append.
template <typename T>
__global__ void k_paged_append(const PagedGeom g, const AppendArgs a) {
    const size_t i = blockIdx.x;
    const int item = blockIdx.y * blockDim.x + threadIdx.x;
    if (item >= a.items) return;
    const int per_head = g.head_dim / 4, nq = a.t.q ? g.n_head * per_head : 0, nk = g.n_head_kv * per_head;
    const int tok_slot = a.t.tok_slot[i];
    const bool is_q = item < nq, is_v = item >= nq + nk;
    const int x = is_q ? item : is_v ? item - nq - nk : item - nq;   // float4 within its row
    const float* src = is_q ? a.t.q + i * a.t.q_stride : (is_v ? a.t.v : a.t.k) + i * a.t.kv_stride;
    float4 v = reinterpret_cast<const float4*>(src)[x];
    if (a.t.rope && !is_v) {
        const int pos = min(max(a.t.tok_pos ? a.t.tok_pos[i] : tok_slot, 0), a.t.rope_len - 1);
        const float4 cs = reinterpret_cast<const float4*>(a.t.rope)[static_cast<size_t>(pos) * per_head + x % per_head];
        v = make_float4(__fmaf_rn(cs.x, v.x, -__fmul_rn(cs.y, v.y)), __fmaf_rn(cs.y, v.x, __fmul_rn(cs.x, v.y)),
                        __fmaf_rn(cs.z, v.z, -__fmul_rn(cs.w, v.w)), __fmaf_rn(cs.w, v.z, __fmul_rn(cs.z, v.w)));
    }
    if (is_q) {
        reinterpret_cast<float4*>(a.t.q_out + i * g.n_head * g.head_dim)[x] = v;
        return;
    }
    const int seq = a.t.tok_seq ? a.t.tok_seq[i] : static_cast<int>(i);
    if (seq < 0 || seq >= a.n_seq || tok_slot < 0 || tok_slot >= g.max_pages * g.page_size) return;
    int page, slot;
    if (!g.locate(a.table + static_cast<size_t>(seq) * g.max_pages, tok_slot, page, slot)) return;
    const int head = x / per_head;
    kv_store4(static_cast<T*>(is_v ? a.vc : a.kc) + g.row(page, slot, head) + 4 * (x % per_head), v);
    if (!is_v && x % per_head == 0 && a.mass) a.mass[g.mass_at(page, slot, head)] = 0.0f;
}

// ---------------------------------------------------------------- eviction
struct EvictArgs {
    void *kc, *vc;
    float* mass;
    const int *table, *len, *dst;
    int *new_len, *kept;
    int n_keep, n_sink, n_recent;
};

constexpr int EV_THREADS = 1024;

// Order-preserving unsigned key of a position: a larger key is kept first.  NaN 0 (lightest), then the
// floats in order (-0 and +0 alike), then the protected positions.
__device__ __forceinline__ uint32_t mass_key(float m) {
    if (m != m) return 0u;
    const uint32_t u = __float_as_uint(m + 0.0f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// One CTA per (KV head, sequence): radix selection of the n_keep-th largest key, 8 bits a pass, then
// the kept positions in order.
__global__ void __launch_bounds__(EV_THREADS, 1) k_paged_evict_select(const PagedGeom g, const EvictArgs a) {
    __shared__ int hist[256], warp_gt[32], warp_eq[32], pick[2];
    const int kv = blockIdx.x, seq = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n = g.clamp_len(a.len[seq]);
    const int* row = a.table + static_cast<size_t>(seq) * g.max_pages;
    int* kept = a.kept + (static_cast<size_t>(seq) * g.n_head_kv + kv) * a.n_keep;
    auto key_of = [&](int j, bool& present) -> uint32_t {
        int page, slot;
        present = g.locate(row, j, page, slot);
        if (!present) return 0u;
        if (j < a.n_sink || j >= n - a.n_recent) return 0xffffffffu;
        return mass_key(a.mass[g.mass_at(page, slot, kv)]);
    };
    // threshold key and how many positions with exactly that key are kept; a length within the budget
    // keeps every present position (threshold 0, no limit)
    uint32_t prefix = 0u;
    int need = a.n_keep, total = 0;
    for (int sh = 24; sh >= 0; sh -= 8) {
        for (int i = tid; i < 256; i += EV_THREADS) hist[i] = 0;
        __syncthreads();
        for (int j = tid; j < n; j += EV_THREADS) {
            bool present;
            const uint32_t k = key_of(j, present);
            if (present && (sh == 24 || (k >> (sh + 8)) == (prefix >> (sh + 8)))) atomicAdd(&hist[(k >> sh) & 255], 1);
        }
        __syncthreads();
        if (tid == 0) {
            int above = 0, b = 255;
            for (; b > 0 && above + hist[b] < need; --b) above += hist[b];
            pick[0] = b;
            pick[1] = above;
            if (sh == 24)
                for (int i = 0; i < 256; ++i) total += hist[i];
        }
        __syncthreads();
        prefix |= static_cast<uint32_t>(pick[0]) << sh;
        need -= pick[1];
        __syncthreads();
    }
    if (tid == 0) pick[0] = total;
    __syncthreads();
    total = pick[0];
    int at = 0, eq_seen = 0;   // kept so far, threshold-equal positions seen so far
    for (int j0 = 0; j0 < n; j0 += EV_THREADS) {
        const int j = j0 + tid;
        bool present = false;
        const uint32_t k = j < n ? key_of(j, present) : 0u;
        const bool gt = present && k > prefix, eq = present && k == prefix;
        const unsigned mg = __ballot_sync(0xffffffffu, gt), me = __ballot_sync(0xffffffffu, eq);
        if (lane == 0) warp_gt[warp] = __popc(mg), warp_eq[warp] = __popc(me);
        __syncthreads();
        int gt_before = 0, eq_before = 0, gt_all = 0, eq_all = 0;
        for (int w = 0; w < 32; ++w) {
            if (w < warp) gt_before += warp_gt[w], eq_before += warp_eq[w];
            gt_all += warp_gt[w], eq_all += warp_eq[w];
        }
        const unsigned below = (1u << lane) - 1u;
        gt_before += __popc(mg & below);
        eq_before += __popc(me & below);
        const int eq_rank = eq_seen + eq_before;
        const int place = at + gt_before + (min(eq_rank, need) - min(eq_seen, need));
        if (gt || (eq && eq_rank < need)) kept[place] = j;
        at += gt_all + min(eq_seen + eq_all, need) - min(eq_seen, need);
        eq_seen += eq_all;
        __syncthreads();
    }
    for (int i = at + tid; i < a.n_keep; i += EV_THREADS) kept[i] = -1;
    if (tid == 0 && kv == 0) a.new_len[seq] = at;
}

// A warp per kept row: K, V (16 bytes a lane) and the mass.
template <typename T>
__global__ void k_paged_evict_copy(const PagedGeom g, const EvictArgs a) {
    const int i = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5), kv = blockIdx.y, seq = blockIdx.z;
    const int lane = threadIdx.x & 31;
    if (i >= a.n_keep) return;
    const int j = a.kept[(static_cast<size_t>(seq) * g.n_head_kv + kv) * a.n_keep + i];
    if (j < 0) return;
    int sp, ss, dp, ds;
    if (!g.locate(a.table + static_cast<size_t>(seq) * g.max_pages, j, sp, ss)) return;
    if (!g.locate(a.dst + static_cast<size_t>(seq) * g.max_pages, i, dp, ds)) return;
    const long long so = g.row(sp, ss, kv), to = g.row(dp, ds, kv);
    T *kc = static_cast<T*>(a.kc), *vc = static_cast<T*>(a.vc);
    const int chunks = g.head_dim * static_cast<int>(sizeof(T)) / 16;
    for (int c = lane; c < chunks; c += 32) {
        reinterpret_cast<uint4*>(kc + to)[c] = reinterpret_cast<const uint4*>(kc + so)[c];
        reinterpret_cast<uint4*>(vc + to)[c] = reinterpret_cast<const uint4*>(vc + so)[c];
    }
    if (lane == 0) a.mass[g.mass_at(dp, ds, kv)] = a.mass[g.mass_at(sp, ss, kv)];
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
    AppendArgs a{*tokens, table, pool->k, pool->v, pool->mass, n_seq, 0};
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
    a.items = ((t.q ? g.n_head : 0) + 2 * g.n_head_kv) * g.head_dim / 4;
    const dim3 grid(t.n_tok, (a.items + 127) / 128);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (cfg->kv_type == MCPM_KV_F32)
        k_paged_append<float><<<grid, 128, 0, s>>>(g, a);
    else if (cfg->kv_type == MCPM_KV_F16)
        k_paged_append<__half><<<grid, 128, 0, s>>>(g, a);
    else
        k_paged_append<__nv_bfloat16><<<grid, 128, 0, s>>>(g, a);
    return status("mcpm_paged_append", cudaGetLastError());
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
    k_paged_evict_select<<<dim3(g.n_head_kv, n_seq), EV_THREADS, 0, s>>>(g, a);
    const dim3 grid((n_keep + 3) / 4, g.n_head_kv, n_seq);
    if (cfg->kv_type == MCPM_KV_F32)
        k_paged_evict_copy<float><<<grid, 128, 0, s>>>(g, a);
    else if (cfg->kv_type == MCPM_KV_F16)
        k_paged_evict_copy<__half><<<grid, 128, 0, s>>>(g, a);
    else
        k_paged_evict_copy<__nv_bfloat16><<<grid, 128, 0, s>>>(g, a);
    return status("mcpm_paged_evict", cudaGetLastError());
}

}  // extern "C"
