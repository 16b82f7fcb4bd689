// Geometry of a paged KV pool as the kernels of mcpm_paged.cu and mcpm_paged_attention.cu see it: which element row a
// position of a sequence lies in, with page ids and positions from device memory that are
// checked before anything is addressed through them.
#pragma once
#include <cstddef>
#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace mcpm {

constexpr int PAGED_MAX_GROUP = 16;   // query heads per KV head

// Unsigned division by a divisor fixed at launch (Granlund and Montgomery, "Division by invariant
// integers using multiplication"): exact for numerators below 2^31, where the sum does not carry.
struct FastDiv {
    uint32_t mul, shift;
    void set(uint32_t d) {
        shift = 0;
        while ((1ull << shift) < d) ++shift;
        mul = static_cast<uint32_t>(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
};

struct PagedGeom {
    int n_head, n_head_kv, head_dim, page_size, n_pages, max_pages;
    long long page_stride, row_stride, head_stride;   // elements
    FastDiv by_page;

    __device__ __forceinline__ int clamp_len(int n) const {   // max_pages * page_size <= 2^30 (host check)
        return min(max(n, 0), max_pages * page_size);
    }
    // Page and slot of position j, 0 <= j < max_pages * page_size; false: the page is absent.
    __device__ __forceinline__ bool locate(const int* __restrict__ table_row, int j, int& page, int& slot) const {
        const int c = static_cast<int>(by_page.div(static_cast<uint32_t>(j)));
        slot = j - c * page_size;
        page = __ldg(table_row + c);
        return static_cast<unsigned>(page) < static_cast<unsigned>(n_pages);
    }
    __device__ __forceinline__ long long row(int page, int slot, int head) const {
        return page * page_stride + slot * row_stride + head * head_stride;
    }
    __device__ __forceinline__ size_t mass_at(int page, int slot, int head) const {   // [page][kv head][slot]
        return (static_cast<size_t>(page) * n_head_kv + head) * page_size + slot;
    }
};

// Attention (mcpm_paged_attention.cu).
constexpr int PAGED_MAX_CTAS = 480;   // most CTAs of a launch: sizes the workspace's partial results
size_t paged_attention_workspace(const PagedGeom& g, int max_seqs);
cudaError_t launch_paged_attention(const PagedGeom& g, int kv_type, int max_seqs, const void* kc, const void* vc, float* mass,
                                   const int* table, const int* len, int n_seq, const float* q, long long q_stride, float* out,
                                   float scale, void* ws, cudaStream_t s);

// Four values rounded to the cache type (nearest, ties to even: the engine's own rounding of an
// fp16 cache) in one store.
__device__ __forceinline__ void kv_store4(float* p, float4 x) { *reinterpret_cast<float4*>(p) = x; }
__device__ __forceinline__ void kv_store4(__half* p, float4 x) {
    __half2 h[2] = {__floats2half2_rn(x.x, x.y), __floats2half2_rn(x.z, x.w)};
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(h);
}
__device__ __forceinline__ void kv_store4(__nv_bfloat16* p, float4 x) {
    __nv_bfloat162 h[2] = {__floats2bfloat162_rn(x.x, x.y), __floats2bfloat162_rn(x.z, x.w)};
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(h);
}

// SMs of a device, asked for once.
inline cudaError_t sm_count(int dev, int& n) {
    static int known[64] = {};
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!known[dev]) {
        int x = 0;
        const cudaError_t e = cudaDeviceGetAttribute(&x, cudaDevAttrMultiProcessorCount, dev);
        if (e != cudaSuccess) return e;
        known[dev] = x;
    }
    n = known[dev];
    return cudaSuccess;
}
// Clusters of `width` CTAs of a kernel that can run at once; -1: the device does not take such a launch.
template <typename... P>
int active_clusters(void (*kernel)(P...), int width, int threads, size_t smem) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(width);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = width;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) == cudaSuccess) return n;
    cudaGetLastError();   // an answer, not a fault of the call that asked
    return -1;
}

// Launches a kernel that may begin while the one before it in the stream ends (programmatic dependent launch).
// The kernel calls grid_dep_wait in every CTA before it touches memory that the kernel before it may write, so streams
// keep their order; what overlaps is the launch itself, 1 to 2 us of a call of 5 to 10 us.  (One kernel reads before
// its wait: the eviction's copy, a table that was final before the selection in front of it began.)
template <typename... P, typename... A>
cudaError_t launch_dependent(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t s, const A&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

}  // namespace mcpm
