// The 4-bit paged cache: what its kernels (kv4_rows.cu, attention_kv4.cu) share.
//
// Pool: uint8 [block][layer][kv head][K, V][16 slots][80]. A row (one token, one kv head, keys or values) is 64 bytes of codes, dim d
// in nibble d % 2 of byte d / 2 (the low one first), and four pairs (scale, minimum) of fp16 for the dims 32g .. 32g + 31; a value
// is minimum + scale * code. Rows of 80 bytes are what makes the attention kernel's shared memory free of bank conflicts
// without a swizzle: 20 words apart, eight consecutive rows start at eight different multiples of four banks. And a page of one
// head, keys and values, is 2560 contiguous bytes: one bulk copy.
#pragma once
#include "common.cuh"
#include "../../include/tenzo_kernels.h"

namespace tz {

constexpr int kK4Slots = 16, kK4Row = 80, kK4Codes = 64;
constexpr int kK4Half = kK4Slots * kK4Row;              // the keys of a page, or its values
constexpr int kK4Page = 2 * kK4Half;

constexpr int kK4ErrWait = 1, kK4ErrIndex = 2;          // bits of the error flags

// Byte offset of the page of `kvh` in block `block`.
__device__ __forceinline__ size_t kv4_page(const tenzo_kv4_cache& c, int layer, int kvh, int block) {
    return (((size_t)block * c.n_layers + layer) * c.n_kv + kvh) * kK4Page;
}

// Loads of what the kernel in front may have written, from L2. They are volatile so that none moves in front of the wait for that kernel: the
// compiler may hoist a load through a const __restrict__ pointer, an __ldg or an __ldcg above it (a table of parents was read early that way, once in some
// hundred launches).
__device__ __forceinline__ int ld_l2(const int* p) { int v; asm volatile("ld.global.cg.b32 %0, [%1];" : "=r"(v) : "l"(p)); return v; }
__device__ __forceinline__ uint32_t ld_l2(const uint32_t* p) { uint32_t v; asm volatile("ld.global.cg.b32 %0, [%1];" : "=r"(v) : "l"(p)); return v; }
__device__ __forceinline__ uint32_t ld_l2(const unsigned short* p) { unsigned short v; asm volatile("ld.global.cg.u16 %0, [%1];" : "=h"(v) : "l"(p)); return v; }
__device__ __forceinline__ float ld_l2(const float* p) { float v; asm volatile("ld.global.cg.f32 %0, [%1];" : "=f"(v) : "l"(p)); return v; }
__device__ __forceinline__ double ld_l2(const double* p) { double v; asm volatile("ld.global.cg.f64 %0, [%1];" : "=d"(v) : "l"(p)); return v; }
__device__ __forceinline__ unsigned long long ld_l2(const unsigned long long* p) { unsigned long long v; asm volatile("ld.global.cg.b64 %0, [%1];" : "=l"(v) : "l"(p)); return v; }
__device__ __forceinline__ float2 ld_l2(const float2* p) { float2 v; asm volatile("ld.global.cg.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "l"(p)); return v; }
__device__ __forceinline__ float4 ld_l2(const float4* p) {
    float4 v;
    asm volatile("ld.global.cg.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint4 ld_l2(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.cg.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

inline bool kv4_cache_ok(const tenzo_kv4_cache& c) {
    return c.pool && c.block_table && !(reinterpret_cast<uintptr_t>(c.pool) & 15) && c.n_blocks > 0 && c.n_layers > 0 && c.n_kv > 0 && c.table_rows > 0 &&
           c.table_stride > 0;
}

// Launch in clusters of `cluster` blocks along x, with (or without) the attribute that lets the kernel become resident while its predecessor drains.
template <typename... KArgs, typename... Args>
inline int kv4_launch_cluster(void (*kernel)(KArgs...), dim3 grid, int threads, int cluster, size_t smem, cudaStream_t st, bool pdl, Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    unsigned n = 0;
    if (pdl) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = (unsigned)cluster;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    return (int)cudaLaunchKernelEx(&cfg, kernel, args...);
}
template <typename... KArgs, typename... Args>
inline int kv4_launch(void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, cudaStream_t st, bool pdl, Args&&... args) {
    return kv4_launch_cluster(kernel, grid, threads, 1, smem, st, pdl, args...);
}

}  // namespace tz
