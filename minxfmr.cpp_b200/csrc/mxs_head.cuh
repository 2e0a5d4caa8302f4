// Shared by the output-head operators (mxs_ce.cu, mxs_fp8.cu): element types,
// workspace carving, and the copy of rows that do not start on 16-byte
// boundaries.
#pragma once
#include <cstddef>
#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/mxs_head.h"

namespace mxs {

__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(float x) { return x; }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }

// Sixteen bytes of values, rounded to their type.
template <typename T>
__device__ __forceinline__ uint4 pack16(const float* v);
template <>
__device__ __forceinline__ uint4 pack16<__nv_bfloat16>(const float* v) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&p);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <>
__device__ __forceinline__ uint4 pack16<__half>(const float* v) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 p = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&p);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <>
__device__ __forceinline__ uint4 pack16<float>(const float* v) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}

inline int64_t round_up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }
__host__ __device__ constexpr int64_t ceil_div(int64_t x, int64_t a) { return (x + a - 1) / a; }

// Hands out 256-byte aligned parts of a workspace (or only counts, from a null base).
struct Carve {
    char* base;
    size_t used = 0;
    explicit Carve(void* p) : base(static_cast<char*>(p)) {}
    template <typename T>
    T* take(size_t n) {
        T* p = base ? reinterpret_cast<T*>(base + used) : nullptr;
        used += (n * sizeof(T) + 255) / 256 * 256;
        return p;
    }
};

inline bool aligned16(const void* p, int64_t row_bytes) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && row_bytes % 16 == 0;
}
inline bool workspace_ok(const void* ws, size_t bytes, size_t need) {
    return need == 0 || (ws && reinterpret_cast<uintptr_t>(ws) % 256 == 0 && bytes >= need);
}

// Rows of `row_bytes` bytes into aligned rows of ld_to bytes, a warp each.
__global__ void copy_rows_kernel(const uint8_t* from, int64_t ld_from, uint8_t* to, int64_t ld_to, int64_t rows,
                                 int64_t row_bytes);
cudaError_t copy_rows(const void* from, int64_t ld_from, void* to, int64_t ld_to, int64_t rows, int64_t row_bytes,
                      int sms, cudaStream_t st);

// Tile width for `n` columns: the multiple of `step` in [lo, 256] whose
// rounds of tiles over the units cost least, a round costing its width and a
// fixed part (filling and draining a tile's pipeline, worth about 16 columns).
int tile_width(int64_t m_tiles, int64_t n, int units, int lo, int step);

}  // namespace mxs
