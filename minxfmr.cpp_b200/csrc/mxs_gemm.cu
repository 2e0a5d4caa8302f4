// Host side of the tensor-core frame: tensor maps.
#include <algorithm>

#include "mxs_gemm.cuh"
#include "mxs_head.cuh"

namespace mxs {

// Sixteen aligned bytes at a time, put together from the two aligned 8-byte
// words on either side of the source (rows may start anywhere); a row's last
// bytes one by one.
__global__ void __launch_bounds__(256) copy_rows_kernel(const uint8_t* from, int64_t ld_from, uint8_t* to,
                                                        int64_t ld_to, int64_t rows, int64_t row_bytes) {
    const int lane = threadIdx.x & 31;
    const int64_t warps = (int64_t)gridDim.x * 8;
    for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += warps) {
        const uint8_t* src = from + r * ld_from;
        uint8_t* dst = to + r * ld_to;
        const int shift = (int)(reinterpret_cast<uintptr_t>(src) & 7) * 8;
        const uint64_t* w = reinterpret_cast<const uint64_t*>(src - shift / 8);
        // words are read whole only where all 24 bytes lie in the row
        const int64_t whole = row_bytes >= 24 ? (row_bytes - 8) / 16 : 0;
        for (int64_t i = lane; i < whole; i += 32) {
            uint64_t a, b;
            if (shift == 0) {
                a = w[2 * i], b = w[2 * i + 1];
            } else if (i > 0) {
                const uint64_t x = w[2 * i], y = w[2 * i + 1], z = w[2 * i + 2];
                a = x >> shift | y << (64 - shift);
                b = y >> shift | z << (64 - shift);
            } else {  // the first word begins before the row
                a = b = 0;
                for (int j = 0; j < 8; ++j) {
                    a |= (uint64_t)src[j] << (8 * j);
                    b |= (uint64_t)src[8 + j] << (8 * j);
                }
            }
            *reinterpret_cast<ulonglong2*>(dst + 16 * i) = make_ulonglong2(a, b);
        }
        for (int64_t i = whole * 16 + lane; i < row_bytes; i += 32) dst[i] = src[i];
    }
}

cudaError_t copy_rows(const void* from, int64_t ld_from, void* to, int64_t ld_to, int64_t rows, int64_t row_bytes,
                      int sms, cudaStream_t st) {
    const int grid = (int)std::min<int64_t>(ceil_div(rows, 8), (int64_t)sms * 8);
    copy_rows_kernel<<<grid, 256, 0, st>>>(static_cast<const uint8_t*>(from), ld_from, static_cast<uint8_t*>(to), ld_to,
                                           rows, row_bytes);
    return cudaGetLastError();
}

int tile_width(int64_t m_tiles, int64_t n, int units, int lo, int step) {
    int best = 256;
    double best_cost = 1e30;
    for (int w = 256; w >= lo; w -= step) {
        const double cost = (double)ceil_div(m_tiles * ceil_div(n, w), units) * (w + 16);
        if (cost < best_cost) best_cost = cost, best = w;
    }
    return best;
}

namespace gemm {

namespace {
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's encoder, looked up once (the library does not link the driver).
EncodeFn encoder() {
    static const EncodeFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) !=
                cudaSuccess || found != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeFn>(p);
    }();
    return fn;
}
}  // namespace

bool make_map(CUtensorMap* map, const void* base, int elem_bytes, int64_t cols, int64_t rows, int64_t ld,
              int box_rows) {
    const EncodeFn fn = encoder();
    if (!fn) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)(ld * elem_bytes)};
    const cuuint32_t box[2] = {(cuuint32_t)(ROW / elem_bytes), (cuuint32_t)box_rows};
    const cuuint32_t steps[2] = {1, 1};
    return fn(map, elem_bytes == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2,
              const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace gemm
}  // namespace mxs
