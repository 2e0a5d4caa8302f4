// 8-bit floats with a scale for each block of 128: the quantiser, the matrix
// product, and the sampler on the logits of an 8-bit output head
// (mxs_quantize_fp8, mxs_matmul_fp8, mxs_sample_from_hidden_fp8).
#include <algorithm>
#include <cfloat>

#include <cuda_fp8.h>

#include "mxs_head.cuh"
#include "mxs_launch.h"

namespace {

using mxs::Carve;
using mxs::ceil_div;
using mxs::round_up;
using mxs::to_f32;

constexpr int BLK = 128;
constexpr float FP8_MAX = 448.0f;

__device__ __forceinline__ float block_scale(float top) {
    return top > 0.0f ? fmaxf(top / FP8_MAX, 1.17549435e-38f) : 1.0f;
}
__device__ __forceinline__ uint8_t to_fp8(float x) {
    return (uint8_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float from_fp8(uint8_t x) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(x, __NV_E4M3)));
}

// One CTA of 256 threads per block: its largest finite magnitude, then its values.
template <typename T>
__global__ void __launch_bounds__(256) quantize_kernel(const T* x, int64_t ldx, int64_t rows, int64_t cols,
                                                       int block_rows, uint8_t* q, int64_t ldq, float* scale) {
    __shared__ float s_max[8];
    const int64_t c0 = (int64_t)blockIdx.x * BLK, r0 = (int64_t)blockIdx.y * block_rows;
    const int64_t nr = min((int64_t)block_rows, rows - r0), nc = min((int64_t)BLK, cols - c0);
    float top = 0.0f;
    for (int i = threadIdx.x; i < block_rows * BLK; i += 256) {
        const int r = i / BLK, c = i % BLK;
        if (r < nr && c < nc) {
            const float v = fabsf(to_f32(x[(r0 + r) * ldx + c0 + c]));
            if (v <= FLT_MAX) top = fmaxf(top, v);
        }
    }
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = top;
    __syncthreads();
    for (int w = 0; w < 8; ++w) top = fmaxf(top, s_max[w]);
    const float s = block_scale(top);
    if (threadIdx.x == 0) scale[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = s;
    for (int i = threadIdx.x; i < block_rows * BLK; i += 256) {
        const int r = i / BLK, c = i % BLK;
        if (r < nr && c < nc) q[(r0 + r) * ldq + c0 + c] = to_fp8(to_f32(x[(r0 + r) * ldx + c0 + c]) / s);
    }
}

struct Mat {
    const uint8_t *a, *b;
    int64_t lda, ldb;
    const float *sa, *sb;
    int rows, n, k, kb;
    void* out;
    int64_t ldo;
};

constexpr int TM = 64, TN = 64, TK = 16;

template <typename O>
__global__ void __launch_bounds__(256) matmul_kernel(const Mat p) {
    __shared__ float sa[TK][TM + 4], sb[TK][TN + 4];
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int m0 = blockIdx.y * TM, n0 = blockIdx.x * TN;
    float acc[4][4] = {};
    for (int kb = 0; kb < p.kb; ++kb) {
        float blk[4][4] = {};
        for (int k0 = kb * BLK; k0 < min(p.k, (kb + 1) * BLK); k0 += TK) {
            __syncthreads();
            for (int i = tid; i < TM * TK; i += 256) {
                const int k = i % TK, m = i / TK;
                const bool in = k0 + k < p.k;
                sa[k][m] = in && m0 + m < p.rows ? from_fp8(p.a[(int64_t)(m0 + m) * p.lda + k0 + k]) : 0.0f;
                sb[k][m] = in && n0 + m < p.n ? from_fp8(p.b[(int64_t)(n0 + m) * p.ldb + k0 + k]) : 0.0f;
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < TK; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) blk[i][j] = fmaf(sa[k][ty * 4 + i], sb[k][tx * 4 + j], blk[i][j]);
        }
        const float s1 = p.sb[(int64_t)(n0 / BLK) * p.kb + kb];
        for (int i = 0; i < 4; ++i) {
            const int r = min(p.rows - 1, m0 + ty * 4 + i);
            const float s = p.sa[(int64_t)r * p.kb + kb] * s1;
            for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(blk[i][j], s, acc[i][j]);
        }
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int r = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
            if (r < p.rows && n < p.n) static_cast<O*>(p.out)[(int64_t)r * p.ldo + n] = mxs::from_f32<O>(acc[i][j]);
        }
}

template <typename T>
void launch_quantize(const void* x, int64_t ldx, int64_t rows, int64_t cols, int br, void* q, int64_t ldq, float* scale,
                     cudaStream_t st) {
    const int64_t gy = ceil_div(rows, br);
    // grid rows are limited to 65535: take the rows in runs of whole blocks
    for (int64_t y = 0; y < gy; y += 65535) {
        const int64_t r = y * br;
        quantize_kernel<T><<<dim3((unsigned)ceil_div(cols, BLK), (unsigned)std::min<int64_t>(65535, gy - y)), 256, 0,
                             st>>>(static_cast<const T*>(x) + r * ldx, ldx, rows - r, cols, br,
                                   static_cast<uint8_t*>(q) + r * ldq, ldq, scale + y * ceil_div(cols, BLK));
    }
}

bool bad_type(int t) { return t != MXS_BF16 && t != MXS_F16 && t != MXS_F32; }
constexpr int64_t LIMIT = INT32_MAX - 256;

// Workspace of mxs_sample_from_hidden_fp8.
struct SamplePlan {
    uint8_t* q;
    float* scale;
    float* logits;
    int64_t ldq, ldl;
    void* mm;
    size_t mm_bytes;
    void* sampler;
    size_t sampler_bytes, bytes;
};

int sample_plan(SamplePlan* pl, void* ws, const void* w, int64_t ldw, int64_t rows, int64_t d, int64_t vocab, int top_k,
                bool own_logits) {
    Carve c(ws);
    pl->ldq = round_up(d, 16);
    pl->ldl = round_up(vocab, 4);
    pl->q = c.take<uint8_t>((size_t)rows * pl->ldq);
    pl->scale = c.take<float>((size_t)rows * ceil_div(d, BLK));
    pl->logits = own_logits ? c.take<float>((size_t)rows * pl->ldl) : nullptr;
    // q's base is 256-byte aligned: any aligned address stands for it in the query
    int rc = mxs_matmul_fp8_workspace_size(nullptr, pl->ldq, w, ldw, rows, vocab, d, &pl->mm_bytes);
    if (rc) return rc;
    pl->mm = c.take<uint8_t>(pl->mm_bytes);
    rc = mxs_workspace_size(rows, vocab, top_k, &pl->sampler_bytes);
    if (rc) return rc;
    pl->sampler = c.take<uint8_t>(pl->sampler_bytes);
    pl->bytes = c.used;
    return MXS_OK;
}

}  // namespace

extern "C" {

int mxs_quantize_fp8(const void* d_x, int64_t ld_x, int dtype, int64_t rows, int64_t cols, int block_rows, void* d_q,
                     int64_t ld_q, float* d_scale, void* stream) {
    if (rows < 0 || cols <= 0 || rows > LIMIT || cols > LIMIT || ld_x < cols || ld_q < cols || bad_type(dtype) ||
        (block_rows != 1 && block_rows != BLK))
        return MXS_ERR_INVALID;
    if (rows == 0) return MXS_OK;
    if (!d_x || !d_q || !d_scale) return MXS_ERR_INVALID;
    int sms = 0;
    uint32_t* status = nullptr;
    int rc = mxs::device_info(&sms, &status);
    if (rc) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == MXS_BF16)
        launch_quantize<__nv_bfloat16>(d_x, ld_x, rows, cols, block_rows, d_q, ld_q, d_scale, st);
    else if (dtype == MXS_F16)
        launch_quantize<__half>(d_x, ld_x, rows, cols, block_rows, d_q, ld_q, d_scale, st);
    else
        launch_quantize<float>(d_x, ld_x, rows, cols, block_rows, d_q, ld_q, d_scale, st);
    return cudaGetLastError() == cudaSuccess ? MXS_OK : MXS_ERR_CUDA;
}

int mxs_matmul_fp8_workspace_size(const void* d_a, int64_t ld_a, const void* d_b, int64_t ld_b, int64_t rows,
                                  int64_t n, int64_t k, size_t* bytes) {
    if (!bytes || rows < 0 || n <= 0 || k <= 0 || ld_a < k || ld_b < k || rows > LIMIT || n > LIMIT || k > LIMIT)
        return MXS_ERR_INVALID;
    (void)d_a;
    (void)d_b;
    *bytes = 0;
    return MXS_OK;
}

int mxs_matmul_fp8(const void* d_a, int64_t ld_a, const float* d_a_scale, const void* d_b, int64_t ld_b,
                   const float* d_b_scale, int64_t rows, int64_t n, int64_t k, void* d_out, int64_t ld_out,
                   int out_dtype, void* d_workspace, size_t workspace_bytes, void* stream) {
    if (rows < 0 || n <= 0 || k <= 0 || rows > LIMIT || n > LIMIT || k > LIMIT || ld_a < k || ld_b < k ||
        ld_out < n || bad_type(out_dtype))
        return MXS_ERR_INVALID;
    if (rows == 0) return MXS_OK;
    if (!d_a || !d_a_scale || !d_b || !d_b_scale || !d_out) return MXS_ERR_INVALID;
    (void)d_workspace;
    (void)workspace_bytes;
    int sms = 0;
    uint32_t* status = nullptr;
    int rc = mxs::device_info(&sms, &status);
    if (rc) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    Mat p{static_cast<const uint8_t*>(d_a), static_cast<const uint8_t*>(d_b), ld_a, ld_b, d_a_scale, d_b_scale,
          (int)rows, (int)n, (int)k, (int)ceil_div(k, BLK), d_out, ld_out};
    const dim3 grid((unsigned)ceil_div(n, TN), (unsigned)ceil_div(rows, TM));
    if (out_dtype == MXS_F32)
        matmul_kernel<float><<<grid, 256, 0, st>>>(p);
    else if (out_dtype == MXS_BF16)
        matmul_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(p);
    else
        matmul_kernel<__half><<<grid, 256, 0, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? MXS_OK : MXS_ERR_CUDA;
}

int mxs_sample_from_hidden_fp8_workspace_size(const void* d_weight_q, int64_t ld_weight, int64_t rows, int64_t d_model,
                                              int64_t vocab, int top_k, size_t* bytes) {
    if (!bytes || rows < 0 || d_model <= 0 || vocab <= 0 || ld_weight < d_model || rows > LIMIT || d_model > LIMIT ||
        vocab > LIMIT)
        return MXS_ERR_INVALID;
    SamplePlan pl{};
    const int rc = sample_plan(&pl, nullptr, d_weight_q, ld_weight, rows, d_model, vocab, top_k, true);
    if (rc) return rc;
    *bytes = pl.bytes;
    return MXS_OK;
}

int mxs_sample_from_hidden_fp8(const void* d_hidden, int64_t ld_hidden, int dtype, const void* d_weight_q,
                               int64_t ld_weight, const float* d_weight_scale, int64_t rows, int64_t d_model,
                               int64_t vocab, double temperature, int top_k, double top_p, double min_p,
                               const double* d_u, int32_t* d_next, int32_t* d_topk_idx, double* d_topk_prob,
                               float* d_logits_out, int64_t ld_logits, void* d_workspace, size_t workspace_bytes,
                               void* stream) {
    if (rows < 0 || d_model <= 0 || vocab <= 0 || rows > LIMIT || d_model > LIMIT || vocab > LIMIT ||
        ld_hidden < d_model || ld_weight < d_model || (dtype != MXS_BF16 && dtype != MXS_F16) ||
        (d_logits_out && ld_logits < vocab))
        return MXS_ERR_INVALID;
    if (rows == 0) return MXS_OK;
    if (!d_hidden || !d_weight_q || !d_weight_scale || !d_u || !d_next) return MXS_ERR_INVALID;
    SamplePlan pl{};
    int rc = sample_plan(&pl, d_workspace, d_weight_q, ld_weight, rows, d_model, vocab, top_k, !d_logits_out);
    if (rc) return rc;
    if (!mxs::workspace_ok(d_workspace, workspace_bytes, pl.bytes)) return MXS_ERR_WORKSPACE;
    float* logits = d_logits_out ? d_logits_out : pl.logits;
    const int64_t ldl = d_logits_out ? ld_logits : pl.ldl;
    // the sampler's counters read zero at the start of a call; the per-row ones it clears itself
    size_t zero = 0;
    rc = mxs::workspace_zero_prefix(&zero);
    if (rc) return rc;
    if (cudaMemsetAsync(pl.sampler, 0, std::min(zero, pl.sampler_bytes), (cudaStream_t)stream) != cudaSuccess)
        return MXS_ERR_CUDA;
    rc = mxs_quantize_fp8(d_hidden, ld_hidden, dtype, rows, d_model, 1, pl.q, pl.ldq, pl.scale, stream);
    if (rc) return rc;
    rc = mxs_matmul_fp8(pl.q, pl.ldq, pl.scale, d_weight_q, ld_weight, d_weight_scale, rows, vocab, d_model, logits,
                        ldl, MXS_F32, pl.mm, pl.mm_bytes, stream);
    if (rc) return rc;
    return mxs_sample_topk_ex(logits, rows, vocab, ldl, temperature, top_k, top_p, min_p, d_u, d_next, d_topk_idx,
                              d_topk_prob, nullptr, pl.sampler, pl.sampler_bytes, stream);
}

}  // extern "C"
