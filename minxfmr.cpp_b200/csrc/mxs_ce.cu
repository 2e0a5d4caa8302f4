// Softmax cross entropy over the vocabulary from hidden states, and its
// gradients (mxs_ce_from_hidden, mxs_ce_from_hidden_backward).
//
// With s = log2(e) / temperature and y_v = s <h, w_v> (logits in units of ln 2),
// a vocabulary tile gives each row the largest y of the tile and
// sum 2^(y - largest) over its entries other than the target; the tiles' pairs
// join into the others' log-sum o, and with the target's y_t kept apart
//   loss = ln(1 + 2^(o - y_t)),   lse = ln 2 * y_t + loss.
// Keeping the target out of the sum is what holds the loss to fp32 accuracy
// where the target's probability is near 1 (lse - logit would cancel there).
//
// Backward, for a piece of the vocabulary at a time: the logits again,
//   G[r][v] = ghat_r (2^(y_v - lse_r log2 e) - (v == t_r)),   ghat = grad / max |grad|,
// held in the operands' type, then grad_hidden += G W and grad_weight = G^T H,
// each times max|grad| / temperature once, in fp32, at the end. Dividing by
// max |grad| keeps a batch mean's 1/rows out of G: the target's entry is then
// near -1, which both types hold with no error common to a whole row.
//
// Rows whose target is out of range are packed away first (pack_rows_kernel), so
// they cost no products; every later kernel reads the number of rows left from
// device memory.
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "mxs_head.cuh"
#include "mxs_launch.h"

namespace {

using mxs::Carve;
using mxs::ceil_div;
using mxs::round_up;
using mxs::to_f32;

constexpr float LN2 = 0.693147180559945309f;
constexpr double LOG2E = 1.4426950408889634074;

struct Head {
    int kept;      // rows with a target in range
    float gmax;    // largest finite |grad_loss| of those rows (1 if none)
};

struct Pack {
    const void* hidden;
    int64_t ld_hidden;
    const void* targets;
    int target_bytes;
    int rows, d, ldk;
    int64_t vocab;
    const float* lse;   // backward: null in forward
    const float* grad;
    Head* head;
    void* packed;       // [rows_pad][ldk]
    int* pos;           // [rows]: packed row or -1
    int* target;        // [packed]
    float* lse2;        // [packed] lse * log2(e)
    float* ghat;        // [packed] grad / gmax
};

__device__ __forceinline__ int64_t target_of(const Pack& p, int64_t r) {
    return p.target_bytes == 8 ? static_cast<const int64_t*>(p.targets)[r]
                               : (int64_t)static_cast<const int32_t*>(p.targets)[r];
}
__device__ __forceinline__ bool kept_row(const Pack& p, int64_t r) {
    const int64_t t = target_of(p, r);
    return t >= 0 && t < p.vocab;
}

constexpr int PACK_T = 256;
constexpr int PACK_TAIL = 256;  // rows after the last kept one that read zero

// Each CTA packs a contiguous range of rows; it counts the kept rows before its
// range itself (a few KB of targets from L2), so one launch does it all.
template <typename T>
__global__ void __launch_bounds__(PACK_T) pack_rows_kernel(const Pack p) {
    __shared__ int s_cnt[PACK_T / 32];
    __shared__ float s_max[PACK_T / 32];
    __shared__ int s_base;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (int)ceil_div(p.rows, gridDim.x);
    const int r0 = min(p.rows, (int)blockIdx.x * per), r1 = min(p.rows, r0 + per);
    int n = 0;
    float gm = 0.0f;
    const int scan_to = p.grad ? p.rows : r0;
    for (int r = tid; r < scan_to; r += PACK_T) {
        if (!kept_row(p, r)) continue;
        if (r < r0) ++n;
        if (p.grad) {
            const float g = fabsf(p.grad[r]);
            if (g <= FLT_MAX) gm = fmaxf(gm, g);
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        n += __shfl_xor_sync(0xffffffffu, n, o);
        gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, o));
    }
    if (lane == 0) {
        s_cnt[warp] = n;
        s_max[warp] = gm;
    }
    __syncthreads();
    n = 0;
    gm = 0.0f;
    for (int w = 0; w < PACK_T / 32; ++w) {
        n += s_cnt[w];
        gm = fmaxf(gm, s_max[w]);
    }
    if (!(gm > 0.0f)) gm = 1.0f;
    int base = n;
    const int step = 16 / sizeof(T);
    const bool vec = reinterpret_cast<uintptr_t>(p.hidden) % 16 == 0 && p.ld_hidden % step == 0;
    for (int c0 = r0; c0 < r1; c0 += PACK_T) {
        __syncthreads();
        const int r = c0 + tid;
        const bool keep = r < r1 && kept_row(p, r);
        const uint32_t b = __ballot_sync(0xffffffffu, keep);
        if (lane == 0) s_cnt[warp] = __popc(b);
        __syncthreads();
        int at = base + __popc(b & ((1u << lane) - 1));
        int all = 0;
        for (int w = 0; w < PACK_T / 32; ++w) {
            if (w < warp) at += s_cnt[w];
            all += s_cnt[w];
        }
        if (r < r1) p.pos[r] = keep ? at : -1;
        if (keep) {
            p.target[at] = (int)target_of(p, r);
            if (p.grad) {
                p.lse2[at] = p.lse[r] * (float)LOG2E;
                p.ghat[at] = p.grad[r] / gm;
            }
        }
        base += all;
        // the rows themselves: a warp each, positions recomputed from the ballots' order
        __syncthreads();
        for (int i = warp; i < min(PACK_T, r1 - c0); i += PACK_T / 32) {
            const int to = p.pos[c0 + i];
            if (to < 0) continue;
            const T* src = static_cast<const T*>(p.hidden) + (int64_t)(c0 + i) * p.ld_hidden;
            T* dst = static_cast<T*>(p.packed) + (int64_t)to * p.ldk;
            int k = 0;
            if (vec) {
                for (k = lane * step; k + step <= p.d; k += 32 * step)
                    *reinterpret_cast<uint4*>(dst + k) = *reinterpret_cast<const uint4*>(src + k);
                k = p.d / step * step;
            }
            for (k += lane; k < p.d; k += 32) dst[k] = src[k];
        }
    }
    if (r1 == p.rows && r0 < r1) {  // the range that ends the rows knows how many were kept
        if (tid == 0) {
            p.head->kept = base;
            p.head->gmax = gm;
        }
        const int end = (int)((base + (int64_t)PACK_TAIL - 1) / PACK_TAIL * PACK_TAIL);
        for (int64_t i = tid; i < (int64_t)(end - base) * p.ldk; i += PACK_T)
            static_cast<T*>(p.packed)[(int64_t)base * p.ldk + i] = mxs::from_f32<T>(0.0f);
    }
    (void)s_base;
}

// ---------------------------------------------------------------------------
// Products: 64 x 64 tiles in fp32 through shared memory.
// ---------------------------------------------------------------------------
constexpr int TM = 64, TN = 64, TK = 16;

template <typename LA, typename LB>
__device__ __forceinline__ void tile_product(float (&acc)[4][4], int K, LA la, LB lb) {
    __shared__ float sa[TK][TM + 4], sb[TK][TN + 4];
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    for (int k0 = 0; k0 < K; k0 += TK) {
        __syncthreads();
        for (int i = tid; i < TM * TK; i += 256) {
            const int k = i % TK, m = i / TK;
            sa[k][m] = k0 + k < K ? la(m, k0 + k) : 0.0f;
            sb[k][m] = k0 + k < K ? lb(m, k0 + k) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < TK; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[k][ty * 4 + i], sb[k][tx * 4 + j], acc[i][j]);
    }
}

struct Score {
    const void* h;   // packed rows
    const void* w;
    int64_t ldw;
    int d, ldk, vocab;
    float c;         // log2(e) / temperature
    const Head* head;
    const int* target;
    float2* part;    // [tile][rows]: largest y of the others, sum 2^(y - largest)
    float* ytarget;  // [rows]
    int rows;
};

template <typename T>
__global__ void __launch_bounds__(256) score_kernel(const Score p) {
    const int kept = p.head->kept;
    const int m0 = blockIdx.y * TM, v0 = blockIdx.x * TN;
    if (m0 >= kept) return;
    float acc[4][4] = {};
    const T *h = static_cast<const T*>(p.h), *w = static_cast<const T*>(p.w);
    tile_product(acc, p.d,
                 [&](int m, int k) { return m0 + m < kept ? to_f32(h[(int64_t)(m0 + m) * p.ldk + k]) : 0.0f; },
                 [&](int n, int k) { return v0 + n < p.vocab ? to_f32(w[(int64_t)(v0 + n) * p.ldw + k]) : 0.0f; });
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    for (int i = 0; i < 4; ++i) {
        const int r = m0 + ty * 4 + i;
        const int t = r < kept ? p.target[r] : -1;
        float m = -INFINITY, s = 0.0f;
        for (int j = 0; j < 4; ++j) {
            const int v = v0 + tx * 4 + j;
            acc[i][j] *= p.c;
            if (v == t) p.ytarget[r] = acc[i][j];
            if (v < p.vocab && v != t) m = fmaxf(m, acc[i][j]);
        }
        for (int o = 8; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float sub = m == -INFINITY ? 0.0f : m;
        for (int j = 0; j < 4; ++j) {
            const int v = v0 + tx * 4 + j;
            if (v < p.vocab && v != t) s += exp2f(acc[i][j] - sub);
        }
        for (int o = 8; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (tx == 0 && r < kept) p.part[(int64_t)blockIdx.x * p.rows + r] = make_float2(m, s);
    }
}

// One warp per row joins the tiles' pairs, in the same order every time.
__global__ void __launch_bounds__(256) score_join_kernel(const float2* part, const float* ytarget, const int* pos,
                                                         int rows, int tiles, float* loss, float* lse) {
    const int lane = threadIdx.x & 31;
    const int r = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (r >= rows) return;
    const int at = pos[r];
    if (at < 0) {
        if (lane == 0) {
            if (loss) loss[r] = 0.0f;
            if (lse) lse[r] = 0.0f;
        }
        return;
    }
    float m = -INFINITY, s = 0.0f;
    for (int i = lane; i < tiles; i += 32) {
        const float2 q = part[(int64_t)i * rows + at];
        const float nm = fmaxf(m, q.x), sub = nm == -INFINITY ? 0.0f : nm;
        s = s * exp2f(m - sub) + q.y * exp2f(q.x - sub);
        m = nm;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const float om = __shfl_xor_sync(0xffffffffu, m, o), os = __shfl_xor_sync(0xffffffffu, s, o);
        const float nm = fmaxf(m, om), sub = nm == -INFINITY ? 0.0f : nm;
        s = s * exp2f(m - sub) + os * exp2f(om - sub);
        m = nm;
    }
    if (lane == 0) {
        const float y = ytarget[at];
        const float diff = (m + log2f(s) - y) * LN2;  // others' log-sum minus the target's logit
        const float l = fmaxf(diff, 0.0f) + log1pf(expf(-fabsf(diff)));
        if (loss) loss[r] = l;
        if (lse) lse[r] = fmaf(y, LN2, l);
    }
}

struct Grad {
    const void *h, *w;
    int64_t ldw;
    int d, ldk, vocab, v0, width, ldg;  // the piece [v0, v0 + width) of the vocabulary; G is [rows][ldg]
    float c;
    float inv_t;
    const Head* head;
    const int* target;
    const float *lse2, *ghat;
    void* g;
    float* acc;  // [rows][d] sums of grad_hidden
    bool first;
    void* dw;
    int64_t lddw;
    float gscale, inv_gscale;  // G is held times gscale (a power of two)
};

template <typename T>
__global__ void __launch_bounds__(256) grad_logits_kernel(const Grad p) {
    const int kept = p.head->kept;
    const int m0 = blockIdx.y * TM, n0 = blockIdx.x * TN;
    if (m0 >= kept) return;
    float acc[4][4] = {};
    const T *h = static_cast<const T*>(p.h), *w = static_cast<const T*>(p.w) + (int64_t)p.v0 * p.ldw;
    tile_product(acc, p.d,
                 [&](int m, int k) { return m0 + m < kept ? to_f32(h[(int64_t)(m0 + m) * p.ldk + k]) : 0.0f; },
                 [&](int n, int k) { return n0 + n < p.width ? to_f32(w[(int64_t)(n0 + n) * p.ldw + k]) : 0.0f; });
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int r = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
            if (r >= kept || n >= p.width) continue;
            const float q = exp2f(fmaf(acc[i][j], p.c, -p.lse2[r])) - (p.v0 + n == p.target[r] ? 1.0f : 0.0f);
            static_cast<T*>(p.g)[(int64_t)r * p.ldg + n] = mxs::from_f32<T>(q * (p.ghat[r] * p.gscale));
        }
}

template <typename T>
__global__ void __launch_bounds__(256) grad_hidden_kernel(const Grad p) {
    const int kept = p.head->kept;
    const int m0 = blockIdx.y * TM, n0 = blockIdx.x * TN;
    if (m0 >= kept) return;
    float acc[4][4] = {};
    const T *g = static_cast<const T*>(p.g), *w = static_cast<const T*>(p.w) + (int64_t)p.v0 * p.ldw;
    tile_product(acc, p.width,
                 [&](int m, int k) { return m0 + m < kept ? to_f32(g[(int64_t)(m0 + m) * p.ldg + k]) : 0.0f; },
                 [&](int n, int k) { return n0 + n < p.d ? to_f32(w[(int64_t)k * p.ldw + n0 + n]) : 0.0f; });
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int r = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
            if (r >= kept || n >= p.d) continue;
            float* a = p.acc + (int64_t)r * p.d + n;
            *a = p.first ? acc[i][j] : *a + acc[i][j];
        }
}

template <typename T>
__global__ void __launch_bounds__(256) grad_weight_kernel(const Grad p) {
    const int kept = p.head->kept;
    const int m0 = blockIdx.y * TM, n0 = blockIdx.x * TN;
    float acc[4][4] = {};
    const T *g = static_cast<const T*>(p.g), *h = static_cast<const T*>(p.h);
    tile_product(acc, kept,
                 [&](int m, int k) { return m0 + m < p.width ? to_f32(g[(int64_t)k * p.ldg + m0 + m]) : 0.0f; },
                 [&](int n, int k) { return n0 + n < p.d ? to_f32(h[(int64_t)k * p.ldk + n0 + n]) : 0.0f; });
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const float s = p.head->gmax * p.inv_t * p.inv_gscale;
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
            if (m >= p.width || n >= p.d) continue;
            static_cast<T*>(p.dw)[(int64_t)(p.v0 + m) * p.lddw + n] = mxs::from_f32<T>(acc[i][j] * s);
        }
}

// grad_hidden of every row from the packed sums (rows left out: zero).
template <typename T>
__global__ void __launch_bounds__(256) grad_hidden_out_kernel(const float* acc, const int* pos, const Head* head,
                                                              int d, float scale, T* out, int64_t ld) {
    const int64_t r = blockIdx.x;
    const int at = pos[r];
    const float s = head->gmax * scale;
    for (int k = threadIdx.x; k < d; k += 256)
        out[r * ld + k] = mxs::from_f32<T>(at < 0 ? 0.0f : acc[(int64_t)at * d + k] * s);
}

// ---------------------------------------------------------------------------
// Plan
// ---------------------------------------------------------------------------
constexpr int PIECE = 8192;  // columns of G held at a time

struct Plan {
    Head* head;
    void* packed;
    int *pos, *target;
    float2* part;
    float *ytarget, *lse2, *ghat, *acc;
    void* g;
    int ldk, ldg;
    size_t bytes;
};

Plan make_plan(void* ws, int64_t rows, int64_t d, int64_t vocab, bool backward) {
    Plan pl{};
    Carve c(ws);
    const int64_t rp = round_up(rows, PACK_TAIL);
    pl.ldk = (int)round_up(d, 8);
    pl.head = c.take<Head>(1);
    pl.packed = c.take<uint16_t>((size_t)rp * pl.ldk);
    pl.pos = c.take<int>(rows);
    pl.target = c.take<int>(rows);
    if (!backward) {
        pl.part = c.take<float2>((size_t)ceil_div(vocab, TN) * rows);
        pl.ytarget = c.take<float>(rows);
    } else {
        pl.lse2 = c.take<float>(rows);
        pl.ghat = c.take<float>(rows);
        pl.ldg = (int)std::min<int64_t>(PIECE, round_up(vocab, 64));
        pl.g = c.take<uint16_t>((size_t)rp * pl.ldg);
        pl.acc = c.take<float>((size_t)rp * d);
    }
    pl.bytes = c.used;
    return pl;
}

bool bad_shape(int64_t ld_hidden, int64_t ld_weight, int dtype, int64_t rows, int64_t d, int64_t vocab,
               int target_bytes, double temperature) {
    return rows < 0 || d <= 0 || vocab <= 0 || rows > INT32_MAX - 256 || d > INT32_MAX - 256 ||
           vocab > INT32_MAX - 256 || ld_hidden < d || ld_weight < d || (dtype != MXS_BF16 && dtype != MXS_F16) ||
           (target_bytes != 4 && target_bytes != 8) || !(temperature > 0.0) || !std::isfinite(temperature);
}

template <typename T>
int launch_pack(const Pack& p, int sms, cudaStream_t st) {
    pack_rows_kernel<T><<<(int)std::min<int64_t>(p.rows, sms * 2), PACK_T, 0, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? MXS_OK : MXS_ERR_CUDA;
}

}  // namespace

extern "C" {

int mxs_ce_workspace_size(const void* d_weight, int64_t ld_weight, int64_t rows, int64_t d_model, int64_t vocab,
                          int backward, size_t* bytes) {
    if (!bytes || rows < 0 || d_model <= 0 || vocab <= 0 || ld_weight < d_model || rows > INT32_MAX - 256 ||
        d_model > INT32_MAX - 256 || vocab > INT32_MAX - 256)
        return MXS_ERR_INVALID;
    (void)d_weight;
    *bytes = make_plan(nullptr, rows, d_model, vocab, backward != 0).bytes;
    return MXS_OK;
}

int mxs_ce_from_hidden(const void* d_hidden, int64_t ld_hidden, const void* d_weight, int64_t ld_weight, int dtype,
                       int64_t rows, int64_t d_model, int64_t vocab, const void* d_targets, int target_bytes,
                       double temperature, float* d_loss, float* d_lse, void* d_workspace, size_t workspace_bytes,
                       void* stream) {
    if (bad_shape(ld_hidden, ld_weight, dtype, rows, d_model, vocab, target_bytes, temperature)) return MXS_ERR_INVALID;
    if (rows == 0) return MXS_OK;
    if (!d_hidden || !d_weight || !d_targets) return MXS_ERR_INVALID;
    int sms = 0;
    uint32_t* status = nullptr;
    int rc = mxs::device_info(&sms, &status);
    if (rc) return rc;
    const Plan pl = make_plan(d_workspace, rows, d_model, vocab, false);
    if (!mxs::workspace_ok(d_workspace, workspace_bytes, pl.bytes)) return MXS_ERR_WORKSPACE;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    Pack pk{d_hidden, ld_hidden, d_targets, target_bytes, (int)rows, (int)d_model, pl.ldk, vocab, nullptr, nullptr,
            pl.head, pl.packed, pl.pos, pl.target, nullptr, nullptr};
    rc = dtype == MXS_BF16 ? launch_pack<__nv_bfloat16>(pk, sms, st) : launch_pack<__half>(pk, sms, st);
    if (rc) return rc;
    const int tiles = (int)ceil_div(vocab, TN);
    Score s{pl.packed, d_weight, ld_weight, (int)d_model, pl.ldk, (int)vocab, (float)(LOG2E / temperature),
            pl.head, pl.target, pl.part, pl.ytarget, (int)rows};
    const dim3 grid(tiles, (unsigned)ceil_div(rows, TM));
    if (dtype == MXS_BF16)
        score_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(s);
    else
        score_kernel<__half><<<grid, 256, 0, st>>>(s);
    score_join_kernel<<<(unsigned)ceil_div(rows, 8), 256, 0, st>>>(pl.part, pl.ytarget, pl.pos, (int)rows, tiles,
                                                                   d_loss, d_lse);
    return cudaGetLastError() == cudaSuccess ? MXS_OK : MXS_ERR_CUDA;
}

int mxs_ce_from_hidden_backward(const void* d_hidden, int64_t ld_hidden, const void* d_weight, int64_t ld_weight,
                                int dtype, int64_t rows, int64_t d_model, int64_t vocab, const void* d_targets,
                                int target_bytes, double temperature, const float* d_lse, const float* d_grad_loss,
                                void* d_grad_hidden, int64_t ld_grad_hidden, void* d_grad_weight,
                                int64_t ld_grad_weight, void* d_workspace, size_t workspace_bytes, void* stream) {
    if (bad_shape(ld_hidden, ld_weight, dtype, rows, d_model, vocab, target_bytes, temperature) ||
        (d_grad_hidden && ld_grad_hidden < d_model) || (d_grad_weight && ld_grad_weight < d_model))
        return MXS_ERR_INVALID;
    if (!d_grad_hidden && !d_grad_weight) return MXS_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (rows == 0) {  // no row: the weight's gradient is zero
        if (d_grad_weight &&
            cudaMemset2DAsync(d_grad_weight, 2 * ld_grad_weight, 0, 2 * d_model, vocab, st) != cudaSuccess)
            return MXS_ERR_CUDA;
        return MXS_OK;
    }
    if (!d_hidden || !d_weight || !d_targets || !d_lse || !d_grad_loss) return MXS_ERR_INVALID;
    int sms = 0;
    uint32_t* status = nullptr;
    int rc = mxs::device_info(&sms, &status);
    if (rc) return rc;
    const Plan pl = make_plan(d_workspace, rows, d_model, vocab, true);
    if (!mxs::workspace_ok(d_workspace, workspace_bytes, pl.bytes)) return MXS_ERR_WORKSPACE;
    Pack pk{d_hidden, ld_hidden, d_targets, target_bytes, (int)rows, (int)d_model, pl.ldk, vocab, d_lse, d_grad_loss,
            pl.head, pl.packed, pl.pos, pl.target, pl.lse2, pl.ghat};
    rc = dtype == MXS_BF16 ? launch_pack<__nv_bfloat16>(pk, sms, st) : launch_pack<__half>(pk, sms, st);
    if (rc) return rc;
    // f16 holds G times 2^14: the target's entry stays below its largest value
    // and probabilities down to 2^-28 stay normal numbers
    const float gscale = dtype == MXS_F16 ? 16384.0f : 1.0f;
    Grad g{};
    g.h = pl.packed, g.w = d_weight, g.ldw = ld_weight, g.d = (int)d_model, g.ldk = pl.ldk, g.vocab = (int)vocab;
    g.ldg = pl.ldg, g.c = (float)(LOG2E / temperature), g.inv_t = (float)(1.0 / temperature), g.head = pl.head;
    g.target = pl.target, g.lse2 = pl.lse2, g.ghat = pl.ghat, g.g = pl.g, g.acc = pl.acc;
    g.dw = d_grad_weight, g.lddw = ld_grad_weight, g.gscale = gscale, g.inv_gscale = 1.0f / gscale;
    for (int64_t v0 = 0; v0 < vocab; v0 += pl.ldg) {
        g.v0 = (int)v0;
        g.width = (int)std::min<int64_t>(pl.ldg, vocab - v0);
        g.first = v0 == 0;
        const unsigned gm = (unsigned)ceil_div(rows, TM), gv = (unsigned)ceil_div(g.width, TN),
                       gd = (unsigned)ceil_div(d_model, TN);
        const bool bf = dtype == MXS_BF16;
        auto go = [&](auto kb, auto kh, dim3 grid) {
            if (bf)
                kb<<<grid, 256, 0, st>>>(g);
            else
                kh<<<grid, 256, 0, st>>>(g);
        };
        go(grad_logits_kernel<__nv_bfloat16>, grad_logits_kernel<__half>, dim3(gv, gm));
        if (d_grad_hidden) go(grad_hidden_kernel<__nv_bfloat16>, grad_hidden_kernel<__half>, dim3(gd, gm));
        if (d_grad_weight) go(grad_weight_kernel<__nv_bfloat16>, grad_weight_kernel<__half>, dim3(gd, gv));
    }
    if (d_grad_hidden) {
        const float sc = g.inv_t * g.inv_gscale;
        if (dtype == MXS_BF16)
            grad_hidden_out_kernel<<<(unsigned)rows, 256, 0, st>>>(pl.acc, pl.pos, pl.head, (int)d_model, sc,
                                                                   static_cast<__nv_bfloat16*>(d_grad_hidden),
                                                                   ld_grad_hidden);
        else
            grad_hidden_out_kernel<<<(unsigned)rows, 256, 0, st>>>(pl.acc, pl.pos, pl.head, (int)d_model, sc,
                                                                   static_cast<__half*>(d_grad_hidden),
                                                                   ld_grad_hidden);
    }
    return cudaGetLastError() == cudaSuccess ? MXS_OK : MXS_ERR_CUDA;
}

}  // extern "C"
