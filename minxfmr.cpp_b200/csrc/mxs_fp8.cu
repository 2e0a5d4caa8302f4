// 8-bit floats with a scale for each block of 128: the quantiser, the matrix
// product, and the sampler on the logits of an 8-bit output head
// (mxs_quantize_fp8, mxs_matmul_fp8, mxs_sample_from_hidden_fp8).
#include <algorithm>
#include <cfloat>
#include <cstring>

#include <cuda_fp8.h>

#include "mxs_gemm.cuh"
#include "mxs_head.cuh"
#include "mxs_launch.h"

namespace {

using mxs::Carve;
using mxs::ceil_div;
using mxs::round_up;
using mxs::gemm::Ctx;
using mxs::gemm::Lane;
using mxs::gemm::Tile;
using mxs::to_f32;

constexpr int BLK = 128;
constexpr float FP8_MAX = 448.0f;

__device__ __forceinline__ float block_scale(float top) {
    return top > 0.0f ? fmaxf(top / FP8_MAX, 1.17549435e-38f) : 1.0f;
}

// Eight values of a row as they lie in memory.
template <typename T>
struct Raw {
    uint4 u[sizeof(T) / 2];
};
__device__ __forceinline__ void values(const Raw<__nv_bfloat16>& x, float (&v)[8]) {
    const uint32_t w[4] = {x.u[0].x, x.u[0].y, x.u[0].z, x.u[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void values(const Raw<__half>& x, float (&v)[8]) {
    const uint32_t w[4] = {x.u[0].x, x.u[0].y, x.u[0].z, x.u[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void values(const Raw<float>& x, float (&v)[8]) {
    const uint32_t w[8] = {x.u[0].x, x.u[0].y, x.u[0].z, x.u[0].w, x.u[1].x, x.u[1].y, x.u[1].z, x.u[1].w};
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
}
// The largest magnitude as the type's own bits without the sign, which order as
// the magnitudes do, infinities and then NaN above every number; two 16-bit
// types in a word, each half by itself.
template <typename T>
__device__ __forceinline__ uint32_t top_bits(const Raw<T>& x) {
    const uint4& u = x.u[0];
    constexpr uint32_t M = 0x7fff7fffu;
    return __vmaxu2(__vmaxu2(u.x & M, u.y & M), __vmaxu2(u.z & M, u.w & M));
}
template <>
__device__ __forceinline__ uint32_t top_bits<float>(const Raw<float>& x) {
    constexpr uint32_t M = 0x7fffffffu;
    const uint4 &u = x.u[0], &w = x.u[1];
    return max(max(max(u.x & M, u.y & M), max(u.z & M, u.w & M)), max(max(w.x & M, w.y & M), max(w.z & M, w.w & M)));
}
template <typename T>
__device__ __forceinline__ uint32_t max_bits(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }
template <>
__device__ __forceinline__ uint32_t max_bits<float>(uint32_t a, uint32_t b) { return max(a, b); }
// Of the (halves of the) word: the magnitude, and whether it is no number.
__device__ __forceinline__ float magnitude(uint32_t m, const __nv_bfloat16*) {
    return __uint_as_float(max(m << 16, m & 0xffff0000u));
}
__device__ __forceinline__ float magnitude(uint32_t m, const __half*) {
    return __half2float(__ushort_as_half((unsigned short)max(m & 0xffffu, m >> 16)));
}
__device__ __forceinline__ float magnitude(uint32_t m, const float*) { return __uint_as_float(m); }

// 16-byte loads where the eight are aligned and inside the row; zeros outside.
template <typename T>
__device__ __forceinline__ Raw<T> load8(const T* x, int n, bool vec) {
    Raw<T> r;
    if (vec && n >= 8) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.u[i] = reinterpret_cast<const uint4*>(x)[i];
    } else {
        T t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = i < n ? x[i] : mxs::from_f32<T>(0.0f);
        memcpy(&r, t, sizeof r);
    }
    return r;
}

// x / s rounded to nearest, from r = 1 / s rounded to nearest: Markstein's
// theorem (IBM J. Res. Dev. 34, 1990) makes q + r (x - q s) the correctly rounded
// quotient for q = x r, as long as the remainder is exact. It is for finite x,
// s >= 2^-90 and quotients of at least 2^-11; smaller ones round to zero in 8
// bits either way.
__device__ __forceinline__ float quotient(float x, float s, float r) {
    const float q = x * r;
    return fmaf(fmaf(-q, s, x), r, q);
}
__device__ __forceinline__ uint32_t quad(const float* y) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
}

// Bound by memory: each value is read once and kept in registers, in its own type,
// between its block's maximum and its rounding. ROWS_OF = 1: sixteen lanes hold a
// block of 128, a warp two neighbouring ones, twice. ROWS_OF = 128: a CTA of 256
// threads holds a block, sixteen lanes a row, eight rows each. A block with an
// infinity or NaN, or with a scale below 2^-90, is read again and divided value
// by value.
template <typename T, int ROWS_OF>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 4 : 2)
    quantize_kernel(const T* __restrict__ x, int64_t ldx, int rows, int cols, uint8_t* __restrict__ q, int64_t ldq,
                    float* __restrict__ scale, bool vec_in, bool vec_out) {
    constexpr int HELD = ROWS_OF == 1 ? 2 : 8, TOPS = ROWS_OF == 1 ? HELD : 1;
    constexpr int DR = ROWS_OF == 1 ? 0 : 16, DC = ROWS_OF == 1 ? 2 * BLK : 0;
    const int tid = threadIdx.x, lane = tid & 31, sub = tid & 15;
    const int bc = (cols + BLK - 1) / BLK;
    int row0, col0;  // of the first eight; the others follow 256 columns or 16 rows on
    if (ROWS_OF == 1) {
        const uint32_t per_row = (bc + 3) / 4, task = blockIdx.x * 8 + (tid >> 5);
        row0 = task / per_row;
        col0 = (task % per_row) * (4 * BLK) + lane * 8;
    } else {
        row0 = (blockIdx.x / bc) * BLK + (tid >> 4);
        col0 = (blockIdx.x % bc) * BLK + sub * 8;
    }
    auto inside = [&](int i) { return row0 + i * DR < rows ? min(8, cols - col0 - i * DC) : 0; };  // may be negative
    const T* from = x + (int64_t)row0 * ldx + col0;
    uint8_t* to = q + (int64_t)row0 * ldq + col0;
    auto put = [&](int i, int n, uint2 w) {
        uint8_t* p = to + (int64_t)(i * DR) * ldq + i * DC;
        if (vec_out && n >= 8) {
            *reinterpret_cast<uint2*>(p) = w;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < n) p[j] = (uint8_t)((j < 4 ? w.x : w.y) >> (8 * (j & 3)));
        }
    };
    Raw<T> v[HELD];
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        const int n = inside(i);
        v[i] = load8(n > 0 ? from + (int64_t)(i * DR) * ldx + i * DC : x, n, vec_in);
    }
    __shared__ uint32_t s_top[8];
    __shared__ float s_slow[8];
    uint32_t bits[TOPS];
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        const uint32_t t = top_bits(v[i]);
        bits[i % TOPS] = i < TOPS ? t : max_bits<T>(bits[i % TOPS], t);
    }
#pragma unroll
    for (int i = 0; i < TOPS; ++i) {
#pragma unroll
        for (int o = 8; o; o >>= 1) bits[i] = max_bits<T>(bits[i], __shfl_xor_sync(0xffffffffu, bits[i], o));
        if (ROWS_OF != 1) {
            bits[i] = max_bits<T>(bits[i], __shfl_xor_sync(0xffffffffu, bits[i], 16));
            if (lane == 0) s_top[tid >> 5] = bits[i];
            __syncthreads();
#pragma unroll
            for (int w = 0; w < 8; ++w) bits[i] = max_bits<T>(bits[i], s_top[w]);
        }
    }
#pragma unroll
    for (int i = 0; i < TOPS; ++i) {
        const float top = magnitude(bits[i], static_cast<const T*>(nullptr));
        float s = block_scale(top);
        // ROWS_OF 1: one of the warp's blocks, so that the warp stays together; 128: the whole CTA agrees
        if (__any_sync(0xffffffffu, !(top <= FLT_MAX) || s < 8.0779357e-28f)) {  // 2^-90
            float m = 0.0f;
            for (int h = i; h < HELD; h += TOPS) {
                const int n = inside(h);
                for (int j = 0; j < n; ++j) {
                    const float a = fabsf(to_f32(from[(int64_t)(h * DR) * ldx + h * DC + j]));
                    if (a <= FLT_MAX) m = fmaxf(m, a);
                }
            }
#pragma unroll
            for (int o = 8; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            if (ROWS_OF != 1) {
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                if (lane == 0) s_slow[tid >> 5] = m;
                __syncthreads();
                for (int w = 0; w < 8; ++w) m = fmaxf(m, s_slow[w]);
            }
            s = block_scale(m);
            for (int h = i; h < HELD; h += TOPS) {
                const int n = inside(h);
                if (n <= 0) continue;
                float y[8];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    y[j] = j < n ? to_f32(from[(int64_t)(h * DR) * ldx + h * DC + j]) / s : 0.0f;
                put(h, n, make_uint2(quad(y), quad(y + 4)));
            }
        } else {
            const float r = 1.0f / s;
#pragma unroll
            for (int h = i; h < HELD; h += TOPS) {
                const int n = inside(h);
                if (n <= 0) continue;
                float y[8];
                values(v[h], y);
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] = quotient(y[j], s, r);
                put(h, n, make_uint2(quad(y), quad(y + 4)));
            }
        }
        if (ROWS_OF != 1 ? tid == 0 : sub == 0 && inside(i) > 0)
            scale[ROWS_OF != 1 ? (int64_t)blockIdx.x : (int64_t)row0 * bc + (col0 + i * DC) / BLK] = s;
    }
}

template <typename T>
cudaError_t launch_quantize(const void* x, int64_t ldx, int64_t rows, int64_t cols, int br, void* q, int64_t ldq,
                            float* scale, cudaStream_t st) {
    const int64_t bc = ceil_div(cols, BLK);
    const bool vin = mxs::aligned16(x, ldx * (int64_t)sizeof(T));
    const bool vout = reinterpret_cast<uintptr_t>(q) % 8 == 0 && ldq % 8 == 0;
    const T* xt = static_cast<const T*>(x);
    uint8_t* qt = static_cast<uint8_t*>(q);
    // runs of rows whose CTAs a grid can count
    const int64_t per = br == 1 ? ceil_div(bc, 4) : bc;      // tasks in a row of blocks
    const int64_t most = std::max<int64_t>(1, ((int64_t)INT32_MAX - 8) / per) * br;
    for (int64_t r = 0; r < rows; r += most) {
        const int64_t n = std::min(most, rows - r);
        float* sc = scale + r / br * bc;
        if (br == 1)
            quantize_kernel<T, 1><<<(unsigned)ceil_div(n * per, 8), 256, 0, st>>>(
                xt + r * ldx, ldx, (int)n, (int)cols, qt + r * ldq, ldq, sc, vin, vout);
        else
            quantize_kernel<T, 128><<<(unsigned)(ceil_div(n, BLK) * per), 256, 0, st>>>(
                xt + r * ldx, ldx, (int)n, (int)cols, qt + r * ldq, ldq, sc, vin, vout);
    }
    return cudaGetLastError();
}

// ---------------------------------------------------------------------------
// The product. A stage of the ring is one block of 128 of K (128 bytes of a
// row), so the accumulator of one block is one group: it is read back, scaled
// by a_scale * b_scale and added in registers while the MMAs of the next block
// fill the other accumulator. That join bounds the product above 128 rows: a block
// takes 930 clocks where its MMAs take 512. Its reads (256 clocks) and its FMAs (256
// a scheduler) would fit below them, but a warp waits for each 32 columns it reads
// before it adds them, and there are two warps a scheduler to fill the gaps.
// ---------------------------------------------------------------------------

// The i-th tile of a CTA that walks its own `span` of the columns, n at a time, so
// that all CTAs read the same amount of the second operand.
__device__ __forceinline__ bool span_tile(int i, const Ctx& x, int span, int n, int cols, int kb, Tile& t) {
    const int64_t at = (int64_t)x.unit * span + (int64_t)i * n;
    const int64_t end = min((int64_t)cols, (int64_t)(x.unit + 1) * span);
    if (at >= end) return false;
    t = Tile{0, (int)at, 0, kb, min(n, ((int)(end - at) + 31) / 32 * 32), 0};
    return true;
}

// RUNS: runs of 32 columns a thread holds, 4 for tiles of up to 256 columns, 2 for
// up to 128. The join has no branch around the sums (a warp without rows joins what
// it finds and stores nothing): where two paths meet the compiler copies all 128.
template <int CG_, typename O, int RUNS>
struct MatmulOp {
    static constexpr int CG = CG_;
    static constexpr int EPI = 8, SWAP = 0, STEP = 8 * EPI;  // columns from one run of a thread to its next
    static constexpr bool F8 = true, PROMOTE = true, ASIDE = false;
    __device__ int group() const { return 1; }
    struct Acc {
        float v[RUNS][32];
        const float *ra, *rb[RUNS];          // scales of this row, and of the runs of columns
        float row_next, next[RUNS];       // those of the next block
        float now[RUNS];                  // their products for this one
    };
    CUtensorMap ma, mb;
    int format;
    int64_t drop;
    uint32_t* status;
    const float *sa, *sb;
    int rows, cols, kb, mt, nt, n, a_rows;
    int span;  // CG 1: columns of a CTA
    O* out;
    int64_t ldo;
    bool vec;

    __device__ void prefetch() const {
        mxs::gemm::prefetch_map(&ma);
        mxs::gemm::prefetch_map(&mb);
    }
    __device__ int kept() const { return rows; }
    // CG 1 (one tile of rows): spans. CG 2: tiles go round the pairs, rows fastest.
    __device__ bool tile(int i, const Ctx& x, Tile& t) const {
        if (CG == 1) return span_tile(i, x, span, n, cols, kb, t);
        const int64_t idx = x.unit + (int64_t)i * x.units;
        if (idx >= (int64_t)mt * nt) return false;
        const int m = (int)(idx % mt), v = (int)(idx / mt);
        t = Tile{m * 128 * CG, v * n, 0, kb, n, 0};
        return true;
    }
    __device__ bool a_mn(const Tile&) const { return false; }
    __device__ bool b_mn(const Tile&) const { return false; }
    __device__ uint32_t bytes(const Tile& t) const { return (uint32_t)(a_rows + t.n / CG) * 128; }
    __device__ void load(const Tile& t, int k, uint32_t s_a, uint32_t s_b, uint32_t bar, const Ctx& x) const {
        mxs::gemm::tma_load<CG>(s_a, &ma, k * BLK, t.m0 + (int)x.rank * 128, bar);
        if (CG == 1)  // boxes of 32 rows: a tile of any multiple of that
            for (int j = 0; j < t.n; j += 32) mxs::gemm::tma_load<CG>(s_b + j * 128, &mb, k * BLK, t.n0 + j, bar);
        else
            mxs::gemm::tma_load<CG>(s_b, &mb, k * BLK, t.n0 + (int)x.rank * (n / CG), bar);
    }
    __device__ void zero(const Tile&, const Lane&, const Ctx&) const {}
    __device__ void fetch(Acc& a, int k) const {
        a.row_next = a.ra[k];
#pragma unroll
        for (int i = 0; i < RUNS; ++i) a.next[i] = a.rb[i][k];
    }
    __device__ void begin(Acc& a, const Tile& t, const Lane& me, const Ctx&) const {
#pragma unroll
        for (int i = 0; i < 32 * RUNS; ++i) a.v[i / 32][i % 32] = 0.0f;
        a.ra = sa + (int64_t)min(rows - 1, t.m0 + me.row) * kb;
#pragma unroll
        for (int i = 0; i < RUNS; ++i)  // 32 columns lie in one block of 128
            a.rb[i] = sb + (int64_t)(min(cols - 1, t.n0 + me.grp * 32 + i * STEP) / BLK) * kb;
        fetch(a, 0);
    }
    __device__ void prepare(Acc& a, const Tile&, int k, const Lane&, const Ctx&) const {
#pragma unroll
        for (int i = 0; i < RUNS; ++i) a.now[i] = a.row_next * a.next[i];
        fetch(a, min(k + 1, kb - 1));
    }
    template <typename Release>
    __device__ void join(Acc& a, const Tile& t, uint32_t tmem, const Lane& me, const Ctx&, Release release) const {
        const int c0 = me.grp * 32, end = t.n - 32;
#pragma unroll
        for (int i = 0; i < RUNS; ++i) {
            float x[32];
            mxs::gemm::tmem_ld32(tmem + min(c0 + i * STEP, end), x);  // a run past the tile's is not kept
            if (i == RUNS - 1) release();
#pragma unroll
            for (int j = 0; j < 32; ++j) a.v[i][j] = fmaf(x[j], a.now[i], a.v[i][j]);
        }
    }
    __device__ bool finish(Acc& a, const Tile& t, const Lane& me, const Ctx&) const {
        const int r0 = t.m0 + me.row - me.lane;
        if (r0 >= rows) return true;
        O* o = out + (int64_t)r0 * ldo + t.n0;
#pragma unroll
        for (int i = 0; i < RUNS; ++i) {
            const int c0 = me.grp * 32 + i * STEP;
            if (c0 >= t.n) break;
            mxs::gemm::store_rows<O, false, 32 * sizeof(O)>(o + c0, ldo, a.v[i], rows - r0, cols - t.n0 - c0, vec, me);
        }
        return true;
    }
};

// Up to 64 rows, as a decode step has them: the weight's rows lie along TMEM's
// lanes, 128 at a time, and NP >= rows rows of a along its columns. A thread holds
// one weight row's sums for NP rows, so the join costs what the rows there are
// cost, not 128, and the tensor core reads 4 KB of weight and NP * 32 bytes of a
// for 128 weight rows (operand reads, 64 bytes a clock, are what bounds an MMA of
// one CTA). Stores are 32 neighbouring columns a warp, whatever their alignment.
// Bound by the weight's bytes.
template <typename O, int NP>
struct DecodeOp {
    static constexpr int CG = 1, EPI = 8, SWAP = NP;
    static constexpr bool F8 = true, PROMOTE = true, ASIDE = false;
    __device__ int group() const { return 1; }
    struct Acc {
        float v[NP];
        const float *ra[NP > 32 ? 2 : 1], *rb;  // scales of rows lane, lane + 32 of a; of the warp's weight rows
        float next_a[NP > 32 ? 2 : 1], next_b;
    };
    CUtensorMap ma, mb;
    int format;
    int64_t drop;
    uint32_t* status;
    const float *sa, *sb;
    int rows, cols, kb, n, a_rows, span;
    O* out;
    int64_t ldo;

    __device__ void prefetch() const {
        mxs::gemm::prefetch_map(&ma);
        mxs::gemm::prefetch_map(&mb);
    }
    __device__ int kept() const { return rows; }
    __device__ bool tile(int i, const Ctx& x, Tile& t) const { return span_tile(i, x, span, n, cols, kb, t); }
    __device__ bool a_mn(const Tile&) const { return false; }
    __device__ bool b_mn(const Tile&) const { return false; }
    __device__ uint32_t bytes(const Tile& t) const { return (uint32_t)(a_rows + t.n) * 128; }
    __device__ void load(const Tile& t, int k, uint32_t s_a, uint32_t s_b, uint32_t bar, const Ctx&) const {
        mxs::gemm::tma_load<CG>(s_a, &ma, k * BLK, 0, bar);
        for (int j = 0; j < t.n; j += 32) mxs::gemm::tma_load<CG>(s_b + j * 128, &mb, k * BLK, t.n0 + j, bar);
    }
    __device__ void zero(const Tile&, const Lane&, const Ctx&) const {}
    // first weight row of the warp, of the tile's
    __device__ int first(const Lane& me) const { return me.grp * 128 + me.quad * 32; }
    __device__ void fetch(Acc& a, int k) const {
#pragma unroll
        for (int i = 0; i < (NP > 32 ? 2 : 1); ++i) a.next_a[i] = a.ra[i][k];
        a.next_b = a.rb[k];
    }
    __device__ void begin(Acc& a, const Tile& t, const Lane& me, const Ctx&) const {
#pragma unroll
        for (int i = 0; i < NP; ++i) a.v[i] = 0.0f;
#pragma unroll
        for (int i = 0; i < (NP > 32 ? 2 : 1); ++i) a.ra[i] = sa + (int64_t)min(rows - 1, me.lane + 32 * i) * kb;
        a.rb = sb + (int64_t)(min(cols - 1, t.n0 + first(me)) / BLK) * kb;  // 32 weight rows lie in one block of 128
        fetch(a, 0);
    }
    // the rows' scales of the block, times the weight's, where every lane can read them
    __device__ void prepare(Acc& a, const Tile&, int k, const Lane& me, const Ctx&) const {
        float* s = reinterpret_cast<float*>(me.xpose);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < (NP > 32 ? 2 : 1); ++i) s[me.lane + 32 * i] = a.next_a[i] * a.next_b;
        __syncwarp();
        fetch(a, min(k + 1, kb - 1));
    }
    template <typename Release>
    __device__ void join(Acc& a, const Tile&, uint32_t tmem, const Lane& me, const Ctx&, Release release) const {
        const float4* s = reinterpret_cast<const float4*>(me.xpose);
        constexpr int W = NP < 32 ? NP : 32;
#pragma unroll
        for (int i = 0; i < NP; i += W) {
            float x[W];
            mxs::gemm::tmem_ld(tmem + me.grp * NP + i, x);
            if (i + W == NP) release();
#pragma unroll
            for (int j = 0; j < W; j += 4) {
                const float4 q = s[(i + j) / 4];
                a.v[i + j] = fmaf(x[j], q.x, a.v[i + j]);
                a.v[i + j + 1] = fmaf(x[j + 1], q.y, a.v[i + j + 1]);
                a.v[i + j + 2] = fmaf(x[j + 2], q.z, a.v[i + j + 2]);
                a.v[i + j + 3] = fmaf(x[j + 3], q.w, a.v[i + j + 3]);
            }
        }
    }
    __device__ bool finish(Acc& a, const Tile& t, const Lane& me, const Ctx&) const {
        const int c = first(me) + me.lane;
        if (c >= t.n || t.n0 + c >= cols) return true;
        O* o = out + t.n0 + c;
#pragma unroll
        for (int i = 0; i < NP; ++i)
            if (i < rows) o[(int64_t)i * ldo] = mxs::from_f32<O>(a.v[i]);
        return true;
    }
};

template <int CG, typename O, int RUNS>
int launch_tiles(const void* a, int64_t lda, const float* sa, const void* b, int64_t ldb, const float* sb, int64_t rows,
                 int64_t n, int64_t k, void* out, int64_t ldo, int width, int span, int sms, uint32_t* status,
                 cudaStream_t st) {
    MatmulOp<CG, O, RUNS> op{};
    op.format = 0;
    op.drop = mxs::test_drop_tile();
    op.status = status;
    op.sa = sa, op.sb = sb;
    op.rows = (int)rows, op.cols = (int)n, op.kb = (int)ceil_div(k, BLK);
    op.mt = (int)ceil_div(rows, 128 * CG);
    op.n = width;
    op.span = span;
    op.nt = (int)ceil_div(n, op.n);
    op.a_rows = CG == 1 ? (int)round_up(rows, 8) : 128;
    op.out = static_cast<O*>(out);
    op.ldo = ldo;
    op.vec = mxs::aligned16(out, ldo * (int64_t)sizeof(O));
    if (!mxs::gemm::make_map(&op.ma, a, 1, k, rows, lda, op.a_rows) ||
        !mxs::gemm::make_map(&op.mb, b, 1, k, n, ldb, CG == 1 ? 32 : op.n / 2))
        return MXS_ERR_CUDA;
    const int64_t units = CG == 1 ? ceil_div(n, span) : (int64_t)op.mt * op.nt;
    return mxs::gemm::launch(op, (int)std::min<int64_t>(sms / CG, units), st) == cudaSuccess ? MXS_OK : MXS_ERR_CUDA;
}

template <typename O, int NP>
int launch_decode(const void* a, int64_t lda, const float* sa, const void* b, int64_t ldb, const float* sb,
                  int64_t rows, int64_t n, int64_t k, void* out, int64_t ldo, int width, int span, int sms, uint32_t* status,
                  cudaStream_t st) {
    DecodeOp<O, NP> op{};
    op.format = 0;
    op.drop = mxs::test_drop_tile();
    op.status = status;
    op.sa = sa, op.sb = sb;
    op.rows = (int)rows, op.cols = (int)n, op.kb = (int)ceil_div(k, BLK);
    op.n = width;
    op.span = span;
    op.a_rows = (int)round_up(rows, 8);  // rows that the box leaves out give columns nobody reads
    op.out = static_cast<O*>(out);
    op.ldo = ldo;
    if (!mxs::gemm::make_map(&op.ma, a, 1, k, rows, lda, op.a_rows) ||
        !mxs::gemm::make_map(&op.mb, b, 1, k, n, ldb, 32))
        return MXS_ERR_CUDA;
    return mxs::gemm::launch(op, (int)ceil_div(n, span), st) == cudaSuccess ? MXS_OK : MXS_ERR_CUDA;
}

template <typename O>
int launch_matmul(const void* a, int64_t lda, const float* sa, const void* b, int64_t ldb, const float* sb,
                  int64_t rows, int64_t n, int64_t k, void* out, int64_t ldo, int sms, uint32_t* status, cudaStream_t st) {
    const int span = (int)round_up(ceil_div(n, sms), 32);  // up to 128 rows: one tile of them
    const int w = rows > 128 ? mxs::tile_width(ceil_div(rows, 256), n, sms / 2, 64, 32)
                             : (int)round_up(ceil_div(span, ceil_div(span, 256)), 32);
    auto go = [&](auto f) { return f(a, lda, sa, b, ldb, sb, rows, n, k, out, ldo, w, span, sms, status, st); };
    // Rows along the columns up to 64 of them; 128 rows' sums no longer fit a thread beside the loads.
    if (rows <= 16) return go(launch_decode<O, 16>);
    if (rows <= 32) return go(launch_decode<O, 32>);
    if (rows <= 64) return go(launch_decode<O, 64>);
    if (rows > 128) return w > 128 ? go(launch_tiles<2, O, 4>) : go(launch_tiles<2, O, 2>);
    return w > 128 ? go(launch_tiles<1, O, 4>) : go(launch_tiles<1, O, 2>);
}

bool bad_type(int t) { return t != MXS_BF16 && t != MXS_F16 && t != MXS_F32; }
constexpr int64_t LIMIT = INT32_MAX - 1024;

// Aligned copies of the operands that need one.
struct Copies {
    void *a, *b;
    size_t bytes;
};
Copies copies(void* ws, const void* a, int64_t lda, const void* b, int64_t ldb, int64_t rows, int64_t n, int64_t k) {
    Carve c(ws);
    const int64_t ldk = round_up(k, 16);
    Copies r{};
    if (!mxs::aligned16(a, lda)) r.a = c.take<uint8_t>((size_t)rows * ldk);
    if (!mxs::aligned16(b, ldb)) r.b = c.take<uint8_t>((size_t)n * ldk);
    r.bytes = c.used;
    return r;
}

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
    const cudaError_t e =
        dtype == MXS_BF16  ? launch_quantize<__nv_bfloat16>(d_x, ld_x, rows, cols, block_rows, d_q, ld_q, d_scale, st)
        : dtype == MXS_F16 ? launch_quantize<__half>(d_x, ld_x, rows, cols, block_rows, d_q, ld_q, d_scale, st)
                           : launch_quantize<float>(d_x, ld_x, rows, cols, block_rows, d_q, ld_q, d_scale, st);
    return e == cudaSuccess ? MXS_OK : MXS_ERR_CUDA;
}

int mxs_matmul_fp8_workspace_size(const void* d_a, int64_t ld_a, const void* d_b, int64_t ld_b, int64_t rows,
                                  int64_t n, int64_t k, size_t* bytes) {
    if (!bytes || rows < 0 || n <= 0 || k <= 0 || ld_a < k || ld_b < k || rows > LIMIT || n > LIMIT || k > LIMIT)
        return MXS_ERR_INVALID;
    *bytes = copies(nullptr, d_a, ld_a, d_b, ld_b, rows, n, k).bytes;
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
    int sms = 0;
    uint32_t* status = nullptr;
    int rc = mxs::device_info(&sms, &status);
    if (rc) return rc;
    const Copies cp = copies(d_workspace, d_a, ld_a, d_b, ld_b, rows, n, k);
    if (!mxs::workspace_ok(d_workspace, workspace_bytes, cp.bytes)) return MXS_ERR_WORKSPACE;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int64_t ldk = round_up(k, 16);
    if (cp.a) {
        if (mxs::copy_rows(d_a, ld_a, cp.a, ldk, rows, k, sms, st) != cudaSuccess) return MXS_ERR_CUDA;
        d_a = cp.a, ld_a = ldk;
    }
    if (cp.b) {
        if (mxs::copy_rows(d_b, ld_b, cp.b, ldk, n, k, sms, st) != cudaSuccess) return MXS_ERR_CUDA;
        d_b = cp.b, ld_b = ldk;
    }
    auto go = [&](auto f) {
        return f(d_a, ld_a, d_a_scale, d_b, ld_b, d_b_scale, rows, n, k, d_out, ld_out, sms, status, st);
    };
    return out_dtype == MXS_F32    ? go(launch_matmul<float>)
           : out_dtype == MXS_BF16 ? go(launch_matmul<__nv_bfloat16>)
                                   : go(launch_matmul<__half>);
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
