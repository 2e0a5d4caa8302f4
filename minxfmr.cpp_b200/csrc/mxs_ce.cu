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
// max |grad| keeps a batch mean's 1/rows out of G and its range in the types';
// what the rounding of a row's target entry, its largest, leaves out is added to
// both gradients in fp32.
//
// Rows whose target is out of range are packed away first (pack_rows_kernel), so
// they cost no products; every later kernel reads the number of rows left from
// device memory. (Forward, up to 128 aligned rows: read in place instead.)
//
// Bound by the tensor cores from some hundred rows on (512 clocks of MMA for each
// 64 of K and 256 x 256 tile; at 4096 x 151936 x 3584 the power limit holds the
// clock near 1.4 GHz), by the weight's bytes below.
#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>
#include <type_traits>

#include "mxs_gemm.cuh"
#include "mxs_head.cuh"
#include "mxs_launch.h"

namespace {

using mxs::Carve;
using mxs::ceil_div;
using mxs::round_up;
using mxs::to_f32;
using mxs::gemm::Ctx;
using mxs::gemm::Lane;
using mxs::gemm::Tile;

constexpr int64_t MAX_DIM = INT32_MAX - 1024;
// What a wait of at most a second spans grows with the rows where more than 16 of them share
// a target: a CTA's warps look for the rows of up to 128 such targets. 2^24 rows of 128 targets
// take 0.4 s.
constexpr int64_t MAX_BACKWARD_ROWS = 1 << 24;
constexpr float LN2 = 0.693147180559945309f;
constexpr double LOG2E = 1.4426950408889634074;

struct Head {
    int kept;      // rows with a target in range
    float gmax;    // largest finite |grad_loss| of those rows (1 if none)
};

// Splits of K for the grad_hidden tiles of a piece of `width` columns: so many that
// one split takes about a unit's share of the launch's work, grad_weight's tiles
// included (a tile of few blocks counts as 8: its epilogue takes as long as those),
// at least 8 blocks of 64 columns each, and no more than fill the units. A fixed
// function of the shape: the same sums in the same order every time. (A step of
// 200 x 32000 x 512: 91 us with the 36 splits that fill the units, 80 us with these 13.)
__host__ __device__ inline int grad_hidden_splits(int kept, int nt, int width, int units, bool want_w) {
    const int64_t tiles = (int64_t)((kept + 255) / 256) * nt;
    if (tiles == 0) return 1;
    const int64_t blocks = (width + 63) / 64, rows = (kept + 63) / 64;
    const int64_t other = want_w ? (int64_t)((width + 255) / 256) * nt * (rows > 8 ? rows : 8) : 0;
    const int64_t work = tiles * blocks + other;
    int64_t s = (blocks * units + work - 1) / work;
    const int64_t most = (blocks + 7) / 8, fill = units / tiles;
    s = s < most ? s : most;
    s = s < fill ? s : fill;
    s = s < 1 ? 1 : s;
    const int64_t per = (blocks + s - 1) / s;
    return (int)((blocks + per - 1) / per);  // none of them empty
}

// The caller's targets: the row's, or -1 where it is outside the vocabulary.
struct Targets {
    const void* at;
    int bytes;
    int vocab;
    __device__ __forceinline__ int operator()(int64_t r) const {
        const int64_t t = bytes == 8 ? static_cast<const int64_t*>(at)[r]
                                     : (int64_t)static_cast<const int32_t*>(at)[r];
        return t >= 0 && t < vocab ? (int)t : -1;
    }
};

// The packed rows whose target is one vocabulary row and whose entry of G its rounding
// changed are its group: counted for every vocabulary row, and the first LISTED of them,
// in any order, written down with what the rounding left out.
constexpr int LISTED = 16;
struct alignas(8) Left {
    int row;
    float rest;
};

struct Pack {
    const void* hidden;
    int64_t ld_hidden;
    Targets targets;
    int rows, d, ldk;
    const float* lse;   // backward: null in forward
    const float* grad;
    Head* head;
    void* packed;       // [rows_pad][ldk]
    int* pos;           // [rows]: packed row or -1
    int* target;        // [packed]
    float* lse2;        // [packed] lse * log2(e)
    float* ghat;        // [packed] grad / gmax
    int* counts;        // [vocab]: zeroed for GradLogitsOp (null: no gradient of the weight)
};

constexpr int PACK_T = 256;
constexpr int PACK_ROWS = 256;  // packed rows are allocated in multiples of this

// Each CTA packs a contiguous range of rows; it counts the kept rows before its
// range itself (a few KB of targets from L2), so one launch does it all. In
// backward every CTA scans all rows (for the largest gradient weight) and so
// knows how many are kept: together they zero the rows up to the next multiple
// of 64, which grad_weight's product reads as its last block of K.
template <typename T>
__global__ void __launch_bounds__(PACK_T) pack_rows_kernel(const Pack p) {
    mxs::gemm::grid_wait();
    mxs::gemm::grid_launch_dependents();
    __shared__ int s_cnt[PACK_T / 32], s_all[PACK_T / 32], s_pos[PACK_T];
    __shared__ float s_max[PACK_T / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (int)ceil_div(p.rows, gridDim.x);
    const int r0 = min(p.rows, (int)blockIdx.x * per), r1 = min(p.rows, r0 + per);
    int n = 0, all = 0;
    float gm = 0.0f;
    const int scan_to = p.grad ? p.rows : r0;
#pragma unroll 4
    for (int r = tid; r < scan_to; r += PACK_T) {
        const bool keep = p.targets(r) >= 0;
        const float g = p.grad ? fabsf(p.grad[r]) : 0.0f;
        all += keep;
        n += keep && r < r0;
        if (keep && g <= FLT_MAX) gm = fmaxf(gm, g);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        n += __shfl_xor_sync(0xffffffffu, n, o);
        all += __shfl_xor_sync(0xffffffffu, all, o);
        gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, o));
    }
    if (lane == 0) s_cnt[warp] = n, s_all[warp] = all, s_max[warp] = gm;
    __syncthreads();
    n = all = 0;
    gm = 0.0f;
    for (int w = 0; w < PACK_T / 32; ++w) {
        n += s_cnt[w];
        all += s_all[w];
        gm = fmaxf(gm, s_max[w]);
    }
    if (!(gm > 0.0f)) gm = 1.0f;
    int base = n;
    constexpr int STEP = 16 / sizeof(T);
    const bool vec = reinterpret_cast<uintptr_t>(p.hidden) % 16 == 0 && p.ld_hidden % STEP == 0;
    for (int c0 = r0; c0 < r1; c0 += PACK_T) {
        const int r = c0 + tid;
        const int tgt = r < r1 ? p.targets(r) : -1;
        const bool keep = tgt >= 0;
        const uint32_t b = __ballot_sync(0xffffffffu, keep);
        __syncthreads();
        if (lane == 0) s_cnt[warp] = __popc(b);
        __syncthreads();
        int at = base + __popc(b & ((1u << lane) - 1)), here = 0;
        for (int w = 0; w < PACK_T / 32; ++w) {
            if (w < warp) at += s_cnt[w];
            here += s_cnt[w];
        }
        s_pos[tid] = keep ? at : -1;
        if (r < r1) p.pos[r] = keep ? at : -1;
        if (keep) {
            p.target[at] = tgt;
            if (p.grad) {
                p.lse2[at] = p.lse[r] * (float)LOG2E;
                p.ghat[at] = p.grad[r] / gm;
            }
        }
        base += here;
        __syncthreads();
        // the rows themselves, a warp each
        for (int i = warp; i < min(PACK_T, r1 - c0); i += PACK_T / 32) {
            const int to = s_pos[i];
            if (to < 0) continue;
            const T* src = static_cast<const T*>(p.hidden) + (int64_t)(c0 + i) * p.ld_hidden;
            T* dst = static_cast<T*>(p.packed) + (int64_t)to * p.ldk;
            int k = lane;
            if (vec) {
#pragma unroll 4
                for (int j = lane; j < p.d / STEP; j += 32)
                    reinterpret_cast<uint4*>(dst)[j] = reinterpret_cast<const uint4*>(src)[j];
                k += p.d / STEP * STEP;
            }
            for (; k < p.d; k += 32) dst[k] = src[k];
        }
    }
    if (p.grad) {
        for (int64_t i = blockIdx.x * (int64_t)PACK_T + tid; p.counts && i < p.targets.vocab;
             i += (int64_t)gridDim.x * PACK_T)
            p.counts[i] = 0;
        const int64_t words = (int64_t)((64 - all % 64) % 64) * p.ldk / STEP;  // ldk is a multiple of 8
        uint4* tail = reinterpret_cast<uint4*>(static_cast<T*>(p.packed) + (int64_t)all * p.ldk);
        for (int64_t i = blockIdx.x * (int64_t)PACK_T + tid; i < words; i += (int64_t)gridDim.x * PACK_T)
            tail[i] = make_uint4(0, 0, 0, 0);
    }
    if (r1 == p.rows && r0 < r1 && tid == 0) {  // the range that ends the rows knows how many were kept
        p.head->kept = base;
        p.head->gmax = gm;
    }
}

// ---------------------------------------------------------------------------
// Logit tiles (forward): rows of H against rows of W, both K-major.
// ---------------------------------------------------------------------------

__device__ __forceinline__ float ex2(float x) {  // 2^x, 2^-22 relative; results below 2^-126 are 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// What the two passes over the logits share: the tiles' walk (rows fastest, so
// the tiles in flight share their weight rows in L2) and the loads.
template <int CG_>
struct LogitTiles {
    static constexpr int CG = CG_;
    static constexpr int EPI = 16, SWAP = 0;
    static constexpr bool F8 = false, PROMOTE = false, ASIDE = false;
    __device__ int group() const { return INT32_MAX; }
    CUtensorMap mh, mw;
    int format;
    int64_t drop;
    uint32_t* status;
    const Head* head;    // null: the rows lie as the caller has them, none packed away
    const int* target;
    Targets targets;     // read where the rows are not packed
    int rows, vocab;     // vocab: columns of this pass (its piece), starting at v0
    int v0, n, nt, kblocks, a_rows;
    int span;            // CG 1: columns of a CTA
    float c;             // log2(e) / temperature

    __device__ void prefetch() const {
        mxs::gemm::prefetch_map(&mh);
        mxs::gemm::prefetch_map(&mw);
    }
    __device__ int kept() const {
        if (head) return *(volatile const int*)&head->kept;
        return rows;  // not one conditional of two lvalues: that would load from either address
    }
    __device__ int target_of(int r) const {
        if (head) return target[r];
        return targets(r);
    }
    // CG 1 (one tile of rows): a CTA walks its own span of columns, so that all read
    // the same amount of weight. CG 2: tiles go round the pairs.
    __device__ bool tile(int i, const Ctx& x, Tile& t) const {
        if (CG == 1) {
            const int64_t at = (int64_t)x.unit * span + (int64_t)i * n;
            const int64_t end = min((int64_t)vocab, (int64_t)(x.unit + 1) * span);
            if (at >= end || x.kept == 0) return false;
            const int w = min(n, ((int)(end - at) + 31) / 32 * 32);
            t = Tile{0, (int)at, 0, kblocks, w, x.unit * ((span + n - 1) / n) + i};
            return true;
        }
        const int mt = (x.kept + 128 * CG - 1) / (128 * CG);
        const int64_t idx = x.unit + (int64_t)i * x.units;
        if (idx >= (int64_t)mt * nt) return false;
        const int m = (int)(idx % mt), v = (int)(idx / mt);
        t = Tile{m * 128 * CG, v * n, 0, kblocks, n, v};
        return true;
    }
    __device__ bool a_mn(const Tile&) const { return false; }
    __device__ bool b_mn(const Tile&) const { return false; }
    __device__ uint32_t bytes(const Tile& t) const { return (uint32_t)(a_rows + t.n / CG) * 128; }
    __device__ void load(const Tile& t, int kb, uint32_t sa, uint32_t sb, uint32_t bar, const Ctx& x) const {
        mxs::gemm::tma_load<CG>(sa, &mh, kb * 64, t.m0 + (int)x.rank * 128, bar);
        if (CG == 1)  // boxes of 32 rows: a tile of any multiple of that
            for (int j = 0; j < t.n; j += 32) mxs::gemm::tma_load<CG>(sb + j * 128, &mw, kb * 64, v0 + t.n0 + j, bar);
        else
            mxs::gemm::tma_load<CG>(sb, &mw, kb * 64, v0 + t.n0 + (int)x.rank * (n / CG), bar);
    }
    __device__ void zero(const Tile&, const Lane&, const Ctx&) const {}
};

// Each thread holds a quarter of a tile's columns of one row: the largest y of
// the others and sum 2^(y - largest); the four of a row meet in shared memory. The
// exponentials run at 16 a clock and SM: 2048 clocks for 128 x 256, against 512
// clocks of MMA for each 64 of d_model.
// The MMA's own fp32 sum rounds towards zero at every 16 products, which at
// d_model 3584 leaves 2e-6 of the logits' size; the accumulator is joined in
// registers (round to nearest) after a run of products, which costs one more read of
// it for each. Above 128 rows every 512: loss and lse of 4096 x 151936 x 3584 are 2.9e-7
// from 64 bits (a plain fp32 form: 5.5e-7) in 3.27 ms; every 256 would leave 1.5e-7 and
// take 3.51. Up to 128 rows, where the weight's bytes are waited for, every 128, and the
// targets' logits, whose products lean to one sign where a model has learnt something, are
// plain fp32 dot products, a row a CTA, by a warp that has nothing else to do: the loss of one
// row of d 896, median, 95th percentile and largest of 200: 1.3e-7, 1.0e-6 and 2.2e-6 (a plain
// fp32 form: 6.8e-8, 8.9e-7, 1.9e-6) in 55.3 us; every 256 2.0e-7, 1.5e-6, 2.6e-6 in 53.4; every
// 512 without the dot products 2.5e-7, 4.8e-6, 7.8e-6 in 53.4. Products of one sign lose 3e-7 of
// a logit in bf16 and 2.6e-6 in f16, whose products have more bits to lose, in runs of 512, a
// fifth of that and less in runs of 128.
template <int CG_>
struct ScoreOp : LogitTiles<CG_> {
    static constexpr bool PROMOTE = true, ASIDE = CG_ == 1;
    __device__ int group() const { return CG_ == 1 ? 2 : 8; }
    struct Acc {
        float v[2][32];
    };
    float2* part;    // [tile][rows]
    float* ytarget;  // [rows]: the target's logit times the temperature
    const uint16_t *h, *w;  // ASIDE: the operands that the maps read
    int64_t ldh, ldw;
    int d;

    __device__ __forceinline__ float2 pair(uint32_t x) const {
        if (this->format == 0) return __half22float2(*reinterpret_cast<const __half2*>(&x));
        return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
    }
    __device__ void aside(const Ctx& x, int lane) const {
        for (int r = x.unit; r < x.kept; r += x.units) {
            const int v = this->target_of(r);
            if (v < 0) continue;
            const uint16_t *a = h + r * ldh, *b = w + v * ldw;  // rows start on 16-byte boundaries
            float s = 0.0f, s2 = 0.0f;
            for (int j = lane; j < d / 8; j += 32) {
                const uint4 p = reinterpret_cast<const uint4*>(a)[j], q = reinterpret_cast<const uint4*>(b)[j];
                const uint32_t pw[4] = {p.x, p.y, p.z, p.w}, qw[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 f = pair(pw[i]), g = pair(qw[i]);
                    s = fmaf(f.x, g.x, s);
                    s2 = fmaf(f.y, g.y, s2);
                }
            }
            for (int k = d / 8 * 8 + lane; k < d; k += 32) s = fmaf(pair(a[k]).x, pair(b[k]).x, s);
            s += s2;
#pragma unroll
            for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            if (lane == 0) ytarget[r] = s;
        }
    }
    __device__ void begin(Acc& a, const Tile&, const Lane&, const Ctx&) const {
#pragma unroll
        for (int i = 0; i < 64; ++i) a.v[i / 32][i % 32] = 0.0f;
    }
    __device__ void prepare(Acc&, const Tile&, int, const Lane&, const Ctx&) const {}
    template <typename Release>
    __device__ void join(Acc& a, const Tile& t, uint32_t tmem, const Lane& me, const Ctx& x, Release release) const {
        if (((t.m0 + me.row) & ~31) < x.kept) {  // a row of this warp
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int c0 = me.grp * 32 + i * 128;
                if (c0 < t.n) {
                    float v[32];
                    mxs::gemm::tmem_ld32(tmem + c0, v);
#pragma unroll
                    for (int j = 0; j < 32; ++j) a.v[i][j] += v[j];
                }
            }
        }
        release();
    }
    __device__ bool finish(Acc& a, const Tile& t, Lane& me, const Ctx& x) const {
        const int r = t.m0 + me.row;
        if ((r & ~31) >= x.kept) return true;  // the four warps of these rows agree
        const int hit = r < x.kept ? this->target_of(r) - t.n0 : -1;  // the target's column of this tile
        const int cols = min(t.n, this->vocab - t.n0);
        float m = -INFINITY, s = 0.0f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int c0 = me.grp * 32 + i * 128;
            if (c0 >= t.n) break;
            float(&v)[32] = a.v[i];
            if (hit >= c0 && hit < c0 + 32) {
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    if (mxs::gemm::is_column(hit - c0, j)) {
                        if (!ASIDE) ytarget[r] = v[j];
                        v[j] = -INFINITY;
                    }
            }
            if (c0 + 32 > cols) {
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    if (c0 + j >= cols) v[j] = -INFINITY;
            }
            float top = v[0];
#pragma unroll
            for (int j = 1; j < 32; ++j) top = fmaxf(top, v[j]);
            const float nm = fmaxf(m, top * this->c);
            const float sub = nm == -INFINITY ? 0.0f : nm;
            float sum[4] = {s * ex2(m - sub), 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < 32; ++j) sum[j & 3] += ex2(fmaf(v[j], this->c, -sub));
            s = (sum[0] + sum[1]) + (sum[2] + sum[3]);
            m = nm;
        }
        // Two buffers, taken in turn by the meetings (not by the tiles, some of which these warps
        // skip): what is written for one meeting is read before that warp comes to the next, and
        // overwritten only after it.
        float2* mine = reinterpret_cast<float2*>(me.xpose) + (me.meetings & 1) * 32 + me.lane;
        *mine = make_float2(m, s);
        if (!mxs::gemm::meet(me, x)) return false;
        if (me.grp != 0 || r >= x.kept) return true;
#pragma unroll
        for (int g = 1; g < 4; ++g) {  // group g's warp is four places on
            const float2 q = mine[g * 4 * (mxs::gemm::XPOSE_ALL / LogitTiles<CG_>::EPI / 8)];
            const float nm = fmaxf(m, q.x), sub = nm == -INFINITY ? 0.0f : nm;
            s = s * ex2(m - sub) + q.y * ex2(q.x - sub);
            m = nm;
        }
        part[(int64_t)t.kind * this->rows + r] = make_float2(m, s);
        return true;
    }
};

__device__ __forceinline__ void join_pair(float& m, float& s, float om, float os) {
    const float nm = fmaxf(m, om), sub = nm == -INFINITY ? 0.0f : nm;
    s = s * ex2(m - sub) + os * ex2(om - sub);
    m = nm;
}

// Joins the tiles' pairs of a row, in the same order every time. Few rows (WHOLE): a
// CTA a row. Many: a CTA for 32 rows, a lane each, so that the pairs of neighbouring
// rows are read together, its 32 warps a part of the tiles each.
template <bool WHOLE>
__global__ void __launch_bounds__(1024) score_join_kernel(const float2* part, const float* ytarget, const int* pos,
                                                         Targets targets, int rows, int tiles, float c, float* loss,
                                                         float* lse) {
    constexpr int WARPS = WHOLE ? 8 : 32;
    __shared__ float2 s_pair[WARPS][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int r = WHOLE ? blockIdx.x : blockIdx.x * 32 + lane;
    mxs::gemm::grid_wait();
    mxs::gemm::grid_launch_dependents();
    int at = -1;
    if (r < rows) {
        at = targets(r) >= 0 ? r : -1;
        if (pos) at = pos[r];
    }
    float m = -INFINITY, s = 0.0f;
    if (at >= 0) {
        const int per = (tiles + WARPS - 1) / WARPS;
        const int from = WHOLE ? threadIdx.x : warp * per, to = WHOLE ? tiles : min(tiles, from + per);
#pragma unroll 8
        for (int i = from; i < to; i += WHOLE ? 256 : 1) {
            const float2 q = part[(int64_t)i * rows + at];
            join_pair(m, s, q.x, q.y);
        }
    }
    if (WHOLE) {
#pragma unroll
        for (int o = 16; o; o >>= 1)
            join_pair(m, s, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
    }
    if (!WHOLE || lane == 0) s_pair[warp][WHOLE ? 0 : lane] = make_float2(m, s);
    __syncthreads();
    if (WHOLE ? threadIdx.x != 0 : warp != 0 || r >= rows) return;
    for (int w = 1; w < WARPS; ++w) {
        const float2 q = s_pair[w][WHOLE ? 0 : lane];
        join_pair(m, s, q.x, q.y);
    }
    float l = 0.0f, e = 0.0f;  // a row left out
    if (at >= 0) {
        // the others' log-sum minus the target's logit. The sums are relative to m as it is, so one
        // rounding of m - y c, at the difference's size, is all that the logits' own size costs.
        const float y = ytarget[at];
        const float diff = (fmaf(-y, c, m) + log2f(s)) * LN2;
        l = fmaxf(diff, 0.0f) + log1pf(expf(-fabsf(diff)));
        e = fmaf(y * c, LN2, l);
    }
    if (loss) loss[r] = l;
    if (lse) lse[r] = e;
}

// The logits of a piece again, left as G = ghat (softmax - hot) in the operands'
// type (rounded once; the products that read it accumulate in fp32). They are the
// MMA's own sums over all of d_model: the 2e-6 of the logits' size that the loss's
// join spares is little beside that rounding. A row's target entry outweighs the
// others, and its rounding would be an error common to the whole row, so what it
// leaves out is kept in fp32 and added to both gradients where they are finished
// (errors against 64 bits of bf16 gradients with weights of all sizes: 0.0024
// without, 0.0018 with, 0.0017 for the result's own rounding). The rows that leave
// something are counted, and the first few listed, for each target.
// Rows after the last kept one and columns after the piece read zero.
template <int CG_, typename T>
struct GradLogitsOp : LogitTiles<CG_> {
    const float *lse2, *ghat;
    T* g;
    float* rest;  // [packed]: what the rounding of each row's target entry leaves out
    int* counts;    // [vocab]; null: no gradient of the weight
    Left* listed;   // [piece][LISTED]
    int ldg;
    float gscale;

    struct Ahead {
        static constexpr bool ok = true;
    };
    __device__ Ahead ahead(const Tile&, const Lane&, const Ctx&) const { return {}; }
    __device__ void epilogue(const Tile& t, uint32_t tmem, const Lane& me, const Ctx& x, Ahead, int) const {
        const int r = t.m0 + me.row;
        const bool live = r < x.kept;
        const int hit = live ? this->target[r] - this->v0 - t.n0 : -1;
        const float l2 = live ? lse2[r] : 0.0f;
        const float gr = live ? ghat[r] * gscale : 0.0f;
        const int cols = this->vocab - t.n0;
        T* out = g + (int64_t)(r - me.lane) * ldg + t.n0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int c0 = me.grp * 32 + i * 128;
            if (c0 >= t.n || t.n0 + c0 >= ldg) break;
            float v[32];
            mxs::gemm::tmem_ld32(tmem + c0, v);
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = ex2(fmaf(v[j], this->c, -l2)) * gr;
            if (hit >= c0 && hit < c0 + 32) {
                float left = 0.0f;
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    if (mxs::gemm::is_column(hit - c0, j)) {
                        v[j] -= gr;
                        left = v[j] - to_f32(mxs::from_f32<T>(v[j]));
                    }
                rest[r] = left;
                if (counts && left != 0.0f) {
                    const int64_t v = t.n0 + hit;
                    const int k = atomicAdd(counts + this->v0 + v, 1);
                    if (k < LISTED) listed[v * LISTED + k] = Left{r, left};
                }
            }
            if (!live || c0 + 32 > cols) {
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    if (!live || c0 + j >= cols) v[j] = 0.0f;
            }
            mxs::gemm::store_rows<T, false>(out + c0, ldg, v, 32, 32, true, me);
        }
    }
};

// Both products of a piece in one launch. kind >= 0: grad_hidden += G W (M rows, N
// d_model, K the piece's columns, cut into `splits` where the tiles alone are
// fewer than the pairs); kind < 0: grad_weight = G^T H (M the piece's columns, N
// d_model, K rows). G is read K-major for the first and M-major for the second.
template <typename T>
struct ProductOp {
    static constexpr int CG = 2;
    static constexpr int EPI = 16, SWAP = 0;
    static constexpr bool F8 = false, PROMOTE = false, ASIDE = false;
    // Sums of more than 32768 products are added up in fp32 after so many: the MMA's own
    // sum rounds towards zero at every 16 of them, which by then may have cost 2^-13 of it
    // (2 million rows of one sign, in one run: 8 parts in a thousand).
    static constexpr int RUN = 512;
    __device__ int group() const { return RUN; }
    CUtensorMap g_k, g_m, w_n, h_n;
    int format;
    int64_t drop;
    uint32_t* status;
    const Head* head;
    int v0, width, d, n, nt;  // nt tiles of n columns over d
    int split_width;          // the widest piece: what the number of splits goes by
    float* acc;               // sums of grad_hidden, a block of 256 x 256 per tile and split
    float* runs;              // [CTA][128][256]: sums of grad_weight so far, where they take several runs
    bool first, want_h, want_w;
    const int* counts;        // GradLogitsOp's
    const Left* listed;
    const float* rest;
    const int* target;
    float* sums;              // [first listed row][lds]: of a group's rests * hidden
    int lds;
    const T* h;               // the packed rows
    int ldh;
    T* dw;
    int64_t lddw;
    float scale;              // 1 / temperature / (G's own power of two)
    bool vec;

    __device__ void prefetch() const {
        mxs::gemm::prefetch_map(&g_k);
        mxs::gemm::prefetch_map(&g_m);
        mxs::gemm::prefetch_map(&w_n);
        mxs::gemm::prefetch_map(&h_n);
    }
    __device__ int kept() const { return *(volatile const int*)&head->kept; }
    // The grad_hidden tiles go round the pairs first; when they leave some pairs
    // with one tile fewer, those take the grad_weight tiles of the same cost before the rest go round.
    __device__ bool tile(int i, const Ctx& x, Tile& t) const {
        const int mh = want_h ? (x.kept + 255) / 256 : 0, th = mh * nt;
        const int splits = grad_hidden_splits(want_h ? x.kept : 0, nt, split_width, x.units, want_w);
        const int kh = (width + 63) / 64, kw = (x.kept + 63) / 64;
        const int nh = th * splits;
        const int mine = (nh - x.unit + x.units - 1) / x.units;  // grad_hidden tiles of this unit
        if (i < mine) {
            const int idx = x.unit + i * x.units;
            const int tileno = idx % th, s = idx / th;
            const int per = (kh + splits - 1) / splits;
            const int k0 = min(kh, s * per);
            t = Tile{tileno / nt * 256, tileno % nt * n, k0, min(kh, k0 + per) - k0, n, tileno * splits + s};
            return true;
        }
        if (!want_w) return false;
        const int64_t total = (int64_t)((width + 255) / 256) * nt;
        const int over = nh % x.units;  // units [0, over) have one tile more
        const int cost = max(kw, 8);  // of a grad_weight tile, in blocks
        const int ahead = over == 0 ? 0 : ((kh + splits - 1) / splits + cost / 2) / cost;
        int j = i - mine;
        int64_t idx;
        if (x.unit >= over && j < ahead) {
            idx = x.unit - over + (int64_t)j * (x.units - over);
        } else {
            if (x.unit >= over) j -= ahead;
            idx = (int64_t)ahead * (x.units - over) + x.unit + (int64_t)j * x.units;
        }
        if (idx >= total) return false;
        t = Tile{(int)(idx / nt) * 256, (int)(idx % nt) * n, 0, kw, n, -1};
        return true;
    }
    __device__ bool a_mn(const Tile& t) const { return t.kind < 0; }
    __device__ bool b_mn(const Tile&) const { return true; }
    __device__ uint32_t bytes(const Tile&) const { return (uint32_t)(128 + n / 2) * 128; }
    __device__ void load(const Tile& t, int kb, uint32_t sa, uint32_t sb, uint32_t bar, const Ctx& x) const {
        const int m = t.m0 + (int)x.rank * 128, c = t.n0 + (int)x.rank * (n / 2), k = kb * 64;
        if (t.kind >= 0) {
            mxs::gemm::tma_load<2>(sa, &g_k, k, m, bar);
        } else {
            mxs::gemm::tma_load<2>(sa, &g_m, m, k, bar);
            mxs::gemm::tma_load<2>(sa + 8192, &g_m, m + 64, k, bar);
        }
        const CUtensorMap* b = t.kind >= 0 ? &w_n : &h_n;
        const int kr = t.kind >= 0 ? v0 + k : k;
        for (int j = 0; j < n / 128; ++j) mxs::gemm::tma_load<2>(sb + j * 8192, b, c + 64 * j, kr, bar);
    }
    // What the rests of rows that share a target add to its grad_weight row, in ascending
    // order of the rows whatever the order they were counted in. One row or two: the thread
    // that holds the vocabulary row adds them (add_rest). More, for the CTA's 128 vocabulary
    // rows and the tile's columns, before the tile's accumulator is waited for, under its
    // products, whose time grows with the rows too: up to LISTED rows are sorted and summed
    // by a warp, up to FEW found among all targets by a warp, more found and summed by all
    // warps, each a sixteenth of the rows, and these sums added in order. Both gradients of
    // 4096 x 32000 x 512: uniform targets 348 us, Zipf 408, 60 % on one id 396, all on one 374,
    // on 32 neighbours 416.
    static constexpr int FEW = 256;
    static constexpr int EACH = 128, LIST = EACH + 32;  // targets looked at at once, and a warp's list

    // a += rest * hidden of n listed rows, eight columns from `from` on, eight rows' loads in flight.
    __device__ void add_rows(float (&a)[8], const int* list, int n, const T* from) const {
        for (int e = 0; e < n; e += 8) {
            uint4 u[8];
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int r = list[min(e + i, n - 1)];
                f[i] = rest[r];
                u[i] = *reinterpret_cast<const uint4*>(from + (int64_t)r * ldh);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (e + i >= n) f[i] = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) a[j] = fmaf(f[i], to_f32(reinterpret_cast<const T*>(&u[i])[j]), a[j]);
            }
        }
    }
    // The same for the rows with target v among blocks [b0, b1) of EACH rows.
    __device__ void find_rows(float (&a)[8], int* list, int v, int b0, int b1, const T* from, int lane,
                              int kept) const {
        const int4* at = reinterpret_cast<const int4*>(target) + lane;
        int found = 0;
        __syncwarp();
        for (int k0 = b0; k0 < b1; k0 += 4) {  // four blocks' loads in flight
            int4 u[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] = at[(int64_t)min(k0 + i, b1 - 1) * (EACH / 4)];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = (k0 + i) * EACH + 4 * lane, here[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
                bool hit[4], any = false;
#pragma unroll
                for (int j = 0; j < 4; ++j) any |= hit[j] = here[j] == v && r + j < kept && k0 + i < b1;
                if (!__any_sync(0xffffffffu, any)) continue;
                int to = found;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t w = __ballot_sync(0xffffffffu, hit[j]);
                    to += __popc(w & ((1u << lane) - 1));
                    found += __popc(w);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (hit[j]) list[to++] = r + j;
                if (found <= LIST - EACH) continue;
                __syncwarp();
                add_rows(a, list, found, from);
                __syncwarp();
                found = 0;
            }
        }
        __syncwarp();
        add_rows(a, list, found, from);
        __syncwarp();
    }
    __device__ bool sum_groups(const Tile& t, int m, Lane& me, const Ctx& x) const {
        constexpr int XPOSE = mxs::gemm::Geo<ProductOp>::XPOSE;
        const int warp = me.grp * 4 + me.quad, c = t.n0 + me.lane * 8;
        const bool mine = me.lane * 8 < n && c < ldh;  // rows are whole 16-byte pieces
        const T* from = h + (mine ? c : 0);
        float* part = reinterpret_cast<float*>(me.xpose);  // 256 columns' sums of this warp
        int* list = reinterpret_cast<int*>(me.xpose + 1024);
        const int blocks = (x.kept + EACH - 1) / EACH, per = (blocks + EPI - 1) / EPI;
        int turn = 0;
        for (int q = 0; q < 4; ++q) {
            const int row = m + q * 32 + me.lane, count = row < width ? counts[v0 + row] : 0;
            for (uint32_t b = __ballot_sync(0xffffffffu, count > 2 && count <= FEW); b; b &= b - 1) {
                if (turn++ % EPI != warp) continue;
                const int i = __ffs(b) - 1, n_rows = __shfl_sync(0xffffffffu, count, i), v = m + q * 32 + i;
                const Left* of = listed + (int64_t)v * LISTED;
                float a[8] = {};
                if (n_rows <= LISTED) {
                    const int r = me.lane < n_rows ? of[me.lane].row : INT_MAX;
                    int to = 0;
#pragma unroll
                    for (int k = 0; k < LISTED; ++k) to += __shfl_sync(0xffffffffu, r, k) < r;
                    __syncwarp();
                    if (me.lane < n_rows) list[to] = r;
                    __syncwarp();
                    add_rows(a, list, n_rows, from);
                } else {
                    find_rows(a, list, v0 + v, 0, blocks, from, me.lane, x.kept);
                }
                if (mine) {
                    float4* to = reinterpret_cast<float4*>(sums + (int64_t)of[0].row * lds + c);
                    to[0] = make_float4(a[0], a[1], a[2], a[3]);
                    to[1] = make_float4(a[4], a[5], a[6], a[7]);
                }
            }
        }
        for (int q = 0; q < 4; ++q) {
            const int row = m + q * 32 + me.lane, count = row < width ? counts[v0 + row] : 0;
            for (uint32_t b = __ballot_sync(0xffffffffu, count > FEW); b; b &= b - 1) {
                const int v = m + q * 32 + __ffs(b) - 1;
                float a[8] = {};
                const int b0 = min(blocks, warp * per), b1 = min(blocks, b0 + per);
                find_rows(a, list, v0 + v, b0, b1, from, me.lane, x.kept);
                reinterpret_cast<float4*>(part)[me.lane * 2] = make_float4(a[0], a[1], a[2], a[3]);
                reinterpret_cast<float4*>(part)[me.lane * 2 + 1] = make_float4(a[4], a[5], a[6], a[7]);
                if (!mxs::gemm::gather(me, x)) return false;
                const int col = warp * 32 + me.lane;
                if (col < n && t.n0 + col < d) {
                    const float* first = reinterpret_cast<const float*>(me.xpose - warp * XPOSE) + col;
                    float s = 0.0f;
                    for (int w = 0; w < EPI; ++w) s += first[w * (XPOSE / 4)];
                    sums[(int64_t)listed[(int64_t)v * LISTED].row * lds + t.n0 + col] = s;
                }
                if (!mxs::gemm::gather(me, x)) return false;  // before the parts are written again
            }
        }
        return mxs::gemm::gather(me, x);
    }
    // The group of this thread's vocabulary row: its size and its first two (as they are listed).
    struct Ahead {
        int count;
        int4 left;
        bool ok;
    };
    __device__ Ahead ahead(const Tile& t, Lane& me, const Ctx& x) const {
        Ahead it{0, make_int4(0, 0, 0, 0), true};
        if (t.kind >= 0) return it;
        const int m = t.m0 + (int)x.rank * 128;
        bool many = false;  // a group to be summed among the CTA's
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int row = m + q * 32 + me.lane, count = row < width ? counts[v0 + row] : 0;
            if (q == me.quad) it.count = count;
            many |= count > 2;
        }
        if (m + me.row % 128 < width)
            it.left = *reinterpret_cast<const int4*>(listed + (int64_t)(t.m0 + me.row) * LISTED);
        if (__any_sync(0xffffffffu, many)) it.ok = sum_groups(t, m, me, x);
        return it;
    }
    // v += rest * hidden of a row, columns [c, c + 32).
    __device__ void add_row(float (&v)[32], int r, float left, int c) const {
        const T* row = h + (int64_t)r * ldh + c;
        if (c + 32 <= ldh) {  // rows are whole 16-byte pieces; what lies past d is not stored
#pragma unroll
            for (int j = 0; j < 32; j += 8) {
                const uint4 u = *reinterpret_cast<const uint4*>(row + j);
                const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
                for (int q = 0; q < 8; ++q) v[j + q] = fmaf(left, to_f32(e[q]), v[j + q]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (c + j < d) v[j] = fmaf(left, to_f32(row[j]), v[j]);
        }
    }
    // What the target entries' roundings left out of this thread's vocabulary row, columns [c, c + 32).
    __device__ void add_rest(float (&v)[32], const Ahead& it, int c) const {
        if (it.count > 2) {
            if (c < d) {  // lds is a multiple of 32
                const float4* row = reinterpret_cast<const float4*>(sums + (int64_t)it.left.x * lds + c);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float4 u = row[j];
                    v[4 * j] += u.x;
                    v[4 * j + 1] += u.y;
                    v[4 * j + 2] += u.z;
                    v[4 * j + 3] += u.w;
                }
            }
        } else {
            const bool swap = it.count == 2 && it.left.z < it.left.x;
            for (int k = 0; k < it.count; ++k) {
                const bool second = (k == 1) != swap;
                add_row(v, second ? it.left.z : it.left.x, __int_as_float(second ? it.left.w : it.left.y), c);
            }
        }
        __syncwarp();
    }
    __device__ void epilogue(const Tile& t, uint32_t tmem, const Lane& me, const Ctx&, const Ahead& it, int kb) const {
        const bool last = kb + RUN >= t.kn;
        // two factors: their product may leave fp32's range where the results do not
        const float gmax = t.kind >= 0 ? 1.0f : head->gmax;
        const int m = t.m0 + me.row - me.lane;  // first row of the warp
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int c0 = me.grp * 32 + i * 128;
            if (c0 >= n) break;
            float v[32];
            mxs::gemm::tmem_ld32(tmem + c0, v);
            if (t.kind >= 0) {
                float* a = acc + ((int64_t)t.kind * 256 + me.row - me.lane) * 256 + c0;
                if (first && kb == 0)
                    mxs::gemm::store_rows<float, false>(a, 256, v, 32, 32, true, me);
                else
                    mxs::gemm::store_rows<float, true>(a, 256, v, 32, 32, true, me);
            } else {
                if (!last || kb > 0) {
                    float* a = runs + ((int64_t)blockIdx.x * 128 + me.quad * 32) * 256 + c0;
                    if (kb == 0)
                        mxs::gemm::store_rows<float, false>(a, 256, v, 32, 32, true, me);
                    else
                        mxs::gemm::store_rows<float, true>(a, 256, v, 32, 32, true, me);
                    if (!last) continue;
                    __syncwarp();
                    const float4* sum = reinterpret_cast<const float4*>(a + me.lane * 256);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float4 u = sum[j];
                        v[4 * j] = u.x, v[4 * j + 1] = u.y, v[4 * j + 2] = u.z, v[4 * j + 3] = u.w;
                    }
                    __syncwarp();
                }
                add_rest(v, it, t.n0 + c0);
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = v[j] * scale * gmax;
                mxs::gemm::store_rows<T, false>(dw + (int64_t)(v0 + m) * lddw + t.n0 + c0, lddw, v, width - m,
                                                d - t.n0 - c0, vec, me);
            }
        }
    }
    __device__ void zero(const Tile& t, const Lane& me, const Ctx&) const {
        if (t.kind >= 0) return;  // a split without columns, of a last piece: nothing to add
        const int m = t.m0 + me.row - me.lane;
        const float v[32] = {};
        for (int c0 = me.grp * 32; c0 < n; c0 += 128)
            mxs::gemm::store_rows<T, false>(dw + (int64_t)(v0 + m) * lddw + t.n0 + c0, lddw, v, width - m,
                                            d - t.n0 - c0, vec, me);
    }
};

// grad_hidden of every row: its tiles' splits added in order, and what its target
// entry's rounding left out, times the scale (rows left out: zero).
template <typename T>
__global__ void __launch_bounds__(128) grad_hidden_out_kernel(const float* acc, const int* pos, const Head* head,
                                                              const int* target, const float* rest, const T* w,
                                                              int64_t ldw, int d, int n, int width, int units,
                                                              bool want_w, float scale, T* out, int64_t ld) {
    mxs::gemm::grid_wait();
    mxs::gemm::grid_launch_dependents();
    const int64_t r = blockIdx.y;
    const int k = (blockIdx.x * 128 + threadIdx.x) * 4;  // four columns of one tile
    if (k >= d) return;
    const int at = pos[r];
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (at >= 0) {
        const int nt = (d + n - 1) / n, splits = grad_hidden_splits(head->kept, nt, width, units, want_w);
        const int64_t tile = (int64_t)(at / 256) * nt + k / n;
        const float* a = acc + (tile * splits * 256 + at % 256) * 256 + k % n;
#pragma unroll 8
        for (int i = 0; i < splits; ++i) {
            const float4 q = *reinterpret_cast<const float4*>(a + (int64_t)i * 65536);
            v = make_float4(v.x + q.x, v.y + q.y, v.z + q.z, v.w + q.w);
        }
        const T* row = w + (int64_t)target[at] * ldw + k;
        const float left = rest[at];
        v.x = fmaf(left, to_f32(row[0]), v.x);
        if (k + 1 < d) v.y = fmaf(left, to_f32(row[1]), v.y);
        if (k + 2 < d) v.z = fmaf(left, to_f32(row[2]), v.z);
        if (k + 3 < d) v.w = fmaf(left, to_f32(row[3]), v.w);
        const float g = head->gmax;  // as in ProductOp
        v = make_float4(v.x * scale * g, v.y * scale * g, v.z * scale * g, v.w * scale * g);
    }
    T* o = out + r * ld + k;
    const float y[4] = {v.x, v.y, v.z, v.w};
    if (k + 4 <= d && ld % 4 == 0 && reinterpret_cast<uintptr_t>(out) % 8 == 0) {
        T t[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = mxs::from_f32<T>(y[i]);
        *reinterpret_cast<uint2*>(o) = *reinterpret_cast<const uint2*>(t);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (k + i < d) o[i] = mxs::from_f32<T>(y[i]);
    }
}

// ---------------------------------------------------------------------------
// Plan
// ---------------------------------------------------------------------------
// G is held for a piece of the vocabulary at a time, of about this many bytes. A
// piece costs two launches whose last tiles leave pairs idle, so larger ones are
// faster, with less and less to gain; L2 holds none of them beside its operands.
// Loss and gradients of 4096 x 151936 x 3584: 13.57 ms with 64 MB, 13.2 with 128,
// 13.0 with 512.
constexpr int64_t PIECE_BYTES = 256 << 20;

struct Plan {
    Head* head;
    void* packed;
    int *pos, *target;
    int* counts;
    Left* listed;
    float *rest, *sums, *runs;
    float2* part;
    float *ytarget, *lse2, *ghat, *acc;
    void* g;
    void* w;          // the weight in aligned rows, if its own are not
    int ldk, lds;
    int n, nt;        // logit tiles
    int span;         // one tile of rows: columns of a CTA
    bool direct;      // forward on the caller's own rows
    int dn, dnt;      // tiles over d_model
    int64_t piece;
    size_t bytes;
};

// Logit tiles over `cols` columns.
void plan_tiles(Plan& pl, int sms, int64_t rows, int64_t cols) {
    if (rows <= 128) {
        pl.span = (int)round_up(ceil_div(cols, sms), 32);
        pl.n = (int)round_up(ceil_div(pl.span, ceil_div(pl.span, 256)), 32);
        const int64_t before = ceil_div(cols, pl.span) - 1;  // CTAs with a whole span
        pl.nt = (int)(before * ceil_div(pl.span, pl.n) + ceil_div(cols - before * pl.span, pl.n));
    } else {
        pl.n = mxs::tile_width(ceil_div(rows, 256), cols, sms / 2, 64, 64);
        pl.nt = (int)ceil_div(cols, pl.n);
    }
}

Plan make_plan(void* ws, int sms, const void* weight, int64_t ldw, int64_t rows, int64_t d, int64_t vocab,
               bool backward) {
    Plan pl{};
    Carve c(ws);
    rows = std::max<int64_t>(rows, 1);
    const int64_t rp = round_up(rows, PACK_ROWS);
    pl.ldk = (int)round_up(d, 8);
    pl.head = c.take<Head>(1);
    pl.packed = c.take<uint16_t>((size_t)rp * pl.ldk);
    pl.pos = c.take<int>(rows);
    pl.target = c.take<int>(round_up(rows, 128));  // read 128 at a time
    pl.w = mxs::aligned16(weight, 2 * ldw) ? nullptr : c.take<uint16_t>((size_t)vocab * pl.ldk);
    if (!backward) {
        plan_tiles(pl, sms, rows, vocab);
        pl.part = c.take<float2>((size_t)pl.nt * rows);
        pl.ytarget = c.take<float>(rows);
    } else {
        pl.lse2 = c.take<float>(rows);
        pl.ghat = c.take<float>(rows);
        pl.counts = c.take<int>(vocab);
        pl.rest = c.take<float>(rows);
        pl.lds = (int)round_up(d, 32);
        pl.sums = c.take<float>((size_t)rows * pl.lds);
        const int64_t most = std::max<int64_t>(256, PIECE_BYTES / (2 * rp));
        pl.piece = round_up(ceil_div(vocab, ceil_div(vocab, most)), 256);
        plan_tiles(pl, sms, rows, std::min(pl.piece, vocab));
        pl.g = c.take<uint16_t>((size_t)rp * pl.piece);
        pl.listed = c.take<Left>((size_t)pl.piece * LISTED);
        pl.dn = d > 128 ? 256 : 128;
        pl.dnt = (int)ceil_div(d, pl.dn);
        if (rows > 64 * ProductOp<__half>::RUN) pl.runs = c.take<float>((size_t)sms * 128 * 256);
        pl.acc = c.take<float>((size_t)std::max<int64_t>(rp / 256 * pl.dnt, sms / 2) * 65536);
    }
    pl.bytes = c.used;
    return pl;
}

bool bad_shape(int64_t ld_hidden, int64_t ld_weight, int dtype, int64_t rows, int64_t d, int64_t vocab,
               int target_bytes, double temperature) {
    return rows < 0 || d <= 0 || vocab <= 0 || rows > MAX_DIM || d > MAX_DIM || vocab > MAX_DIM || ld_hidden < d ||
           ld_weight < d || (dtype != MXS_BF16 && dtype != MXS_F16) || (target_bytes != 4 && target_bytes != 8) ||
           !(temperature > 0.0) || !std::isfinite(temperature);
}

template <typename T>
constexpr int format_of() { return std::is_same<T, __half>::value ? 0 : 1; }

// A kernel that may start while the one before it drains.
template <typename... P, typename... A>
cudaError_t launch_dependent(void (*k)(P...), dim3 grid, unsigned block, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k, static_cast<P>(args)...);
}

struct Call {
    const void* hidden;
    int64_t ldh;
    const void* weight;
    int64_t ldw;
    int64_t rows, d, vocab;
    Targets targets;
    double temperature;
    int sms;
    uint32_t* status;
    cudaStream_t st;
};

#define MXS_TRY(e)                               \
    do {                                         \
        if ((e) != cudaSuccess) return MXS_ERR_CUDA; \
    } while (0)

template <typename T>
int pack_rows(const Call& a, const Plan& pl, const float* lse, const float* grad, bool want_w) {
    const Pack p{a.hidden, a.ldh, a.targets, (int)a.rows, (int)a.d, pl.ldk, lse, grad, pl.head,
                 pl.packed, pl.pos, pl.target, pl.lse2, pl.ghat, want_w ? pl.counts : nullptr};
    // a CTA for four rows, and for 2048 counts to be zeroed
    const int64_t ctas = std::max(ceil_div(a.rows, 4), want_w ? ceil_div(a.vocab, 8 * PACK_T) : 0);
    MXS_TRY(launch_dependent(pack_rows_kernel<T>, (unsigned)std::min<int64_t>(ctas, a.sms * 4), PACK_T, a.st, p));
    return MXS_OK;
}

template <int CG, typename T>
int logit_tiles(LogitTiles<CG>& op, const Call& a, const Plan& pl, const void* w, int64_t ldw) {
    op.format = format_of<T>();
    op.drop = mxs::test_drop_tile();
    op.status = a.status;
    op.head = pl.direct ? nullptr : pl.head;
    op.target = pl.target;
    op.targets = a.targets;
    op.rows = (int)a.rows;
    op.n = pl.n;
    op.span = pl.span;
    op.kblocks = (int)ceil_div(a.d, 64);
    op.a_rows = CG == 1 ? (int)round_up(a.rows, 8) : 128;
    op.c = (float)(LOG2E / a.temperature);
    // rows of the tile that the box leaves out keep what shared memory held: their results are not read
    const bool rows_ok = pl.direct ? mxs::gemm::make_map(&op.mh, a.hidden, 2, a.d, a.rows, a.ldh, op.a_rows)
                                   : mxs::gemm::make_map(&op.mh, pl.packed, 2, a.d, round_up(a.rows, PACK_ROWS), pl.ldk,
                                                         op.a_rows);
    if (!rows_ok || !mxs::gemm::make_map(&op.mw, w, 2, a.d, a.vocab, ldw, CG == 1 ? 32 : pl.n / 2)) return MXS_ERR_CUDA;
    return MXS_OK;
}

template <int CG, typename T>
int score(const Call& a, const Plan& pl, const void* w, int64_t ldw, float* loss, float* lse) {
    ScoreOp<CG> op{};
    int rc = logit_tiles<CG, T>(op, a, pl, w, ldw);
    if (rc) return rc;
    op.vocab = (int)a.vocab;
    op.nt = pl.nt;
    op.part = pl.part;
    op.ytarget = pl.ytarget;
    op.h = static_cast<const uint16_t*>(pl.direct ? a.hidden : pl.packed);
    op.ldh = pl.direct ? a.ldh : pl.ldk;
    op.w = static_cast<const uint16_t*>(w);
    op.ldw = ldw;
    op.d = (int)a.d;
    // CG 1: a CTA for each span of columns, and for each row's target
    const int64_t units = CG == 1 ? std::max(ceil_div(a.vocab, pl.span), a.rows) : ceil_div(a.rows, 256) * pl.nt;
    MXS_TRY(mxs::gemm::launch(op, (int)std::min<int64_t>(a.sms / CG, units), a.st));
    const int* pos = pl.direct ? nullptr : pl.pos;
    if (a.rows <= 64)
        MXS_TRY(launch_dependent(score_join_kernel<true>, (unsigned)a.rows, 256, a.st, pl.part, pl.ytarget, pos,
                                 a.targets, (int)a.rows, pl.nt, op.c, loss, lse));
    else
        MXS_TRY(launch_dependent(score_join_kernel<false>, (unsigned)ceil_div(a.rows, 32), 1024, a.st, pl.part,
                                 pl.ytarget, pos, a.targets, (int)a.rows, pl.nt, op.c, loss, lse));
    return MXS_OK;
}

template <int CG, typename T>
int grad_piece(const Call& a, const Plan& pl, const void* w, int64_t ldw, int64_t v0, ProductOp<T>& prod) {
    GradLogitsOp<CG, T> op{};
    int rc = logit_tiles<CG, T>(op, a, pl, w, ldw);
    if (rc) return rc;
    op.v0 = (int)v0;
    op.vocab = (int)std::min(pl.piece, a.vocab - v0);
    op.nt = (int)ceil_div(op.vocab, pl.n);  // CG 2
    op.lse2 = pl.lse2;
    op.ghat = pl.ghat;
    op.g = static_cast<T*>(pl.g);
    op.rest = pl.rest;
    op.counts = prod.want_w ? pl.counts : nullptr;
    op.listed = pl.listed;
    op.ldg = (int)pl.piece;
    // f16 holds G times 2^14: the target's entry stays below its largest value
    // and entries down to 2^-28 of the largest gradient weight stay normal numbers
    op.gscale = format_of<T>() == 0 ? 16384.0f : 1.0f;
    const int64_t units = CG == 1 ? ceil_div(op.vocab, pl.span) : ceil_div(a.rows, 256) * op.nt;
    MXS_TRY(mxs::gemm::launch(op, (int)std::min<int64_t>(a.sms / CG, units), a.st));
    prod.v0 = (int)v0;
    prod.width = op.vocab;
    prod.first = v0 == 0;
    // columns after the piece are not read: the map ends there
    if (!mxs::gemm::make_map(&prod.g_k, pl.g, 2, prod.width, round_up(a.rows, PACK_ROWS), pl.piece, 128) ||
        !mxs::gemm::make_map(&prod.g_m, pl.g, 2, prod.width, round_up(a.rows, PACK_ROWS), pl.piece, 64))
        return MXS_ERR_CUDA;
    MXS_TRY(mxs::gemm::launch(prod, a.sms / 2, a.st));
    return MXS_OK;
}

template <typename T>
int forward(const Call& a, Plan pl, float* loss, float* lse) {
    const void* w = a.weight;
    int64_t ldw = a.ldw;
    if (pl.w) {
        MXS_TRY(mxs::copy_rows(a.weight, 2 * a.ldw, pl.w, 2 * pl.ldk, a.vocab, 2 * a.d, a.sms, a.st));
        w = pl.w, ldw = pl.ldk;
    }
    // Up to 128 rows are one tile whether some are left out or not: where they are
    // aligned they are read as they lie (rows left out compute numbers nobody reads).
    pl.direct = a.rows <= 128 && mxs::aligned16(a.hidden, 2 * a.ldh);
    if (!pl.direct)
        if (const int rc = pack_rows<T>(a, pl, nullptr, nullptr, false)) return rc;
    return a.rows > 128 ? score<2, T>(a, pl, w, ldw, loss, lse) : score<1, T>(a, pl, w, ldw, loss, lse);
}

template <typename T>
int backward(const Call& a, const Plan& pl, const float* lse, const float* grad, void* gh, int64_t ldgh, void* gw,
             int64_t ldgw) {
    const void* w = a.weight;
    int64_t ldw = a.ldw;
    if (pl.w) {
        MXS_TRY(mxs::copy_rows(a.weight, 2 * a.ldw, pl.w, 2 * pl.ldk, a.vocab, 2 * a.d, a.sms, a.st));
        w = pl.w, ldw = pl.ldk;
    }
    int rc = pack_rows<T>(a, pl, lse, grad, gw != nullptr);
    if (rc) return rc;
    ProductOp<T> prod{};
    prod.format = format_of<T>();
    prod.drop = mxs::test_drop_tile();
    prod.status = a.status;
    prod.head = pl.head;
    prod.d = (int)a.d;
    prod.n = pl.dn;
    prod.nt = pl.dnt;
    prod.split_width = (int)std::min(pl.piece, a.vocab);
    prod.acc = pl.acc;
    prod.counts = pl.counts;
    prod.rest = pl.rest;
    prod.sums = pl.sums;
    prod.runs = pl.runs;
    prod.listed = pl.listed;
    prod.target = pl.target;
    prod.lds = pl.lds;
    prod.h = static_cast<const T*>(pl.packed);
    prod.ldh = pl.ldk;
    prod.want_h = gh != nullptr;
    prod.want_w = gw != nullptr;
    prod.dw = static_cast<T*>(gw);
    prod.lddw = ldgw;
    prod.scale = (float)(1.0 / a.temperature / (format_of<T>() == 0 ? 16384.0 : 1.0));
    prod.vec = mxs::aligned16(gw, 2 * ldgw);
    if (!mxs::gemm::make_map(&prod.w_n, w, 2, a.d, a.vocab, ldw, 64) ||
        !mxs::gemm::make_map(&prod.h_n, pl.packed, 2, a.d, round_up(a.rows, PACK_ROWS), pl.ldk, 64))
        return MXS_ERR_CUDA;
    for (int64_t v0 = 0; v0 < a.vocab; v0 += pl.piece) {
        rc = a.rows > 128 ? grad_piece<2, T>(a, pl, w, ldw, v0, prod) : grad_piece<1, T>(a, pl, w, ldw, v0, prod);
        if (rc) return rc;
    }
    for (int64_t r = 0; gh && r < a.rows; r += 65535) {  // as many rows as a grid counts
        const dim3 grid((unsigned)ceil_div(a.d, 512), (unsigned)std::min<int64_t>(65535, a.rows - r));
        MXS_TRY(launch_dependent(grad_hidden_out_kernel<T>, grid, 128, a.st, pl.acc, pl.pos + r, pl.head, pl.target,
                                 pl.rest, static_cast<const T*>(w), ldw, (int)a.d, pl.dn, prod.split_width, a.sms / 2,
                                 prod.want_w, prod.scale, static_cast<T*>(gh) + r * ldgh, ldgh));
    }
    return MXS_OK;
}

}  // namespace

extern "C" {

int mxs_ce_workspace_size(const void* d_weight, int64_t ld_weight, int64_t rows, int64_t d_model, int64_t vocab,
                          int backward, size_t* bytes) {
    if (!bytes || rows < 0 || d_model <= 0 || vocab <= 0 || ld_weight < d_model || rows > MAX_DIM ||
        d_model > MAX_DIM || vocab > MAX_DIM || (backward && rows > MAX_BACKWARD_ROWS))
        return MXS_ERR_INVALID;
    int sms = 0;
    uint32_t* status = nullptr;
    const int rc = mxs::device_info(&sms, &status);
    if (rc) return rc;
    *bytes = make_plan(nullptr, sms, d_weight, ld_weight, rows, d_model, vocab, backward != 0).bytes;
    return MXS_OK;
}

int mxs_ce_from_hidden(const void* d_hidden, int64_t ld_hidden, const void* d_weight, int64_t ld_weight, int dtype,
                       int64_t rows, int64_t d_model, int64_t vocab, const void* d_targets, int target_bytes,
                       double temperature, float* d_loss, float* d_lse, void* d_workspace, size_t workspace_bytes,
                       void* stream) {
    if (bad_shape(ld_hidden, ld_weight, dtype, rows, d_model, vocab, target_bytes, temperature)) return MXS_ERR_INVALID;
    if (rows == 0) return MXS_OK;
    if (!d_hidden || !d_weight || !d_targets) return MXS_ERR_INVALID;
    Call a{d_hidden, ld_hidden, d_weight, ld_weight, rows, d_model, vocab,
           Targets{d_targets, target_bytes, (int)vocab}, temperature, 0, nullptr, static_cast<cudaStream_t>(stream)};
    const int rc = mxs::device_info(&a.sms, &a.status);
    if (rc) return rc;
    const Plan pl = make_plan(d_workspace, a.sms, d_weight, ld_weight, rows, d_model, vocab, false);
    if (!mxs::workspace_ok(d_workspace, workspace_bytes, pl.bytes)) return MXS_ERR_WORKSPACE;
    return dtype == MXS_BF16 ? forward<__nv_bfloat16>(a, pl, d_loss, d_lse) : forward<__half>(a, pl, d_loss, d_lse);
}

int mxs_ce_from_hidden_backward(const void* d_hidden, int64_t ld_hidden, const void* d_weight, int64_t ld_weight,
                                int dtype, int64_t rows, int64_t d_model, int64_t vocab, const void* d_targets,
                                int target_bytes, double temperature, const float* d_lse, const float* d_grad_loss,
                                void* d_grad_hidden, int64_t ld_grad_hidden, void* d_grad_weight,
                                int64_t ld_grad_weight, void* d_workspace, size_t workspace_bytes, void* stream) {
    if (bad_shape(ld_hidden, ld_weight, dtype, rows, d_model, vocab, target_bytes, temperature) ||
        rows > MAX_BACKWARD_ROWS || (d_grad_hidden && ld_grad_hidden < d_model) ||
        (d_grad_weight && ld_grad_weight < d_model))
        return MXS_ERR_INVALID;
    if (!d_grad_hidden && !d_grad_weight) return MXS_OK;
    Call a{d_hidden, ld_hidden, d_weight, ld_weight, rows, d_model, vocab,
           Targets{d_targets, target_bytes, (int)vocab}, temperature, 0, nullptr, static_cast<cudaStream_t>(stream)};
    if (rows == 0) {  // no row: the weight's gradient is zero
        if (d_grad_weight)
            MXS_TRY(cudaMemset2DAsync(d_grad_weight, 2 * ld_grad_weight, 0, 2 * d_model, vocab, a.st));
        return MXS_OK;
    }
    if (!d_hidden || !d_weight || !d_targets || !d_lse || !d_grad_loss) return MXS_ERR_INVALID;
    const int rc = mxs::device_info(&a.sms, &a.status);
    if (rc) return rc;
    const Plan pl = make_plan(d_workspace, a.sms, d_weight, ld_weight, rows, d_model, vocab, true);
    if (!mxs::workspace_ok(d_workspace, workspace_bytes, pl.bytes)) return MXS_ERR_WORKSPACE;
    return dtype == MXS_BF16
               ? backward<__nv_bfloat16>(a, pl, d_lse, d_grad_loss, d_grad_hidden, ld_grad_hidden, d_grad_weight,
                                         ld_grad_weight)
               : backward<__half>(a, pl, d_lse, d_grad_loss, d_grad_hidden, ld_grad_hidden, d_grad_weight,
                                  ld_grad_weight);
}

}  // extern "C"
