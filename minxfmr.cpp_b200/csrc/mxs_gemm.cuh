// The tensor-core frame of the output-head operators: a persistent,
// warp-specialised sm_100a kernel body that an Op fills in.
//
//   warp 0      loads operand tiles (TMA, 128-byte swizzle) into a ring of stages
//   warp 1      issues tcgen05.mma (one thread), accumulators in TMEM
//   warp 2      what an Op wants done beside it all, if anything
//   warps 4..   (Op::EPI of them, 8 or 16) read accumulators back (tcgen05.ld) and do
//               the Op's epilogue: EPI / 4 warps share the 32 rows that the hardware
//               gives a warp's place, each taking every (EPI / 4)-th run of 32 columns
//
// Warps 0..3 give up registers for the epilogue's (setmaxnreg). With 16 epilogue
// warps: 640 threads x 96 at launch = 128 x 64 + 512 x 104; with 8: 384 x 168 =
// 128 x 56 + 256 x 224. Sixteen suit epilogues with many instructions, eight the
// 8-bit product, which keeps 128 sums a thread beside the 32 values it has just read
// (a read of the accumulator is waited for before the next one is issued).
//
// A tile is 128 rows per CTA by up to 256 columns. With CG = 2 a pair of CTAs
// works on one 256-row tile: each loads its 128 rows of A and half of B's
// columns, the even CTA issues the pair's MMAs, and every operand byte crosses
// L2 -> shared memory once for 256 x 256 outputs (64 bytes per clock and SM at
// full MMA rate, against 96 for a single CTA's 128 x 256, which L2 does not
// deliver). TMEM's 512 columns hold two accumulators of 256 columns, four of 128
// or eight of 64, so the epilogue of one runs under the products of the next.
//
// Operands are held with 128 bytes of the contiguous direction per row, either
// along K ("K-major": 64 16-bit or 128 8-bit values of K in a row) or along the
// tile's own direction ("MN-major": 64 values of M or N in a row, one row per k),
// so all three products of a loss and its gradients read the same row-major
// matrices without a transposed copy.
//
// Every wait is bounded (about 1 s, as in the streaming kernel), the epilogue warps'
// for one another too; a wait that gives up marks the CTA dead, its roles stop, copies and MMAs in flight are
// waited for (bounded again), TMEM is freed, and the device's status word gets
// FLAG_TIMEOUT. No TMA multicast anywhere.
#pragma once
#include <atomic>

#include <cuda.h>

#include "mxs_common.cuh"
#include "mxs_head.cuh"

namespace mxs {
namespace gemm {

constexpr int EPI_WARP0 = 4;
constexpr int MAX_ACC = 8;  // accumulators that TMEM holds at most
constexpr int XPOSE_ALL = 32768;  // shared memory for the epilogue warps' transposes
constexpr int A_BYTES = 128 * 128;
constexpr int ROW = 128;  // bytes of a stage row (one swizzle row)

template <typename Op>
struct Geo {
    static constexpr int CG = Op::CG, THREADS = 32 * (EPI_WARP0 + Op::EPI);
    static constexpr int XPOSE = XPOSE_ALL / Op::EPI;  // of one warp: 2 or 4 KB
    static constexpr int B_BYTES = 256 / CG * ROW;
    static constexpr int STAGE = A_BYTES + B_BYTES;
    static constexpr int STAGES = 196608 / STAGE;  // 192 KB: 4 or 6
    static constexpr size_t SMEM = 1024 + (size_t)STAGES * STAGE + XPOSE_ALL + 512;
};

struct Tile {
    int m0, n0;   // first row and column of the pair's (or CTA's) tile, in the Op's own terms
    int k0, kn;   // first k block and number of blocks
    int n;        // columns of the MMA
    int kind;     // Op's own
};

// An epilogue thread's place.
struct Lane {
    int lane, quad, grp;  // quad: which 32 rows of the CTA's 128; grp: which column group
    int row;              // of the pair's tile
    uint8_t* xpose;       // its warp's bytes for transposes
    int meetings, gatherings;  // how often the warps of this quad, and all of the CTA's, have met
};

struct Ring {
    uint64_t full[6], empty[6], tfull[MAX_ACC], tempty[MAX_ACC], drain;
    uint64_t meet[5];  // of each quad's warps, and of all epilogue warps, where an Op has them meet
    uint32_t tmem;
    int dead;
};

// --- PTX ---------------------------------------------------------------------

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\n barrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
// True in one thread of a converged warp, the same one every time.
__device__ __forceinline__ bool elect() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_launch_dependents() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// 2-D tile load; `bar` is a shared::cluster address (with CG = 2, the even CTA's barrier).
template <int CG>
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    if (CG == 2)
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t* slot) {
    if (CG == 2)
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(slot))
                     : "memory");
    else
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(slot))
                     : "memory");
}
template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t base) {
    if (CG == 2) {
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(base));
    } else {
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(base));
    }
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Arrives on `bar` (of both CTAs of the pair) when every MMA issued so far has finished.
template <int CG>
__device__ __forceinline__ void commit(uint64_t* bar) {
    if (CG == 2)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                smem_u32(bar)), "h"((uint16_t)3) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                     : "memory");
}

template <int CG, bool F8>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    const uint32_t p = add;
    if (F8) {
        if (CG == 2)
            asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
                         " tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b),
                         "r"(idesc), "r"(p) : "memory");
        else
            asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
                         " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b),
                         "r"(idesc), "r"(p) : "memory");
    } else {
        if (CG == 2)
            asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
                         " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b),
                         "r"(idesc), "r"(p) : "memory");
        else
            asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
                         " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b),
                         "r"(idesc), "r"(p) : "memory");
    }
}

// 32 accumulator columns of this warp's 32 lanes.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
        "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
        " tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_ld(uint32_t addr, float (&v)[32]) { tmem_ld32(addr, v); }
__device__ __forceinline__ void tmem_ld(uint32_t addr, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15},"
        " [%16];\n tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// Whether the unrolled j is the value h, kept as a comparison (the compiler would
// turn the run of them into an index, and the array into local memory).
__device__ __forceinline__ bool is_column(int h, int j) {
    int d = h - j;
    asm("" : "+r"(d));
    return d == 0;
}

// A warp's 32 x 32 values (a row a thread) to row-major memory, through its share
// of shared memory, LINE bytes of a row at a time (64 or 128: 32 rows of it must
// fit): a store from the threads' own rows touches 32 lines for 16 bytes each, one
// from here 4 or 8 lines. `out` is the place of row 0, column 0; `rows` and `cols`
// say how many of the 32 exist; `vec` that rows start on 16-byte boundaries. ADD
// adds to what is there.
template <typename T, bool ADD, int LINE = 64>
__device__ __forceinline__ void store_rows(T* out, int64_t ld, const float (&v)[32], int rows, int cols, bool vec,
                                           const Lane& me) {
    constexpr int EACH = 16 / sizeof(T);                  // values of a 16-byte piece
    constexpr int W = LINE / (int)sizeof(T);              // values of a line
    constexpr int PIECES = LINE / 16, SHIFT = LINE == 64 ? 1 : 0;  // a row's pieces, in an order of its own:
    const int l = me.lane;                                // neighbouring rows' fall into different banks
    auto slot = [&](int r, int p) { return me.xpose + r * LINE + ((p ^ (r >> SHIFT)) & (PIECES - 1)) * 16; };
#pragma unroll
    for (int c0 = 0; c0 < 32; c0 += W) {
        __syncwarp();
#pragma unroll
        for (int p = 0; p < PIECES; ++p) *reinterpret_cast<uint4*>(slot(l, p)) = pack16<T>(v + c0 + p * EACH);
        __syncwarp();
        if (vec && cols >= c0 + W) {
            constexpr int STEP = 32 / PIECES;  // rows of one store
            uint4 u[PIECES];
#pragma unroll
            for (int p = 0; p < PIECES; ++p)
                u[p] = *reinterpret_cast<const uint4*>(slot(p * STEP + l / PIECES, l % PIECES));
#pragma unroll
            for (int p = 0; p < PIECES; ++p) {
                const int r = p * STEP + l / PIECES;
                if (r >= rows) continue;
                uint4* to = reinterpret_cast<uint4*>(out + (int64_t)r * ld + c0 + (l % PIECES) * EACH);
                if (ADD) {
                    const uint4 o = *to;
                    u[p].x = __float_as_uint(__uint_as_float(u[p].x) + __uint_as_float(o.x));
                    u[p].y = __float_as_uint(__uint_as_float(u[p].y) + __uint_as_float(o.y));
                    u[p].z = __float_as_uint(__uint_as_float(u[p].z) + __uint_as_float(o.z));
                    u[p].w = __float_as_uint(__uint_as_float(u[p].w) + __uint_as_float(o.w));
                }
                *to = u[p];
            }
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const int r = i * (32 / W) + l / W, c = l % W;
                if (r < rows && c0 + c < cols)
                    out[(int64_t)r * ld + c0 + c] = reinterpret_cast<const T*>(slot(r, c / EACH))[c % EACH];
            }
        }
    }
}

// Shared-memory matrix descriptor, 128-byte swizzle: start address, leading and
// stride byte offsets (all in 16-byte units), descriptor version 1.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead, uint32_t stride) {
    return (uint64_t)((addr & 0x3ffff) >> 4) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(stride >> 4) << 32 |
           1ull << 46 | 2ull << 61;
}

// Instruction descriptor: fp32 accumulators, operand formats, majors, shape.
// Formats: kind::f16 0 = f16, 1 = bf16; kind::f8f6f4 0 = e4m3.
__device__ __forceinline__ uint32_t instr_desc(int format, bool a_mn, bool b_mn, int m, int n) {
    return 1u << 4 | (uint32_t)format << 7 | (uint32_t)format << 10 | (uint32_t)a_mn << 15 | (uint32_t)b_mn << 16 |
           (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;
}

// --- waits -------------------------------------------------------------------

// False (and the CTA is dead) when the limit ran out or another role gave up. The
// clock is read after 32 polls only: it is a slow read next to a wait of a few
// hundred clocks, and there are several of those for every block of the ring.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, Ring* ring) {
    for (int i = 0; i < 32; ++i)
        if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait(bar, parity)) {
        if (*(volatile int*)&ring->dead) return false;
        if (globaltimer_ns() - t0 > 1000000000ull) {
            *(volatile int*)&ring->dead = 1;
            return false;
        }
    }
    return true;
}
// An accumulator's readers tell the MMA thread of the pair. What they hand over
// is TMEM, ordered by the tcgen05 fences; no memory is published, so the arrival
// is relaxed (a release for the cluster waits for every load and store in flight:
// 1000 to 2000 clocks for each block of the 8-bit product).
__device__ __forceinline__ void arrive(uint32_t addr, bool remote) {
    if (remote)
        asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
    else
        asm volatile("mbarrier.arrive.relaxed.cta.shared::cta.b64 _, [%0];" ::"r"(addr) : "memory");
}

// What an Op needs to know of where it runs.
struct Ctx {
    int units, unit;   // CTAs or pairs in the grid, and this one
    uint32_t rank;     // CTA's place in its pair
    int kept;          // Op's row count, read on the device
    Ring* ring;
};

// Warps meet: what each wrote to memory before is there for all after. False when one of
// them has given up.
__device__ __forceinline__ bool meet_at(uint64_t* bar, int& times, const Lane& me, const Ctx& x) {
    __syncwarp();
    if (me.lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
    return __all_sync(0xffffffffu, wait(bar, times++ & 1, x.ring));
}
__device__ __forceinline__ bool meet(Lane& me, const Ctx& x) {  // of a quad
    return meet_at(&x.ring->meet[me.quad], me.meetings, me, x);
}
__device__ __forceinline__ bool gather(Lane& me, const Ctx& x) {  // all epilogue warps of the CTA
    return meet_at(&x.ring->meet[4], me.gatherings, me, x);
}

// The kernel body. Op (a __grid_constant__ parameter) has
//   SWAP                   compile-time, CG 1: not 0 where the second operand's rows lie along TMEM's
//                          lanes (128 at a time, two runs to an accumulator) and SWAP rows of the first
//                          along its columns: for few rows, whose 128 would be mostly padding
//   CG, F8, PROMOTE, EPI   compile-time: CTAs per tile, 8-bit operands, join accumulators in registers,
//                          epilogue warps
//   format                 operand format of the instruction descriptor
//   drop                   test hook: CTA 0's producer stops before this block (-1: off); below -1
//                          CTA 0's first epilogue warp leaves before its tile -2 - drop
//   n                      columns of a tile at most
//   status                 the device's status word
//   prefetch()             tensor-map prefetch
//   kept()                 the row count
//   tile(i, ctx, tile)     i-th tile of this unit, false when there is none
//   a_mn(t), b_mn(t)       operand majors of a tile
//   bytes(t)               bytes this CTA loads per block
//   load(t, kb, sa, sb, bar, ctx)
//   ASIDE, aside(ctx, lane)                             whether warp 2 has something to do, and what
//   zero(t, me, ctx)                                    the epilogue of a tile without blocks
//   group()                blocks after which an accumulator is read back
//   ahead(t, me, ctx), epilogue(t, tmem, me, ctx, it, kb)  !PROMOTE: kb, the first block of what the
//                          accumulator holds; `it` is what ahead gave, before the tile's first was
//                          waited for; it.ok is false where its warps did not meet
//   Acc, begin(...), prepare(...), join(...), finish(...)  PROMOTE: the accumulators of a tile are
//                          joined in registers; finish says false where its warps did not meet
template <typename Op>
__device__ __forceinline__ void run(const Op& op) {
    constexpr int CG = Op::CG;
    using G = Geo<Op>;
    extern __shared__ uint8_t raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* xpose = base + (size_t)G::STAGES * G::STAGE;
    Ring* ring = reinterpret_cast<Ring*>(xpose + XPOSE_ALL);
    const uint32_t stages = smem_u32(base);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Ctx ctx;
    ctx.rank = CG == 2 ? cluster_rank() : 0;
    ctx.units = gridDim.x / CG;
    ctx.unit = blockIdx.x / CG;
    ctx.ring = ring;
    if (threadIdx.x == 0) {
        for (int i = 0; i < G::STAGES; ++i) {
            mbar_init(&ring->full[i], 1);
            mbar_init(&ring->empty[i], 1);
        }
        for (int i = 0; i < MAX_ACC; ++i) {
            mbar_init(&ring->tfull[i], 1);
            mbar_init(&ring->tempty[i], Op::EPI * CG);
        }
        mbar_init(&ring->drain, 1);
        for (int i = 0; i < 5; ++i) mbar_init(&ring->meet[i], i < 4 ? Op::EPI / 4 : Op::EPI);
        ring->dead = 0;
        fence_mbar_init();
        op.prefetch();
    }
    if (warp == 1) tmem_alloc<CG>(&ring->tmem);
    fence_before();
    __syncthreads();
    if (CG == 2) cluster_sync();
    fence_after();
    const uint32_t tmem = *(volatile uint32_t*)&ring->tmem;
    grid_wait();
    grid_launch_dependents();
    ctx.kept = op.kept();

    Tile t;
    const uint32_t acc_cols = Op::SWAP ? 2 * Op::SWAP : op.n <= 64 ? 64 : op.n <= 128 ? 128 : 256;
    const uint32_t accs = min(512 / acc_cols, (uint32_t)MAX_ACC);
    if (warp < EPI_WARP0) {
        if constexpr (Op::EPI == 16)
            asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        else
            asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        // Both roles run as whole warps with one elected thread at the loads and MMAs:
        // addresses and descriptors then stay in uniform registers, which those
        // instructions want (from a single-thread branch a block's four MMAs took
        // 670 clocks to issue, more than the 512 that they run).
        if (warp == 0) {
            uint32_t s = 0, ph = 0;
            int64_t issued = 0;
            bool ok = true;
            for (int i = 0; ok && op.tile(i, ctx, t); ++i) {
                const uint32_t bytes = CG * op.bytes(t);
                for (int kb = 0; kb < t.kn; ++kb) {
                    ok = wait(&ring->empty[s], ph ^ 1, ring) && !(op.drop >= 0 && blockIdx.x == 0 && issued >= op.drop);
                    if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                    if (elect()) {
                        uint32_t bar = smem_u32(&ring->full[s]);
                        if (ctx.rank == 0) mbar_arrive_expect_tx(&ring->full[s], bytes);
                        if (CG == 2) bar = map_to_rank(bar, 0);
                        const uint32_t sa = stages + s * G::STAGE;
                        op.load(t, t.k0 + kb, sa, sa + A_BYTES, bar, ctx);
                    }
                    __syncwarp();
                    ++issued;
                    if (++s == G::STAGES) s = 0, ph ^= 1;
                }
            }
            // What the last blocks (at most one per stage) still send to this CTA's barriers lands
            // before the CTA ends: the MMAs' hand-backs of their stages, which the pair's even CTA
            // sends to both, or, after a give-up, the copies and the even CTA's word that its MMAs
            // have finished.
            const int64_t last = issued < G::STAGES ? issued : (int64_t)G::STAGES;
            for (int64_t j = issued - last; ok && j < issued; ++j)
                ok = __all_sync(0xffffffffu, wait(&ring->empty[j % G::STAGES], (uint32_t)(j / G::STAGES) & 1, ring));
            if (!ok && ctx.rank == 0)
                for (int64_t j = issued - last; j < issued; ++j)
                    mbar_wait_bounded(&ring->full[j % G::STAGES], (uint32_t)(j / G::STAGES) & 1);
            else if (!ok)
                mbar_wait_bounded(&ring->drain, 0);
        } else if (warp == 1 && ctx.rank == 0) {
            uint32_t s = 0, ph = 0, buf = 0, tph = 0;
            bool ok = true;
            for (int i = 0; ok && op.tile(i, ctx, t); ++i) {
                const bool amn = op.a_mn(t), bmn = op.b_mn(t);
                const uint32_t idesc = instr_desc(op.format, amn, bmn, 128 * CG, Op::SWAP ? Op::SWAP : t.n);
                // K-major: 8-row groups 1024 bytes apart, a step of K is 32 bytes of the row.
                // MN-major: 64-wide slabs of 64 k rows (8192 bytes), 8-k groups 1024 bytes
                // apart, a step of 16 k rows is 2048 bytes.
                const uint64_t step_a = (amn ? 2048 : 32) >> 4, step_b = (bmn ? 2048 : 32) >> 4;
                const uint64_t da0 = smem_desc(stages, amn ? 8192 : 16, 1024);
                const uint64_t db0 = smem_desc(stages + A_BYTES, bmn ? 8192 : 16, 1024);
                const int group = op.group() < t.kn ? op.group() : t.kn;
                int in = 0;  // block of its group
                for (int kb = 0; kb < t.kn; ++kb) {
                    // What comes last is waited for last, since a wait costs 100 clocks even where it
                    // has nothing to wait for: a pair's operands are there long before an accumulator
                    // comes free, up to 128 rows' (CG 1) are what memory is read for.
                    if (CG == 1)
                        ok = (in > 0 || wait(&ring->tempty[buf], tph ^ 1, ring)) && wait(&ring->full[s], ph, ring);
                    else
                        ok = wait(&ring->full[s], ph, ring) && (in > 0 || wait(&ring->tempty[buf], tph ^ 1, ring));
                    if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                    fence_after();
                    const bool last = in + 1 == group || kb == t.kn - 1;
                    if (elect()) {
                        const uint64_t at = s * (G::STAGE >> 4), da = da0 + at, db = db0 + at;
                        const uint32_t d = tmem + buf * acc_cols;
                        if (Op::SWAP) {
                            for (int h = 0; h * 128 < t.n; ++h)
#pragma unroll
                                for (int k = 0; k < 4; ++k)
                                    mma<CG, Op::F8>(d + h * Op::SWAP, db + h * (128 * ROW >> 4) + k * step_b,
                                                    da + k * step_a, idesc, k > 0 || in > 0);
                        } else {
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                mma<CG, Op::F8>(d, da + k * step_a, db + k * step_b, idesc, k > 0 || in > 0);
                        }
                        commit<CG>(&ring->empty[s]);
                        if (last) commit<CG>(&ring->tfull[buf]);
                    }
                    __syncwarp();
                    ++in;
                    if (++s == G::STAGES) s = 0, ph ^= 1;
                    if (last) {
                        in = 0;
                        if (++buf == accs) buf = 0, tph ^= 1;
                    }
                }
            }
            if (!ok) {  // MMAs in flight finish before TMEM is freed
                if (elect()) commit<CG>(&ring->drain);
                __syncwarp();
                mbar_wait_bounded(&ring->drain, 0);
            }
        } else if (Op::ASIDE && warp == 2) {
            if constexpr (Op::ASIDE) op.aside(ctx, lane);
        }
    } else {
        if constexpr (Op::EPI == 16)
            asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
        else
            asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        Lane me;
        me.lane = lane;
        me.quad = warp & 3;
        me.grp = (warp - EPI_WARP0) >> 2;
        me.row = (int)ctx.rank * 128 + me.quad * 32 + lane;
        me.xpose = xpose + (warp - EPI_WARP0) * G::XPOSE;
        me.meetings = me.gatherings = 0;
        const uint32_t lanes = (uint32_t)(me.quad * 32) << 16;
        const bool remote = CG == 2 && ctx.rank != 0;
        const uint32_t te0 = remote ? map_to_rank(smem_u32(&ring->tempty[0]), 0) : smem_u32(&ring->tempty[0]);
        uint32_t buf = 0, tph = 0;
        bool ok = true;
        for (int i = 0; ok && op.tile(i, ctx, t); ++i) {
            if (op.drop < -1 && blockIdx.x == 0 && warp == EPI_WARP0 && i == -2 - op.drop) break;
            if (t.kn == 0) {  // an empty sum: no product, no accumulator
                op.zero(t, me, ctx);
                continue;
            }
            if constexpr (Op::PROMOTE) {
                typename Op::Acc acc;
                op.begin(acc, t, me, ctx);
                for (int kb = 0; kb < t.kn; kb += op.group()) {
                    op.prepare(acc, t, t.k0 + kb, me, ctx);
                    ok = __all_sync(0xffffffffu, wait(&ring->tfull[buf], tph, ring));
                    if (!ok) break;
                    fence_after();
                    // the accumulator goes back to the MMAs as soon as it has been read
                    op.join(acc, t, tmem + buf * acc_cols + lanes, me, ctx, [&] {
                        fence_before();
                        __syncwarp();
                        if (lane == 0) arrive(te0 + buf * 8, remote);
                    });
                    if (++buf == accs) buf = 0, tph ^= 1;
                }
                if (ok) ok = op.finish(acc, t, me, ctx);
            } else {
                const auto it = op.ahead(t, me, ctx);
                ok = it.ok;
                for (int kb = 0; ok && kb < t.kn; kb += min(op.group(), t.kn)) {
                    ok = __all_sync(0xffffffffu, wait(&ring->tfull[buf], tph, ring));
                    if (!ok) break;
                    fence_after();
                    op.epilogue(t, tmem + buf * acc_cols + lanes, me, ctx, it, kb);
                    fence_before();
                    __syncwarp();
                    if (lane == 0) arrive(te0 + buf * 8, remote);
                    if (++buf == accs) buf = 0, tph ^= 1;
                }
            }
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    if (CG == 2) cluster_sync();
    fence_after();
    if (warp == 1) tmem_free<CG>(tmem);
    if (threadIdx.x == 0 && ring->dead) atomicOr(op.status, FLAG_TIMEOUT);
}

// --- host --------------------------------------------------------------------

// A row-major [rows][cols] matrix of 1- or 2-byte elements, read in boxes of
// 128 bytes by box_rows rows, 128-byte swizzle; what lies outside reads zero.
// False when the encoder is missing or refuses.
bool make_map(CUtensorMap* map, const void* base, int elem_bytes, int64_t cols, int64_t rows, int64_t ld, int box_rows);

template <typename Op>
__global__ void __launch_bounds__(Geo<Op>::THREADS, 1) kernel(const __grid_constant__ Op op) {
    run(op);
}

// Launches the Op on units * CG CTAs, allowed to start while the kernel before it
// on the stream drains (it waits on the device).
template <typename Op>
cudaError_t launch(const Op& op, int units, cudaStream_t st) {
    constexpr int CG = Op::CG;
    static std::atomic<uint64_t> configured{0};  // a bit for each device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (!(configured.load(std::memory_order_relaxed) >> dev & 1)) {
        e = cudaFuncSetAttribute(kernel<Op>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Geo<Op>::SMEM);
        if (e != cudaSuccess) return e;
        configured.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(units * CG);
    cfg.blockDim = dim3(Geo<Op>::THREADS);
    cfg.dynamicSmemBytes = Geo<Op>::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = CG;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel<Op>, op);
}

}  // namespace gemm
}  // namespace mxs
