// grouped.cu -- matrix products grouped by expert with ragged sizes, on the
// tcgen05 tensor cores.
//
// Rows of x are sorted by expert; offsets[e] .. offsets[e + 1] (on the
// device) are expert e's.
//   forward       y[t][n]     = sum_k x[t][k] w[e(t)][n][k]      (16-bit, or
//                               e4m3 times x_scale[t] w_scale[e][n])
//   token grad    dx[t][k]    = sum_n dy[t][n] w[e(t)][n][k]: the forward
//                               product with w's two dimensions exchanged
//   weight grad   dw[e][n][k] = sum_{t of e} dy[t][n] x[t][k]
//
// One persistent kernel does all three.  A CTA pair (cta_group::2) computes
// a tile of 256 features x up to 256 rows; the features -- the contiguous
// dimension of the result -- are the instruction's M side, the rows its N
// side, because N is a run-time number: an expert's last tile is an
// instruction of 32, 64, ... 256 rows, so ragged ends cost what they hold
// (rounded to 32) and a few decoded tokens do not pay for 128 rows.
// The accumulator then has features along TMEM's lanes and rows along its
// columns, the other way round than the result: the storing warps read it in
// the shape of 8 x 8 fragments, round pairs to 16 bits, and stmatrix.trans
// turns the fragments on the way into shared memory, from where 16 rows of 64
// bytes go out as one tensor store, or, at an expert's end, row by row.
// (One 2-byte store per element, straight from a lane per feature, took
// longer than the multiplication: 17800 clocks a tile.  Weight gradient of
// 8192 rows over 16 experts, 4096 x 2048, with this and with the waits and
// tails below: 259 -> 146 us.)
//
//   warp 0     TMA producer (both CTAs): k-blocks of 128 bytes, 128 features
//              and half the rows per CTA, into a ring of stages; completion
//              counted on the leader's barrier
//   warp 1     allocates TMEM; the leader's lane 0 issues the MMAs into one
//              of two 256-column accumulators
//   warps 2-9  read the other accumulator, scale, round once and store
//   warp 10    weight gradient only: clears the rows of other experts
//
// No host synchronisation: every CTA reads the offsets and walks the same
// list of tiles, in rounds of one tile per pair.  Offsets are clamped to [0,
// rows] and to ascending order, so that bad ones cannot reach memory outside
// the operands.  Tiles at an expert's end are cheaper than whole ones, and
// they come back at regular distances in the list; a pair that always took
// the same place of a round would meet them in every other round or never
// (16384 rows over 16 experts, 4096 x 4096: 496 us against 400 with even
// experts).  So the places rotate by the golden section from round to round.
//
// Weight gradient: the contraction runs over an expert's rows, and its last
// k-block of 64 may hold rows of the next expert.  Those must not be
// multiplied (0 * NaN): whole instructions of 16 are left out, and where the
// last one holds other rows, the stage's copies complete on barriers of
// their own, where warp 10 of both CTAs clears the up to 15 rows before the
// stage is released to the MMA.  (The producer doing this itself waits for
// the copies once per tile: 213 us for the gradient above; clearing the whole
// rest of the block, against the tensor core's own reads of shared memory,
// took 1400 clocks.)  An expert without rows gets zeros.
//
// The accumulator is 32 bits wide in TMEM over the whole contraction.
//
// Every wait is bounded by a wall-clock deadline, as in the graph GEMMs: a
// role that runs out raises the CTA's abort flag and the device's error
// word, every role leaves its loop, copies and MMAs in flight are drained
// (bounded again), TMEM is freed and the kernel returns.
#include "common.cuh"
#include "tc_launch.h"

#include "bafe_dev.cuh"
#include "gemm_tc.cuh"

#include <cuda.h>

#include <cstdlib>
#include <cstring>

namespace bafe_cuda {
namespace lm {
namespace {

using bafe::TmaDesc;
typedef unsigned int u32;
typedef unsigned long long u64;

constexpr int TILE_F = 256;            // features per pair
constexpr int TILE_R = 256;            // rows per tile, at most
constexpr int THREADS = 320;           // and a warp more for the weight gradient
constexpr u32 A_BYTES = 16384;
constexpr u32 MN_BOX = 8192;           // 64 features x 64 of the contraction, 16-bit
constexpr int MAX_EXPERTS = 1024;
constexpr u32 BAR_BYTES = 512;
constexpr u32 OFFSET_BYTES = 2 * 4 * (MAX_EXPERTS + 2) + 496;     // keeps the staging 512-byte aligned (its swizzle's period)
constexpr u32 STAGING_BYTES = 2048;    // per storing warp: two times 16 rows x 32 features, 16-bit
// The ring for calls of up to ROWS rows.  What a pair has on its way divided
// by the memory's latency is what it can read; with few rows the weights are
// all of it, so the rows' share of a stage becomes more stages.  A k-block's
// four small products take less time than the barriers around them, so a
// stage of these calls is two k-blocks.  (8 rows of 4 experts: 4096 features
// x 4096 29.7 -> 27.6 us, 2048 x 4096 24.5 -> 18.8, with a ring of 6 whole
// stages and one k-block each before.)
template <int ROWS> struct Ring {
    static constexpr int KPS = ROWS == 256 ? 1 : 2;                    // k-blocks per stage
    static constexpr u32 B_BYTES = ROWS / 2 * 128, STAGE_BYTES = KPS * (A_BYTES + B_BYTES);
    static constexpr int STAGES = ROWS == 256 ? 6 : ROWS == 128 ? 4 : 5;
    static constexpr int SMEM_BYTES = 1024 + STAGES * (int)STAGE_BYTES + (int)BAR_BYTES + (int)OFFSET_BYTES + 8 * (int)STAGING_BYTES;
    static_assert((STAGES * STAGE_BYTES + BAR_BYTES + OFFSET_BYTES) % 512 == 0, "staging alignment");
    static_assert(SMEM_BYTES <= 227 * 1024, "shared memory");
};

struct GroupedArgs {
    TmaDesc a;                         // features: 3-D (.., .., expert)
    TmaDesc b;                         // rows, 128 at a time
    TmaDesc b_part[3];                 // rows, 64, 32 and 16 at a time
    TmaDesc c;                         // result, 16 rows x 32 features (with vec_out)
    const int* offsets;                // [experts + 1]
    void* out;
    const float* x_scale;              // [rows], or null
    const float* w_scale;              // [experts][features], or null
    int64_t w_scale_ld;
    int64_t out_ld, out_estride;       // estride: weight gradient
    unsigned* err;
    unsigned long long timeout_ns;
    int rows, experts;
    int features;                      // contiguous dimension of the result
    int out_rows;                      // weight gradient: rows of one expert's result
    int k;                             // contraction, in elements (forward)
    int vec_out;                       // result rows on 16-byte boundaries, features a multiple of 8: 2;
                                       // on 4-byte boundaries, features even: 1; else 0
};

struct Shared {
    u32 abort;
    u32 tmem_base;
};

__device__ __forceinline__ bool raise(volatile Shared* sh, const GroupedArgs& g, u32 code) {
    sh->abort = 1u;
    atomicCAS(g.err, 0u, code);
    return false;
}
// Bounded wait on an mbarrier phase; acquire at cluster scope where the
// peer's arrivals complete the phase.
template <bool CLUSTER>
__device__ __forceinline__ bool wait(u32 bar, u32 parity, volatile Shared* sh, const GroupedArgs& g, u32 code) {
    using namespace bafe::tc;
    auto ready = [&]() { return CLUSTER ? mbar_try_cluster(bar, parity) : mbar_try(bar, parity); };
    // The clock and the flag are looked at every 32nd time only: reading the
    // global timer takes longer than most waits.
    for (int i = 0; i < 32; ++i)
        if (ready()) return true;
    const u64 t0 = now_ns();
    while (true) {
        for (int i = 0; i < 32; ++i)
            if (ready()) return true;
        if (sh->abort) return false;
        if (now_ns() - t0 > g.timeout_ns) return raise(sh, g, code);
    }
}
__device__ __forceinline__ u64 drain_ns(const GroupedArgs& g) {
    return g.timeout_ns > 200000000ull ? g.timeout_ns : 200000000ull;
}

__device__ __forceinline__ void mma_f8_pair(u32 tmem_d, u64 adesc, u64 bdesc, u32 idesc, u32 accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, {%5, %6, %7, %8, %9, %10, %11, %12}, p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate),
          "r"(0u), "r"(0u), "r"(0u), "r"(0u), "r"(0u), "r"(0u), "r"(0u), "r"(0u) : "memory");
}

// 32 lanes x 16 consecutive 32-bit columns; the wait names the registers so
// that no use of them moves above it.
__device__ __forceinline__ void tmem_ld16(u32 taddr, u32 (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :: "memory");
}

// 16 lanes x 32 consecutive 32-bit columns as 8 x 8 fragments: registers 4 i
// + {0, 1} are lane row t / 4, columns 8 i + 2 (t % 4) + {0, 1} of thread t,
// + {2, 3} the same columns of row t / 4 + 8.
__device__ __forceinline__ void tmem_ld_16x256(u32 taddr, u32 (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait(u32 (&r)[16], u32 (&s)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(s[0]), "+r"(s[1]), "+r"(s[2]), "+r"(s[3]), "+r"(s[4]), "+r"(s[5]), "+r"(s[6]), "+r"(s[7]),
                   "+r"(s[8]), "+r"(s[9]), "+r"(s[10]), "+r"(s[11]), "+r"(s[12]), "+r"(s[13]), "+r"(s[14]), "+r"(s[15])
                 :: "memory");
}
// Four 8 x 8 matrices of 16-bit elements stored transposed; lane 8 m + k
// gives the address of row k of matrix m (16 bytes).
__device__ __forceinline__ void stmatrix_trans(u32 addr, u32 a, u32 b, u32 c, u32 d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};"
                 ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
template <class T> __device__ __forceinline__ u32 pack2(u32 lo, u32 hi);
template <> __device__ __forceinline__ u32 pack2<__nv_bfloat16>(u32 lo, u32 hi) {
    u32 r;
    asm("cvt.rn.bf16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(__uint_as_float(lo)), "f"(__uint_as_float(hi)));
    return r;
}
template <> __device__ __forceinline__ u32 pack2<__half>(u32 lo, u32 hi) {
    u32 r;
    asm("cvt.rn.f16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(__uint_as_float(lo)), "f"(__uint_as_float(hi)));
    return r;
}

enum class Mode { Rows, Weights };     // forward and token gradient; weight gradient

// Element of the operands: what the instruction reads and what is stored.
struct EBf16 { typedef __nv_bfloat16 Out; static constexpr u32 FMT = 1; static constexpr int BK = 64; static constexpr bool F8 = false; };
struct EF16 { typedef __half Out; static constexpr u32 FMT = 0; static constexpr int BK = 64; static constexpr bool F8 = false; };
struct EE4m3Bf16 { typedef __nv_bfloat16 Out; static constexpr u32 FMT = 0; static constexpr int BK = 128; static constexpr bool F8 = true; };
struct EE4m3F16 { typedef __half Out; static constexpr u32 FMT = 0; static constexpr int BK = 128; static constexpr bool F8 = true; };

// One tile of the walk.
struct Tile {
    int e, row, n, f, kblocks;         // expert; first row; rows (multiple of 32); first feature; k-blocks
    int valid;                         // rows that are stored
    int k_row, k_rows;                 // weight gradient: first row and rows of the contraction
};

template <Mode M> constexpr int ALL_THREADS = THREADS + (M == Mode::Weights ? 32 : 0);

template <class E, Mode MODE, bool A_MN, int ROWS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(ALL_THREADS<MODE>, 1) grouped_kernel(const __grid_constant__ GroupedArgs g) {
    using namespace bafe::tc;
    constexpr bool B_MN = MODE == Mode::Weights;
    constexpr int STAGES = Ring<ROWS>::STAGES, KPS = Ring<ROWS>::KPS;
    constexpr u32 B_BYTES = Ring<ROWS>::B_BYTES, STAGE_BYTES = Ring<ROWS>::STAGE_BYTES;
    static_assert(!E::F8 || (!A_MN && !B_MN), "e4m3 operands are contiguous along the contraction");
    extern __shared__ unsigned char smem_raw[];
    const u32 raw_addr = smem_u32(smem_raw);
    const u32 base = (raw_addr + 1023u) & ~1023u;
    unsigned char* smem = smem_raw + (base - raw_addr);
    const u32 bars = base + STAGES * STAGE_BYTES;
    auto FULL = [&](int s) { return bars + 8u * s; };
    auto EMPTY = [&](int s) { return bars + 8u * (STAGES + s); };
    auto TFULL = [&](int b) { return bars + 8u * (2 * STAGES + b); };
    auto TEMPTY = [&](int b) { return bars + 8u * (2 * STAGES + 2 + b); };
    const u32 DRAIN = bars + 8u * (2 * STAGES + 4);
    // Tail k-blocks, per stage (a CTA may be several tails ahead of the
    // other, but not within a stage): this CTA's copies have arrived; leader:
    // both CTAs cleared their parts.
    auto TAIL = [&](int s) { return bars + 8u * (2 * STAGES + 5 + s); };
    auto CLEARED = [&](int s) { return bars + 8u * (3 * STAGES + 5 + s); };
    static_assert(8 * (4 * STAGES + 5) + sizeof(Shared) <= BAR_BYTES, "barriers overlap the offsets");
    volatile Shared* sh = reinterpret_cast<volatile Shared*>(smem + STAGES * STAGE_BYTES + 8 * (4 * STAGES + 5));
    int* off = reinterpret_cast<int*>(smem + STAGES * STAGE_BYTES + BAR_BYTES);   // [experts + 1], clamped
    int* first = off + MAX_EXPERTS + 2;                                           // first tile of each expert, [experts + 1]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const u32 cta = cluster_rank();
    const int pair = (int)(blockIdx.x >> 1), num_pairs = (int)(gridDim.x >> 1);
    const int f_tiles = (g.features + TILE_F - 1) / TILE_F;
    const int r_tiles = MODE == Mode::Weights ? (g.out_rows + TILE_R - 1) / TILE_R : 0;

    for (int e = threadIdx.x; e <= g.experts; e += ALL_THREADS<MODE>) {
        const int v = g.offsets[e];
        off[e] = v < 0 ? 0 : v > g.rows ? g.rows : v;
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(FULL(s), 1);
            mbar_init(EMPTY(s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(TFULL(b), 1);
            mbar_init(TEMPTY(b), 16);                    // the 8 storing warps of both CTAs
        }
        mbar_init(DRAIN, 1);
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(TAIL(s), 1);
            mbar_init(CLEARED(s), 2);
        }
        sh->abort = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32((const void*)&sh->tmem_base)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    __syncthreads();
    if (warp == 0) {
        // Never below an earlier offset, whatever the array holds: the
        // experts' rows stay apart and the tiles as many as the host expects.
        int top = 0, carry = 0;
        for (int b = 0; b <= g.experts; b += 32) {
            const int e = b + lane;
            int v = e <= g.experts ? max(off[e], top) : top;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xFFFFFFFFu, v, o);
                if (lane >= o) v = max(v, u);
            }
            if (e <= g.experts) off[e] = v;
            top = __shfl_sync(0xFFFFFFFFu, v, 31);
        }
        __syncwarp();
        for (int b = 0; b < g.experts; b += 32) {
            const int e = b + lane;
            int t = 0;
            if (e < g.experts) {
                const int c = off[e + 1] - off[e];
                t = MODE == Mode::Weights ? r_tiles * f_tiles : (c + TILE_R - 1) / TILE_R * f_tiles;
            }
            int v = t;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xFFFFFFFFu, v, o);
                if (lane >= o) v += u;
            }
            if (e < g.experts) first[e] = carry + v - t;
            carry += __shfl_sync(0xFFFFFFFFu, v, 31);
        }
        if (lane == 0) first[g.experts] = carry;
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();                                      // both CTAs' barriers exist
    tc_fence_after();
    const u32 tmem = sh->tmem_base;
    const int tiles = first[g.experts];

    // This pair's tile in a round (tiles or above: none left).
    const int turn = (int)(num_pairs * 0.618f);
    auto tile_of = [&](int round) { return round * num_pairs + (int)((pair + (u32)round * turn) % num_pairs); };

    // Tile u of the walk; e only moves forward.
    auto tile_at = [&](int u, int& e) {
        while (u >= first[e + 1]) ++e;
        Tile t;
        t.e = e;
        const int local = u - first[e], c = off[e + 1] - off[e];
        t.f = local % f_tiles * TILE_F;
        if (MODE == Mode::Weights) {
            t.row = local / f_tiles * TILE_R;
            t.valid = min(TILE_R, g.out_rows - t.row);
            t.n = TILE_R;
            t.k_row = off[e];
            t.k_rows = c;
            t.kblocks = (t.k_rows + E::BK - 1) / E::BK;
        } else {
            const int r = local / f_tiles * TILE_R;
            t.row = off[e] + r;
            t.valid = min(TILE_R, c - r);
            t.n = (t.valid + 31) & ~31;
            t.k_row = t.k_rows = 0;
            t.kblocks = (g.k + KPS * E::BK - 1) / (KPS * E::BK);       // what is behind the last column is read as 0
        }
        return t;
    };

    if (warp == 0) {
        // ---------------------------------------- TMA producer (both CTAs) --
        int s = 0, e = 0;
        u32 phase = 0;
        u32 tail_phase = 0, tail_used = 0;               // a bit per stage: parity of its next tail, any so far
        bool ok = true;
        u32 armed[STAGES];
#pragma unroll
        for (int i = 0; i < STAGES; ++i) armed[i] = 0xFFFFFFFFu;
        for (int round = 0, u; lane == 0 && ok && (u = tile_of(round)) < tiles; ++round) {
            const Tile t = tile_at(u, e);
            const int fa = t.f + (int)cta * (TILE_F / 2);
            const int half = t.n / 2;
            const int rb = t.row + (int)cta * half;
            for (int kb = 0; kb < t.kblocks; ++kb) {
                if (!wait<false>(EMPTY(s), phase ^ 1u, sh, g, 1u)) { ok = false; break; }
                const u32 a_dst = base + s * STAGE_BYTES, b_dst = a_dst + KPS * A_BYTES;
                const int left = t.k_rows - kb * E::BK;
                const bool tail = MODE == Mode::Weights && left < E::BK && left % 16;
                if (tail) {
                    // the expert's last rows: see warp 10
                    mbar_expect_tx(TAIL(s), A_BYTES + B_BYTES);
                    const int y = t.k_row + kb * E::BK;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        tma_load_3d(a_dst + j * MN_BOX, &g.a, TAIL(s), fa + 64 * j, y, 0);
                        tma_load_3d(b_dst + j * MN_BOX, &g.b, TAIL(s), rb + 64 * j, y, 0);
                    }
                    tail_phase ^= 1u << s;
                    tail_used |= 1u << s;
                    armed[s] = 0xFFFFFFFFu;
                } else {
                    if (cta == 0) mbar_expect_tx(FULL(s), KPS * (2 * A_BYTES + (u32)t.n * 128u));   // both CTAs' bytes
                    if (MODE == Mode::Weights) {
                        const int y = t.k_row + kb * E::BK;
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            tma_load_3d_pair(a_dst + j * MN_BOX, &g.a, FULL(s), fa + 64 * j, y, 0);
                            tma_load_3d_pair(b_dst + j * MN_BOX, &g.b, FULL(s), rb + 64 * j, y, 0);
                        }
                    } else {
#pragma unroll
                        for (int h = 0; h < KPS; ++h) {
                            const u32 ah = a_dst + h * A_BYTES, bh = b_dst + h * B_BYTES;
                            const int kx = (kb * KPS + h) * E::BK;
                            if (A_MN) {
#pragma unroll
                                for (int j = 0; j < 2; ++j)
                                    tma_load_3d_pair(ah + j * MN_BOX, &g.a, FULL(s), fa + 64 * j, kx, t.e);
                            } else {
                                tma_load_3d_pair(ah, &g.a, FULL(s), kx, fa, t.e);
                            }
                            if (half == 128) {
                                tma_load_3d_pair(bh, &g.b, FULL(s), kx, rb, 0);
                            } else {
                                // few copies: many small ones keep the copy
                                // engine longer than the bytes do
                                int j = 0;
#pragma unroll
                                for (int i = 0; i < 3; ++i)
                                    if (half & (64 >> i)) {
                                        tma_load_3d_pair(bh + j * 128, &g.b_part[i], FULL(s), kx, rb + j, 0);
                                        j += 64 >> i;
                                    }
                            }
                        }
                    }
                    armed[s] = phase;
                }
                if (++s == STAGES) { s = 0; phase ^= 1u; }
            }
        }
        // Drain (bounded): copies in flight on the leader's FULL phases,
        // which count both CTAs' bytes, and on this CTA's tails.
        if (lane == 0) {
#pragma unroll
            for (int i = 0; i < STAGES; ++i) {
                const u64 t0 = now_ns();
                if (cta == 0 && armed[i] != 0xFFFFFFFFu)
                    while (!mbar_try(FULL(i), armed[i]) && now_ns() - t0 < drain_ns(g)) {}
                if (tail_used >> i & 1u)
                    while (!mbar_try(TAIL(i), (tail_phase >> i & 1u) ^ 1u) && now_ns() - t0 < drain_ns(g)) {}
            }
        }
        __syncwarp();
    } else if (MODE == Mode::Weights && warp == 10) {
        // ---------------------- clear other experts' rows (both CTAs) --
        int e = 0;
        u32 stage = 0, tail_phase = 0;                   // stage: of the next tile's first k-block
        for (int round = 0, u; (u = tile_of(round)) < tiles; ++round) {
            const Tile t = tile_at(u, e);
            const int left = t.k_rows % E::BK;
            if (left % 16) {
                const int s = (int)((stage + t.kblocks - 1) % STAGES);
                const u32 par = tail_phase >> s & 1u;
                int got = 1;
                if (lane == 0) got = wait<false>(TAIL(s), par, sh, g, 5u);
                if (!__shfl_sync(0xFFFFFFFFu, got, 0)) break;
                __syncwarp();
                // four boxes of 64 rows x 128 bytes (a row keeps its 128
                // bytes under the swizzle)
                const u32 box = base + s * STAGE_BYTES;
                const int zeros = (16 - left % 16) * 8;                 // 16-byte units per box, to the instruction's end
                for (int i = lane; i < zeros; i += 32)
#pragma unroll
                    for (int b = 0; b < 4; ++b)
                        sts128(box + (u32)b * MN_BOX + (u32)left * 128u + (u32)i * 16u, make_uint4(0u, 0u, 0u, 0u));
                fence_async_smem();
                __syncwarp();
                if (lane == 0) {
                    if (cta != 0) {
                        mbar_arrive_cluster(CLEARED(s), 0u);
                    } else {
                        mbar_arrive(CLEARED(s));
                        mbar_arrive(FULL(s));            // nothing was counted on it: keeps the ring's parity
                    }
                }
                tail_phase ^= 1u << s;
            }
            stage = (stage + (u32)t.kblocks) % STAGES;
        }
    } else if (warp == 1) {
        // --------------------------------------- MMA issuer (leader CTA) --
        if (lane == 0 && cta == 0) {
            // With few rows this thread's own time is what a k-block takes:
            // descriptors are moved on (in 16 bytes), not made.
            constexpr u32 A_LBO = A_MN ? MN_BOX : 16u, B_LBO = B_MN ? MN_BOX : 16u;
            constexpr u32 A_KK = (A_MN ? 2048u : 32u) >> 4, B_KK = (B_MN ? 2048u : 32u) >> 4;
            const u64 a_first = smem_desc(base, A_LBO, 1024u, 2u), b_first = smem_desc(base + KPS * A_BYTES, B_LBO, 1024u, 2u);
            u64 a = a_first, b = b_first;
            int s = 0, e = 0;
            u32 phase = 0, count = 0, tail_phase = 0;
            bool ok = true;
            for (int round = 0, u; ok && (u = tile_of(round)) < tiles; ++round) {
                const Tile t = tile_at(u, e);
                if (t.kblocks == 0) continue;            // nothing to add: zeros are stored
                const u32 buf = count & 1u;
                if (!wait<true>(TEMPTY(buf), ((count >> 1) & 1u) ^ 1u, sh, g, 2u)) { ok = false; break; }
                tc_fence_after();
                const u32 d = tmem + buf * 256u;
                const u32 idesc = instr_desc(A_MN, B_MN, t.n, 256, E::FMT);
                for (int kb = 0; kb < t.kblocks; ++kb) {
                    if (!wait<true>(FULL(s), phase, sh, g, 3u)) { ok = false; break; }
                    if (MODE == Mode::Weights && t.k_rows % 16 && kb == t.kblocks - 1) {
                        if (!wait<true>(CLEARED(s), tail_phase >> s & 1u, sh, g, 6u)) { ok = false; break; }
                        tail_phase ^= 1u << s;
                    }
                    tc_fence_after();
                    auto mma = [&](int kk) {             // fourths of k-blocks
                        const u32 acc = kb > 0 || kk > 0 ? 1u : 0u;
                        const u64 ak = a + (kk >> 2) * (A_BYTES >> 4) + (kk & 3) * A_KK, bk = b + (kk >> 2) * (B_BYTES >> 4) + (kk & 3) * B_KK;
                        if (E::F8) mma_f8_pair(d, ak, bk, idesc, acc);
                        else tc_mma_f16kind_pair(d, ak, bk, idesc, acc);
                    };
                    if (MODE == Mode::Weights && t.k_rows - kb * E::BK <= E::BK - 16) {
                        // the last rows of an expert: no instruction behind them
                        for (int kk = 0; kk * 16 < t.k_rows - kb * E::BK; ++kk) mma(kk);
                    } else {
#pragma unroll
                        for (int kk = 0; kk < 4 * KPS; ++kk) mma(kk);
                    }
                    tc_commit_pair(EMPTY(s));            // both CTAs' stage s is free
                    a += STAGE_BYTES >> 4;
                    b += STAGE_BYTES >> 4;
                    if (++s == STAGES) { s = 0; phase ^= 1u; a = a_first; b = b_first; }
                }
                if (!ok) break;
                tc_commit_pair(TFULL(buf));
                ++count;
            }
            tc_commit_pair(DRAIN);
            const u64 t0 = now_ns();
            while (!mbar_try(DRAIN, 0u) && now_ns() - t0 < drain_ns(g)) {}
        }
        __syncwarp();
    } else {
        // ------------------------------------- store (both CTAs, 8 warps) --
        typedef typename E::Out Out;
        const int q = warp & 3, half = (warp - 2) >> 2;
        int e = 0;
        u32 count = 0;
        for (int round = 0, u; (u = tile_of(round)) < tiles; ++round) {
            const Tile t = tile_at(u, e);
            const int f = t.f + (int)cta * (TILE_F / 2) + q * 32 + lane;
            Out* out = static_cast<Out*>(g.out) + (MODE == Mode::Weights ? t.e * g.out_estride : 0) + t.row * g.out_ld + f;
            const bool mine = f < g.features;
            if (t.kblocks == 0) {
                if (g.vec_out == 1) {
                    const int lc = lane & 15;            // two rows of 64 bytes at a time
                    if (f - lane + 2 * lc < g.features)
                        for (int j = half * 2 + (lane >> 4); j < t.valid; j += 4)
                            *reinterpret_cast<u32*>(out - lane + 2 * lc + j * g.out_ld) = 0u;
                } else if (g.vec_out) {
                    // eight rows of 64 bytes at a time
                    const int lc = lane & 3;
                    if (f - lane + lc * 8 < g.features)
                        for (int j = half * 8 + (lane >> 2); j < t.valid; j += 16)
                            *reinterpret_cast<uint4*>(out - lane + lc * 8 + j * g.out_ld) = make_uint4(0u, 0u, 0u, 0u);
                } else if (mine) {
                    for (int j = half; j < t.valid; j += 2) out[j * g.out_ld] = from_f32<Out>(0.0f);
                }
                continue;
            }
            const u32 buf = count & 1u;
            const bool ready = wait<false>(TFULL(buf), (count >> 1) & 1u, sh, g, 4u);
            if (!__all_sync(0xFFFFFFFFu, ready)) break;
            tc_fence_after();
            const u32 src = tmem + ((u32)(q * 32) << 16) + buf * 256u;
            if (g.vec_out) {
                // the warp's 32 features as fragments: this lane's are
                // lane / 4 + {0, 8, 16, 24}
                float ws[4];
                if (E::F8) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int fi = f - lane + (lane >> 2) + 8 * i;
                        ws[i] = fi < g.features ? g.w_scale[t.e * g.w_scale_ld + fi] : 0.0f;
                    }
                }
                const u32 stg = base + STAGES * STAGE_BYTES + BAR_BYTES + OFFSET_BYTES + (u32)(warp - 2) * STAGING_BYTES;
                // 16-byte chunk c of row r at c ^ (r / 2 % 4), which is the
                // tensor store's 64-byte swizzle: neither the fragments'
                // stores nor the rows' loads meet in a bank
                const int sr = lane & 7, sm = lane >> 3;                // fragment row and matrix of stmatrix's address
                const int lr = lane >> 2, lc = lane & 3;                // row (of 8) and chunk of the store
                const bool in = f - lane + lc * 8 < g.features;
                Out* dst = out - lane + lc * 8;
                for (int j = half * 32; j < t.n; j += 64) {
                    u32 v[2][16];
                    tmem_ld_16x256(src + (u32)j, v[0]);
                    tmem_ld_16x256(src + (16u << 16) + (u32)j, v[1]);
                    tmem_wait(v[0], v[1]);
                    if (E::F8) {
                        const float xs = j + lane < t.valid ? g.x_scale[t.row + j + lane] : 0.0f;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const float s = __shfl_sync(0xFFFFFFFFu, xs, 8 * i + 2 * (lane & 3) + e);
#pragma unroll
                                for (int h = 0; h < 4; ++h)
                                    v[h >> 1][4 * i + 2 * (h & 1) + e] =
                                        __float_as_uint(__uint_as_float(v[h >> 1][4 * i + 2 * (h & 1) + e]) * (s * ws[h]));
                            }
                    }
                    // matrices m = 0 .. 3 of one stmatrix: features 8 m .. 8 m + 7
#pragma unroll
                    for (int hb = 0; hb < 2; ++hb) {     // 16 rows: half of the staging
                        // the store before the last one has read this half
                        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
                        __syncwarp();
                        const u32 part = stg + (u32)hb * (STAGING_BYTES / 2);
#pragma unroll
                        for (int i2 = 0; i2 < 2; ++i2) {
                            const int i = 2 * hb + i2, row = 8 * i2 + sr;
                            stmatrix_trans(part + (u32)(row * 64 + ((sm ^ (row >> 1 & 3)) * 16)),
                                           pack2<Out>(v[0][4 * i], v[0][4 * i + 1]), pack2<Out>(v[0][4 * i + 2], v[0][4 * i + 3]),
                                           pack2<Out>(v[1][4 * i], v[1][4 * i + 1]), pack2<Out>(v[1][4 * i + 2], v[1][4 * i + 3]));
                        }
                        const int row0 = j + 16 * hb;
                        // whole, or cut off by the tensor's own end (the
                        // weight gradient's rows are all of its matrix)
                        const bool whole = MODE == Mode::Weights ? row0 < t.valid : row0 + 16 <= t.valid;
                        if (g.vec_out == 1) {
                            __syncwarp();
                            const int word = lane & 15;  // of a row's 16; two rows at a time
                            const bool mine2 = f - lane + 2 * word < g.features;
#pragma unroll
                            for (int i2 = 0; i2 < 8; ++i2) {
                                const int row = 2 * i2 + (lane >> 4);
                                u32 w;
                                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w)
                                             : "r"(part + (u32)(row * 64 + (((word >> 2) ^ (row >> 1 & 3)) * 16) + (word & 3) * 4)) : "memory");
                                if (mine2 && row0 + row < t.valid)
                                    *reinterpret_cast<u32*>(out - lane + 2 * word + (row0 + row) * g.out_ld) = w;
                            }
                            __syncwarp();
                        } else if (whole) {
                            fence_async_smem();
                            __syncwarp();
                            if (lane == 0 && f < g.features)     // lane 0: the warp's first feature
                                asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];"
                                             ::"l"(&g.c), "r"(f), "r"(t.row + row0), "r"(MODE == Mode::Weights ? t.e : 0), "r"(part)
                                             : "memory");
                        } else {
                            __syncwarp();
#pragma unroll
                            for (int i2 = 0; i2 < 2; ++i2) {
                                const int row = 8 * i2 + lr;
                                const uint4 w = lds128(part + (u32)(row * 64 + ((lc ^ (row >> 1 & 3)) * 16)));
                                if (in && row0 + row < t.valid) *reinterpret_cast<uint4*>(dst + (row0 + row) * g.out_ld) = w;
                            }
                            __syncwarp();
                        }
                        if (lane == 0) asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                }
            } else {
                float ws = 1.0f;
                if (E::F8 && mine) ws = g.w_scale[t.e * g.w_scale_ld + f];
                for (int j = half * 16; j < t.n; j += 32) {
                    u32 v[16];
                    tmem_ld16(src + (u32)j, v);
                    if (E::F8) {
                        // this warp's 16 row scales, one load for all of them
                        const int rr = j + (lane & 15);
                        const float xs = rr < t.valid ? g.x_scale[t.row + rr] : 0.0f;
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            v[i] = __float_as_uint(__uint_as_float(v[i]) * (__shfl_sync(0xFFFFFFFFu, xs, i) * ws));
                    }
                    if (mine) {
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if (j + i < t.valid) out[(j + i) * g.out_ld] = from_f32<Out>(__uint_as_float(v[i]));
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (cta == 0) mbar_arrive(TEMPTY(buf));
                else mbar_arrive_cluster(TEMPTY(buf), 0u);
            }
            ++count;
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        __syncwarp();
    }

    // ------------------------------------------------------- teardown --
    tc_fence_before();
    __syncthreads();
    cluster_sync();                                      // the peer is done with our barriers and TMEM
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// Rows of a matrix (or of a stack of them, one per blockIdx.y) copied to rows
// that start on a 16-byte boundary, which TMA needs; row_bytes, src_ld and
// src_stride in bytes.  Four bytes a thread, put together from the two aligned
// words that hold them (words without a byte of the row are not read).  With
// offsets: only the matrices of experts that have rows; one whose clamped
// offsets do not ascend has none, whatever the others are.
__global__ void __launch_bounds__(256) align_rows_kernel(const unsigned char* __restrict__ src, int64_t src_ld, int64_t src_stride,
                                                         u32* __restrict__ dst, int64_t dst_words, int64_t n, int row_bytes,
                                                         const int* __restrict__ offsets, int all_rows) {
    if (offsets && min(max(offsets[blockIdx.y + 1], 0), all_rows) <= min(max(offsets[blockIdx.y], 0), all_rows)) return;
    constexpr int UP = 4;                                // words of a thread on their way at once
    const int words = (row_bytes + 3) / 4;
    for (int64_t r = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; r < n; r += (int64_t)gridDim.x * blockDim.y) {
        const unsigned char* s = src + blockIdx.y * src_stride + r * src_ld;
        u32* d = dst + (blockIdx.y * n + r) * dst_words;
        const int off = (int)(reinterpret_cast<uintptr_t>(s) & 3u);
        const u32* from = reinterpret_cast<const u32*>(s - off);
        for (int w0 = threadIdx.x; w0 < words; w0 += UP * blockDim.x) {
            u32 lo[UP], hi[UP];
#pragma unroll
            for (int u = 0; u < UP; ++u) {
                const int w = w0 + u * blockDim.x;
                if (w < words) {
                    lo[u] = from[w];
                    hi[u] = off && 4 * (w + 1) - off < row_bytes ? from[w + 1] : 0u;
                }
            }
#pragma unroll
            for (int u = 0; u < UP; ++u) {
                const int w = w0 + u * blockDim.x;
                if (w < words) d[w] = __funnelshift_r(lo[u], hi[u], 8 * off);
            }
        }
    }
}

constexpr int64_t MAX_DIM = int64_t(1) << 30;

// A matrix operand: rows of `cols` contiguous elements.
struct Matrix {
    const void* p;
    int64_t ld, stride;                // elements; stride between the experts' matrices
    int64_t rows, cols, count;
};

bool tma_ready(const Matrix& m, int es) {
    return aligned16(m.p) && (m.ld * es) % 16 == 0 && (m.count == 1 || (m.stride * es) % 16 == 0);
}
int64_t aligned_ld(int64_t cols, int es) {
    const int64_t per = 16 / es;
    return (cols + per - 1) / per * per;
}
// Workspace bytes of an operand's aligned copy; 0 when TMA can read it in place.
int64_t copy_bytes(const Matrix& m, int es) {
    if (tma_ready(m, es)) return 0;
    return (m.count * m.rows * aligned_ld(m.cols, es) * es + 255) / 256 * 256;
}

// offsets: the stack's matrices are the experts'.
int make_ready(Matrix& m, int es, char*& ws, int sms, cudaStream_t st, const int* offsets = nullptr, int64_t all_rows = 0) {
    const int64_t bytes = copy_bytes(m, es);
    if (!bytes) return 0;
    if (m.cols * es > MAX_DIM) return fail(8, "grouped_matmul: rows of more than 2^30 bytes must start on 16-byte boundaries");
    const int64_t ld = aligned_ld(m.cols, es), words = ld * es / 4;
    // enough blocks for the device with all experts, and with one
    const int64_t want = (m.rows + 3) / 4, share = (int64_t)sms * 16 / m.count, most = share > sms ? share : sms;
    const dim3 grid((unsigned)(want < most ? want : most), (unsigned)m.count), block(64, 4);
    align_rows_kernel<<<grid, block, 0, st>>>(static_cast<const unsigned char*>(m.p), m.ld * es, m.stride * es, reinterpret_cast<u32*>(ws),
                                              words, m.rows, (int)(m.cols * es), offsets, (int)all_rows);
    if (int rc = launched("grouped_matmul: aligned copy")) return rc;
    m.p = ws;
    m.ld = ld;
    m.stride = m.rows * ld;
    ws += bytes;
    return 0;
}

// Tensor map of a matrix operand: boxes of 128 bytes x `box_rows` rows.
int encode(TmaDesc* d, const Matrix& m, int es, uint32_t box_rows, std::string& err) {
    uint64_t dims[3] = {(uint64_t)m.cols, (uint64_t)m.rows, (uint64_t)m.count};
    uint64_t strides[2] = {(uint64_t)(m.ld * es), (uint64_t)((m.count == 1 ? m.rows * m.ld : m.stride) * es)};
    uint32_t box[3] = {(uint32_t)(128 / es), box_rows, 1};
    return tc_encode_tensor_map(d, es == 1 ? 0 : 2, 3, const_cast<void*>(m.p), dims, strides, box, 1, err);
}

// Tensor map of the result: 16 rows x 64 bytes.
int encode_out(GroupedArgs& a, void* p, int64_t ld, int64_t stride, int64_t rows, int64_t features, int64_t count, std::string& err) {
    const int64_t all = ld | features | (count == 1 ? 0 : stride);
    a.vec_out = aligned16(p) && all % 8 == 0 ? 2 : element_aligned(4, {p}) && all % 2 == 0 ? 1 : 0;
    if (a.vec_out != 2) return 0;
    uint64_t dims[3] = {(uint64_t)features, (uint64_t)rows, (uint64_t)count};
    uint64_t strides[2] = {(uint64_t)(ld * 2), (uint64_t)((count == 1 ? rows * ld : stride) * 2)};
    uint32_t box[3] = {32, 16, 1};
    return tc_encode_tensor_map(&a.c, 2, 3, p, dims, strides, box, 3, err);
}

template <class E, Mode MODE, bool A_MN, int ROWS>
int launch_ring(const GroupedArgs& a, int pairs, int dev, cudaStream_t st) {
    auto k = grouped_kernel<E, MODE, A_MN, ROWS>;
    static bool ready[64] = {false};
    if (!ready[dev]) {
        if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, Ring<ROWS>::SMEM_BYTES) != cudaSuccess) {
            cudaGetLastError();
            return fail(14, "grouped_matmul: cudaFuncSetAttribute");
        }
        ready[dev] = true;
    }
    k<<<2 * pairs, ALL_THREADS<MODE>, Ring<ROWS>::SMEM_BYTES, st>>>(a);
    return launched("grouped_matmul");
}
template <class E, Mode MODE, bool A_MN>
int launch(const GroupedArgs& a, int pairs, int dev, cudaStream_t st) {
    if constexpr (MODE == Mode::Rows) {
        if (a.rows <= 32) return launch_ring<E, MODE, A_MN, 32>(a, pairs, dev, st);
        if (a.rows <= 128) return launch_ring<E, MODE, A_MN, 128>(a, pairs, dev, st);
    }
    return launch_ring<E, MODE, A_MN, TILE_R>(a, pairs, dev, st);
}

int check_common(const char* what, int64_t rows, int64_t experts, int64_t n, int64_t k) {
    if (rows < 0 || rows > MAX_DIM || experts < 1 || experts > MAX_EXPERTS || n < 1 || n > MAX_DIM || k < 1 || k > MAX_DIM)
        return fail(8, std::string(what) + ": sizes out of range (0 <= rows <= 2^30, 1 <= experts <= 1024, 1 <= n, k <= 2^30)");
    return 0;
}

unsigned long long timeout_ns() {
    const char* to = getenv("BAFE_TC_TIMEOUT_MS");
    return (unsigned long long)(to ? atof(to) : 2000.0) * 1000000ull;
}

// The storing warps wait for a whole contraction: 4 us per 64 of it on top
// of the limit, some ten times what a pair needs at full clocks.
unsigned long long contraction_ns(int64_t n) { return (unsigned long long)n / 64 * 4000; }

int start(GroupedArgs& a, int& dev, int& sms) {
    if (int rc = current_device(dev, sms)) return rc;
    memset(&a, 0, sizeof(a));
    a.err = device_error_word(dev);
    if (!a.err) return fail(6, "cannot allocate the device error word");
    a.timeout_ns = timeout_ns();
    return 0;
}

int elem_size(int dtype) { return dtype == DTYPE_E4M3 ? 1 : 2; }

// Forward operands of the call: x [rows][k]; w as stored, [experts] matrices
// of n x k (w_kmajor) or k x n rows.
void forward_operands(Matrix& x, Matrix& w, const void* xp, int64_t x_ld, const void* wp, int64_t w_ld, int64_t w_stride,
                      int w_kmajor, int64_t rows, int64_t experts, int64_t n, int64_t k) {
    x = {xp, x_ld, 0, rows, k, 1};
    w = {wp, w_ld, w_stride, w_kmajor ? n : k, w_kmajor ? k : n, experts};
}

}  // namespace
}  // namespace lm
}  // namespace bafe_cuda

#define BAFE_API extern "C" __attribute__((visibility("default")))

using namespace bafe_cuda;
using namespace bafe_cuda::lm;

BAFE_API int64_t bafe_cuda_grouped_matmul_workspace(const void* x, int64_t x_ld, const void* w, int64_t w_ld,
                                                    int64_t w_stride, int w_kmajor, int64_t rows, int64_t experts,
                                                    int64_t n, int64_t k, int dtype) {
    if (check_common("grouped_matmul", rows, experts, n, k)) return -1;
    Matrix mx, mw;
    forward_operands(mx, mw, x, x_ld, w, w_ld, w_stride, w_kmajor, rows, experts, n, k);
    return copy_bytes(mx, elem_size(dtype)) + copy_bytes(mw, elem_size(dtype));
}

BAFE_API int bafe_cuda_grouped_matmul(const void* x, int64_t x_ld, const void* w, int64_t w_ld, int64_t w_stride,
                                      int w_kmajor, const int* offsets, const float* x_scale, const float* w_scale,
                                      int64_t w_scale_ld, void* y, int64_t y_ld, int64_t rows, int64_t experts, int64_t n,
                                      int64_t k, int dtype, int y_dtype, void* workspace, int64_t workspace_bytes,
                                      void* stream) {
    if (int rc = check_common("grouped_matmul", rows, experts, n, k)) return rc;
    const bool f8 = dtype == DTYPE_E4M3;
    if (!f8 && dtype != BAFE_DTYPE_F16 && dtype != BAFE_DTYPE_BF16)
        return fail(8, "grouped_matmul: operands must be f16, bf16 or e4m3");
    if (y_dtype != BAFE_DTYPE_F16 && y_dtype != BAFE_DTYPE_BF16) return fail(8, "grouped_matmul: y must be f16 or bf16");
    if (!f8 && y_dtype != dtype) return fail(8, "grouped_matmul: y must have the operands' 16-bit type");
    if (f8 != (x_scale != nullptr) || f8 != (w_scale != nullptr))
        return fail(8, "grouped_matmul: e4m3 operands take x_scale and w_scale, 16-bit ones none");
    if (f8 && !w_kmajor) return fail(8, "grouped_matmul: e4m3 weights must be contiguous along k");
    if (rows == 0) return 0;
    if (!x || !w || !offsets || !y) return fail(8, "grouped_matmul: null operand");
    if (x_ld < k || y_ld < n || w_ld < (w_kmajor ? k : n) ||
        (experts > 1 && w_stride < ((w_kmajor ? n : k) - 1) * w_ld + (w_kmajor ? k : n)) || (f8 && w_scale_ld < n))
        return fail(8, "grouped_matmul: strides must be at least the rows' lengths");
    const int es = elem_size(dtype);
    if (!element_aligned(es, {x, w}) || !element_aligned(2, {y}) || !element_aligned(4, {offsets, x_scale, w_scale}))
        return fail(8, "grouped_matmul: operands must start on a multiple of their element's size");
    Matrix mx, mw;
    forward_operands(mx, mw, x, x_ld, w, w_ld, w_stride, w_kmajor, rows, experts, n, k);
    const int64_t need = copy_bytes(mx, es) + copy_bytes(mw, es);
    if (need && (!workspace || workspace_bytes < need || !aligned16(workspace)))
        return fail(8, "grouped_matmul: workspace too small or unaligned (see bafe_cuda_grouped_matmul_workspace)");
    GroupedArgs a;
    int dev = 0, sms = 0;
    if (int rc = start(a, dev, sms)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    char* ws = static_cast<char*>(workspace);
    if (int rc = make_ready(mx, es, ws, sms, st)) return rc;
    if (int rc = make_ready(mw, es, ws, sms, st, offsets, rows)) return rc;
    std::string err;
    int rc = encode(&a.a, mw, es, w_kmajor ? 128 : 64, err);
    if (!rc) rc = encode(&a.b, mx, es, 128, err);
    for (int i = 0; i < 3 && !rc; ++i) rc = encode(&a.b_part[i], mx, es, 64 >> i, err);
    if (!rc) rc = encode_out(a, y, y_ld, 0, rows, n, 1, err);
    if (rc) return fail(rc, err);
    a.offsets = offsets;
    a.out = y;
    a.x_scale = x_scale;
    a.w_scale = w_scale;
    a.w_scale_ld = w_scale_ld;
    a.out_ld = y_ld;
    a.rows = (int)rows;
    a.experts = (int)experts;
    a.features = (int)n;
    a.k = (int)k;
    a.timeout_ns += contraction_ns(k);
    // no more pairs than tiles there can be: every expert with rows may end
    // in a part of a tile
    const int64_t most = (rows / TILE_R + (rows < experts ? rows : experts)) * ((n + TILE_F - 1) / TILE_F);
    if (most > (int64_t(1) << 30)) return fail(8, "grouped_matmul: too many tiles");
    const int pairs = (int)(most < sms / 2 ? most : sms / 2);
    if (f8) return y_dtype == BAFE_DTYPE_BF16 ? launch<EE4m3Bf16, Mode::Rows, false>(a, pairs, dev, st)
                                              : launch<EE4m3F16, Mode::Rows, false>(a, pairs, dev, st);
    if (dtype == BAFE_DTYPE_BF16)
        return w_kmajor ? launch<EBf16, Mode::Rows, false>(a, pairs, dev, st) : launch<EBf16, Mode::Rows, true>(a, pairs, dev, st);
    return w_kmajor ? launch<EF16, Mode::Rows, false>(a, pairs, dev, st) : launch<EF16, Mode::Rows, true>(a, pairs, dev, st);
}

BAFE_API int64_t bafe_cuda_grouped_matmul_grad_weight_workspace(const void* dy, int64_t dy_ld, const void* x,
                                                                int64_t x_ld, int64_t rows, int64_t n, int64_t k) {
    if (check_common("grouped_matmul_grad_weight", rows, 1, n, k)) return -1;
    return copy_bytes({dy, dy_ld, 0, rows, n, 1}, 2) + copy_bytes({x, x_ld, 0, rows, k, 1}, 2);
}

BAFE_API int bafe_cuda_grouped_matmul_grad_weight(const void* dy, int64_t dy_ld, const void* x, int64_t x_ld,
                                                  const int* offsets, void* dw, int64_t dw_ld, int64_t dw_stride,
                                                  int64_t rows, int64_t experts, int64_t n, int64_t k, int dtype,
                                                  void* workspace, int64_t workspace_bytes, void* stream) {
    if (int rc = check_common("grouped_matmul_grad_weight", rows, experts, n, k)) return rc;
    if (dtype != BAFE_DTYPE_F16 && dtype != BAFE_DTYPE_BF16)
        return fail(8, "grouped_matmul_grad_weight: operands must be f16 or bf16");
    if (!dw || !offsets || (rows && (!dy || !x))) return fail(8, "grouped_matmul_grad_weight: null operand");
    if (dy_ld < n || x_ld < k || dw_ld < k || (experts > 1 && dw_stride < (n - 1) * dw_ld + k))
        return fail(8, "grouped_matmul_grad_weight: strides must be at least the rows' lengths");
    if (!element_aligned(2, {dy, x, dw}) || !element_aligned(4, {offsets}))
        return fail(8, "grouped_matmul_grad_weight: operands must start on a multiple of their element's size");
    GroupedArgs a;
    int dev = 0, sms = 0;
    if (int rc = start(a, dev, sms)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (rows == 0) {
        cudaError_t e = cudaSuccess;
        for (int64_t i = 0; i < experts && e == cudaSuccess; ++i)
            e = cudaMemset2DAsync(static_cast<char*>(dw) + i * dw_stride * 2, (size_t)dw_ld * 2, 0, (size_t)k * 2, (size_t)n, st);
        return e == cudaSuccess ? 0 : (cudaGetLastError(), fail(7, "grouped_matmul_grad_weight: cudaMemset2DAsync"));
    }
    Matrix mdy = {dy, dy_ld, 0, rows, n, 1}, mx = {x, x_ld, 0, rows, k, 1};
    const int64_t need = copy_bytes(mdy, 2) + copy_bytes(mx, 2);
    if (need && (!workspace || workspace_bytes < need || !aligned16(workspace)))
        return fail(8, "grouped_matmul_grad_weight: workspace too small or unaligned "
                       "(see bafe_cuda_grouped_matmul_grad_weight_workspace)");
    char* ws = static_cast<char*>(workspace);
    if (int rc = make_ready(mdy, 2, ws, sms, st)) return rc;
    if (int rc = make_ready(mx, 2, ws, sms, st)) return rc;
    std::string err;
    int rc = encode(&a.a, mx, 2, 64, err);
    if (!rc) rc = encode(&a.b, mdy, 2, 64, err);
    if (!rc) rc = encode_out(a, dw, dw_ld, dw_stride, n, k, experts, err);
    if (rc) return fail(rc, err);
    a.offsets = offsets;
    a.out = dw;
    a.out_ld = dw_ld;
    a.out_estride = dw_stride;
    a.rows = (int)rows;
    a.experts = (int)experts;
    a.features = (int)k;
    a.out_rows = (int)n;
    a.timeout_ns += contraction_ns(rows);
    const int64_t most = experts * ((n + TILE_R - 1) / TILE_R) * ((k + TILE_F - 1) / TILE_F);
    if (most > (int64_t(1) << 30)) return fail(8, "grouped_matmul_grad_weight: too many tiles");
    const int pairs = (int)(most < sms / 2 ? most : sms / 2);
    return dtype == BAFE_DTYPE_BF16 ? launch<EBf16, Mode::Weights, true>(a, pairs, dev, st)
                                    : launch<EF16, Mode::Weights, true>(a, pairs, dev, st);
}
