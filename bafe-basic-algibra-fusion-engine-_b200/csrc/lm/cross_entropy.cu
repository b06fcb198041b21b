// cross_entropy.cu -- softmax cross entropy over a vocabulary, from the hidden
// states and the output weights, without keeping the logits; and its gradient.
//
//   z = x w^T              x [rows][width], w [vocab][width], 16-bit
//   lse_t = log sum_v exp z[t][v],   loss_t = lse_t - z[t][target_t]
//   g[t][v] = dloss_t (exp(z[t][v] - lse_t) - (v = target_t))
//   dx = g w,  dw = g^T x
//
// Products of 2 rows vocab width operations each, one forward and three in
// the gradient: the tensor cores bound them, the weights' bytes where rows are
// few.  8192 x 4096 x 131072 bf16 5.6 to 6.8 ms (1300 to 1570 TFLOP/s, by the power
// cap; the library's bare product of that size 5.7 to 6.4), the gradient of 8192 x
// 4096 x 32768 4.7 to 5.2 ms, the tensor cores 79 to 85 % busy at full clock.
// One persistent tcgen05 kernel on CTA pairs does all of them, a tile of 256
// x 256 a pair, with an epilogue per role:
//
//   Lse    z of a tile goes from TMEM to registers, where a thread has a row's
//          columns, and no further: their maximum and sum of exponentials go to
//          memory, one of each per row, tile and half, and a second kernel joins them.
//   Grad   z again, made g from the given lse, 16 bits, into a piece of up to
//          PIECE_BYTES: the vocabulary is walked in pieces.
//   Acc    g w over a piece, 32 bits; pieces (and the splits of a long
//          contraction over more pairs than there are tiles) are added up in a
//          fixed order.
//   Out    a finished product in 16 bits: dw of a piece (its contraction over
//          the rows is whole), and dx where there is one piece.
//
// g is rounded to 16 bits once: the products take their operands in that
// type, and its errors (half a step relative each) are independent and
// average out over the sums.  It is divided by the largest |dloss| of the rows
// that count before, which the products' epilogues take back in 32 bits: with
// one dloss for all rows, the mean's, the targets' entries would otherwise all
// be rounded the same way (777 x 50001 x 1150 f16: dw off by 4.4e-4, with it
// 2.6e-4, the result's own rounding).  Other rows' entries keep the type's half
// step.  f16's g is multiplied by 2^15 too, to use its range: entries below
// 2^-29 of the largest dloss are among its smallest numbers, and off by up to 2^-40
// of that dloss (with 2^12, as it was, by 2^-37: dx of a row with 2^-24 of the
// largest dloss, 50000 words, was off by six times what the roundings account for).
//
// The tensor core truncates its 32-bit sum at each of its steps of 16
// products: a step is short by some 2^-26 of a logit of random terms (lse of
// 4096-long products off by 1.3e-6 of itself) and by 2^-23 where all terms have one
// sign.  So Lse sums CHUNK k-blocks at a time there and adds them up in
// registers, rounded to nearest (8192 x 4096 x 131072 on one machine: chunks of 256 took 7.5
// ms and were off by 0.8e-7, of 512 6.6 ms, of 1024 6.2 ms and 3e-7, no chunks 6.2
// ms; short ones wait for the drain).  Grad's logits have to be those that lse was made
// of, to the last bit: a likely target's entry of g is p - 1, and with whole sums
// here p was off by 2e-4 of itself at a logit of 16, as much as 1 - p.  (In the
// same parts: 16 rows x 4096 x 32768 178.8 us instead of 176.8, 128 rows 200 instead
// of 198, the gradient of 4096 rows as before.)  The sums of dx and dw, whose terms
// may all have one sign, go in longer parts, short by a sixteenth of their
// type's half step at most: 4096 terms in f16, 16384 in bf16.  (In one go dw
// over 2^22 rows was 2.6 % short.)
//
//   warp 0     TMA producer (both CTAs), k-blocks of 64 into a ring of stages
//   warp 1     allocates TMEM; the leader's lane 0 issues the MMAs into one
//              of two 256-column accumulators
//   warps 2-9  the epilogue, on the other accumulator
//
// Waits are bounded as in the grouped products (operand.cuh).
#include "operand.cuh"

#include <cmath>
#include <cstring>

namespace bafe_cuda {
namespace lm {
namespace {

constexpr int TILE = 256;
constexpr int BK = 64;
constexpr int THREADS = 320;
constexpr int STAGES = 6;
constexpr u32 A_BYTES = 16384, B_BYTES = 16384, STAGE_BYTES = A_BYTES + B_BYTES;
constexpr u32 MN_BOX = 8192;           // 64 of a tile x 64 of the contraction
constexpr u32 STAGING = 4096;          // what an epilogue warp stores at a time: 32 rows x 128 bytes
constexpr int SMEM_BYTES = 1024 + STAGES * (int)STAGE_BYTES + 8 * (int)STAGING + 512;
static_assert(SMEM_BYTES <= 227 * 1024, "shared memory");
constexpr float LOG2E = 1.4426950408889634f;

enum class Role { Lse, Grad, Acc, Out };
// k-blocks that are summed on the tensor core at a time.
template <class T, Role R> constexpr int CHUNK = R == Role::Lse || R == Role::Grad ? 16 : std::is_same<T, __half>::value ? 64 : 256;

struct CeArgs {
    TmaDesc a, b, c;
    const float* dloss;                // Grad
    const void* target;                // int64 or int32
    const float* lse;                  // Grad
    const float* scale;                // gradient: what dloss is multiplied with in g, and the results; null: see scales_of
    float range;                       // of the largest counted |dloss| in g
    int losses, vocab;                 // rows of dloss and target; words
    float2* part;                      // Lse: [runs of tiles, two halves][rows]: maximum (times log2 e) and sum
    float* hit;                        // Lse: [rows], the target's logit
    void* out;                         // Out, without tensor stores; turned Grad: g of the piece
    float* acc;                        // turned Acc
    int64_t acc_stride;                // from split to split
    unsigned* err;
    u64 timeout_ns;
    int64_t dloss_stride, out_ld, ignore;
    int target_bytes;
    int rows, cols;                    // of the result
    int m_tiles, n_tiles, group_m;
    int tile_n;                        // turned: rows of the tile
    int units, run, runs;              // Lse: `run` tiles along the vocabulary are a unit; runs in all
    int splits, kblocks;               // parts of the contraction
    int b_row, out_row;                // first row of b, of the result
    int v0, held;                      // Grad: first word and columns of the piece
    int tma_out, add;                  // result rows on 16-byte boundaries; Acc: onto what is there
};

// kind::f16 result of a pair of values.
template <class T> __device__ __forceinline__ u32 pack2(float lo, float hi);
template <> __device__ __forceinline__ u32 pack2<__nv_bfloat16>(float lo, float hi) {
    u32 r;
    asm("cvt.rn.bf16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(lo), "f"(hi));
    return r;
}
template <> __device__ __forceinline__ u32 pack2<__half>(float lo, float hi) {
    u32 r;
    asm("cvt.rn.f16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float exp2_fast(float v) {    // within 2^-22 of the value
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// v[at], by masks: an index would put v into memory.
template <int N> __device__ __forceinline__ float pick(const float (&v)[N], int at) {
    u32 h = 0u;
#pragma unroll
    for (int i = 0; i < N; ++i) h |= __float_as_uint(v[i]) & (i == at ? 0xFFFFFFFFu : 0u);
    return __uint_as_float(h);
}
__device__ __forceinline__ int64_t target_of(const CeArgs& g, int row) {
    return g.target_bytes == 8 ? static_cast<const int64_t*>(g.target)[row] : (int64_t)static_cast<const int*>(g.target)[row];
}
// |dloss| of a row, 0 where it counts for nothing in the others' factor: rows
// that are ignored or whose target is out of range, infinities and NaN.
__device__ __forceinline__ float counted(const CeArgs& g, int row) {
    const int64_t word = target_of(g, row);
    const float v = fabsf(g.dloss[row * g.dloss_stride]);
    return word != g.ignore && word >= 0 && word < g.vocab && v < INFINITY ? v : 0.0f;
}

// g's factor and the results' (see scale_kernel), by the 256 epilogue threads
// themselves, where the losses are few: a launch less.  `part`: 8 floats of shared memory.
__device__ __forceinline__ float2 scales_of(float m, float range) {
    if (!(m >= 1e-30f)) m = 1e-30f;                      // zeros, and what divisions could not keep
    return make_float2(range / m, m / range);
}
__device__ __forceinline__ float2 scales_of(const CeArgs& g, volatile float* part) {
    if (g.scale) return make_float2(__ldcg(&g.scale[0]), __ldcg(&g.scale[1]));
    const int warp = (int)(threadIdx.x >> 5) - 2, lane = threadIdx.x & 31;
    float m = 0.0f;
#pragma unroll 4
    for (int i = warp * 32 + lane; i < g.losses; i += 256) m = fmaxf(m, counted(g, i));
    m = warp_max_nan(m);
    if (lane == 0) part[warp] = m;
    asm volatile("bar.sync 1, 256;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, part[i]);
    return scales_of(m, g.range);
}

struct Unit {
    int m, n, count, split, run;       // row tile; first column tile and their number
};

template <class T, Role R, bool PARTS, bool A_MN, bool B_MN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1) ce_kernel(const __grid_constant__ CeArgs g) {
    using namespace bafe::tc;
    constexpr int PART = PARTS ? CHUNK<T, R> : 1 << 30;
    second_may_start();
    extern __shared__ unsigned char smem_raw[];
    const u32 raw_addr = smem_u32(smem_raw);
    const u32 base = (raw_addr + 1023u) & ~1023u;
    unsigned char* smem = smem_raw + (base - raw_addr);
    const u32 staging = base + STAGES * STAGE_BYTES, bars = staging + 8 * STAGING;
    auto FULL = [&](int s) { return bars + 8u * s; };
    auto EMPTY = [&](int s) { return bars + 8u * (STAGES + s); };
    auto TFULL = [&](int b) { return bars + 8u * (2 * STAGES + b); };
    auto TEMPTY = [&](int b) { return bars + 8u * (2 * STAGES + 2 + b); };
    const u32 DRAIN = bars + 8u * (2 * STAGES + 4);
    volatile Shared* sh = reinterpret_cast<volatile Shared*>(smem + STAGES * STAGE_BYTES + 8 * STAGING + 8 * (2 * STAGES + 5));
    volatile float* part = reinterpret_cast<volatile float*>(sh + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const u32 cta = cluster_rank();
    const int pair = (int)(blockIdx.x >> 1), num_pairs = (int)(gridDim.x >> 1);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(FULL(s), 1);
            mbar_init(EMPTY(s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(TFULL(b), 1);
            mbar_init(TEMPTY(b), 16);                    // the 8 epilogue warps of both CTAs
        }
        mbar_init(DRAIN, 1);
        sh->abort = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32((const void*)&sh->tmem_base)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();                                      // both CTAs' barriers exist
    tc_fence_after();
    const u32 tmem = sh->tmem_base;
    first_is_done();                                     // a piece's products follow one another closely

    // Units in groups of group_m row tiles, row tiles first: what the pairs
    // work on at a time shares its operands through L2.
    const int columns = R == Role::Lse ? g.runs : g.n_tiles;
    auto unit_at = [&](int u) {
        Unit t;
        t.split = 0;
        if (R == Role::Acc) {
            const int tiles = g.m_tiles * g.n_tiles;
            t.split = u / tiles;
            u -= t.split * tiles;
        }
        const int per_group = g.group_m * columns, group = u / per_group, first = group * g.group_m;
        const int size = min(g.group_m, g.m_tiles - first), local = u - group * per_group;
        t.m = first + local % size;
        t.run = local / size;
        t.n = R == Role::Lse ? t.run * g.run : t.run;
        t.count = R == Role::Lse ? min(g.run, g.n_tiles - t.n) : 1;
        return t;
    };
    auto k_first = [&](const Unit& t) { return R == Role::Acc ? (int)((int64_t)g.kblocks * t.split / g.splits) : 0; };
    auto k_end = [&](const Unit& t) { return R == Role::Acc ? (int)((int64_t)g.kblocks * (t.split + 1) / g.splits) : g.kblocks; };

    if (warp == 0) {
        // ---------------------------------------- TMA producer (both CTAs) --
        int s = 0;
        u32 phase = 0;
        bool ok = true;
        u32 armed[STAGES];
#pragma unroll
        for (int i = 0; i < STAGES; ++i) armed[i] = 0xFFFFFFFFu;
        constexpr u32 both = 2 * (A_BYTES + B_BYTES);    // bytes of both CTAs
        for (int u = pair; lane == 0 && ok && u < g.units; u += num_pairs) {
            const Unit t = unit_at(u);
            const int ra = t.m * TILE + (int)cta * (TILE / 2);
            for (int n = t.n; n < t.n + t.count && ok; ++n) {
                const int rb = n * TILE + (int)cta * (TILE / 2);
                const int k1 = k_end(t);
                for (int kb = k_first(t); kb < k1; ++kb) {
                    if (!wait<false>(EMPTY(s), phase ^ 1u, sh, g, 1u)) { ok = false; break; }
                    const u32 a_dst = base + s * STAGE_BYTES, b_dst = a_dst + A_BYTES;
                    if (cta == 0) mbar_expect_tx(FULL(s), both);
                    const int k = kb * BK;
                    if (A_MN) {
#pragma unroll
                        for (int j = 0; j < 2; ++j) tma_load_3d_pair(a_dst + j * MN_BOX, &g.a, FULL(s), ra + 64 * j, k, 0);
                    } else {
                        tma_load_3d_pair(a_dst, &g.a, FULL(s), k, ra, 0);
                    }
                    if (B_MN) {
#pragma unroll
                        for (int j = 0; j < 2; ++j) tma_load_3d_pair(b_dst + j * MN_BOX, &g.b, FULL(s), rb + 64 * j, g.b_row + k, 0);
                    } else {
                        tma_load_3d_pair(b_dst, &g.b, FULL(s), k, g.b_row + rb, 0);
                    }
                    armed[s] = phase;
                    if (++s == STAGES) { s = 0; phase ^= 1u; }
                }
            }
        }
        // Drain (bounded): copies in flight, both CTAs' on the leader's barriers.
        if (lane == 0 && cta == 0) {
#pragma unroll
            for (int i = 0; i < STAGES; ++i) {
                const u64 t0 = now_ns();
                if (armed[i] != 0xFFFFFFFFu)
                    while (!mbar_try(FULL(i), armed[i]) && now_ns() - t0 < drain_ns(g)) {}
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // --------------------------------------- MMA issuer (leader CTA) --
        if (lane == 0 && cta == 0) {
            constexpr u32 FMT = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
            constexpr u32 A_LBO = A_MN ? MN_BOX : 16u, B_LBO = B_MN ? MN_BOX : 16u;
            constexpr u32 A_KK = (A_MN ? 2048u : 32u) >> 4, B_KK = (B_MN ? 2048u : 32u) >> 4;
            const u64 a_first = smem_desc(base, A_LBO, 1024u, 2u), b_first = smem_desc(base + A_BYTES, B_LBO, 1024u, 2u);
            const u32 idesc = instr_desc(A_MN, B_MN, TILE, 256, FMT);
            u64 a = a_first, b = b_first;
            int s = 0;
            u32 phase = 0, count = 0;
            bool ok = true;
            for (int u = pair; ok && u < g.units; u += num_pairs) {
                const Unit t = unit_at(u);
                for (int n = 0; n < t.count && ok; ++n) {
                    const int first = k_first(t), last = k_end(t);
                    for (int k0 = first, k1; k0 < last; k0 = k1) {
                    k1 = last - k0 > PART ? k0 + PART : last;
                    const u32 buf = count & 1u;
                    if (!wait<true>(TEMPTY(buf), ((count >> 1) & 1u) ^ 1u, sh, g, 2u)) { ok = false; break; }
                    tc_fence_after();
                    const u32 d = tmem + buf * 256u;
                    for (int kb = k0; kb < k1; ++kb) {
                        if (!wait<true>(FULL(s), phase, sh, g, 3u)) { ok = false; break; }
                        tc_fence_after();
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            tc_mma_f16kind_pair(d, a + kk * A_KK, b + kk * B_KK, idesc, kb > k0 || kk > 0 ? 1u : 0u);
                        tc_commit_pair(EMPTY(s));        // both CTAs' stage s is free
                        a += STAGE_BYTES >> 4;
                        b += STAGE_BYTES >> 4;
                        if (++s == STAGES) { s = 0; phase ^= 1u; a = a_first; b = b_first; }
                    }
                    if (!ok) break;
                    tc_commit_pair(TFULL(buf));
                    ++count;
                    }
                }
            }
            tc_commit_pair(DRAIN);
            const u64 t0 = now_ns();
            while (!mbar_try(DRAIN, 0u) && now_ns() - t0 < drain_ns(g)) {}
        }
        __syncwarp();
    } else {
        // ---------------------------------- epilogue (both CTAs, 8 warps) --
        // A thread has one row of the tile (TMEM's lane); the two warps of a
        // lane quarter take turns along its columns.
        const int q = warp & 3, half = (warp - 2) >> 2;
        const u32 stg = staging + (u32)(warp - 2) * STAGING;
        float2 scale = make_float2(1.0f, 1.0f);
        if (R != Role::Lse) scale = scales_of(g, part);
        const float unscale = scale.y;
        u32 count = 0;
        bool ok = true;
        for (int u = pair; ok && u < g.units; u += num_pairs) {
            const Unit t = unit_at(u);
            const int row0 = t.m * TILE + (int)cta * (TILE / 2) + q * 32, row = row0 + lane;
            const bool mine = row < g.rows;
            int64_t target = -1;
            float top = -INFINITY, sum = 0.0f;           // Lse
            float weight = 0.0f, lse = 0.0f;             // Grad
            if ((R == Role::Lse || R == Role::Grad) && mine) target = target_of(g, row);
            if (R == Role::Grad && mine) {
                lse = g.lse[row];
                weight = g.dloss[row * g.dloss_stride] * scale.x;
                if (target == g.ignore) weight = 0.0f;   // and nothing that lse holds counts: see below
                else if (target < 0 || target >= g.cols) weight = NAN;
            }
            const bool skip = R == Role::Grad && (!mine || target == g.ignore);
            for (int n = t.n; n < t.n + t.count; ++n) {
                // This thread's columns of the tile, four times 32 of them from
                // first(0) .. first(3) on: the sums of the contraction's parts.
                auto first = [&](int j) { return R == Role::Lse || R == Role::Acc ? half * 32 + 64 * j : half * 64 + (j >> 1) * 128 + (j & 1) * 32; };
                float z[4][32];
                u32 src = 0u;
                auto next = [&]() {                      // the next sums are there
                    const u32 buf = count & 1u;
                    const bool ready = wait<false>(TFULL(buf), (count >> 1) & 1u, sh, g, 4u);
                    if (!__all_sync(0xFFFFFFFFu, ready)) return false;
                    tc_fence_after();
                    src = tmem + ((u32)(q * 32) << 16) + buf * 256u;
                    return true;
                };
                auto taken = [&]() {                     // their columns may be written again
                    const u32 buf = count & 1u;
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        if (cta == 0) mbar_arrive(TEMPTY(buf));
                        else mbar_arrive_cluster(TEMPTY(buf), 0u);
                    }
                    ++count;
                };
                const int begin = k_first(t), last = k_end(t);
                for (int k0 = begin; PARTS && k0 < last; k0 += PART) {
                    if (!next()) { ok = false; break; }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
#pragma unroll
                        for (int h = 0; h < 32; h += 16) {
                            u32 v[16];
                            tmem_ld16(src + (u32)(first(j) + h), v);
                            if (k0 == begin) {
#pragma unroll
                                for (int i = 0; i < 16; ++i) z[j][h + i] = __uint_as_float(v[i]);
                            } else {
#pragma unroll
                                for (int i = 0; i < 16; i += 2) bafe::fadd2_rn(z[j][h + i], z[j][h + i + 1], v[i], v[i + 1]);
                            }
                        }
                    }
                    taken();
                }
                if (!PARTS) ok = next();
                if (!ok) break;
                auto column = [&](int j) { if (!PARTS) tmem_ld32(src + (u32)first(j), reinterpret_cast<u32 (&)[32]>(z[j])); };
                if (R == Role::Lse) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        column(j);
                        const int col = n * TILE + first(j), left = g.cols - col;
                        if (left < 32) {
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (i >= left) z[j][i] = -INFINITY;
                        }
                        float mx[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) mx[i] = z[j][i];
#pragma unroll
                        for (int i = 4; i < 32; ++i) mx[i & 3] = fmaxf(mx[i & 3], z[j][i]);
                        const float m = fmaxf(top, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * LOG2E);
                        const float from = m == -INFINITY ? 0.0f : m;
                        float part[4] = {sum * exp2_fast(top - from), 0.0f, 0.0f, 0.0f};
                        const int64_t at = target - col;
                        if (mine && at >= 0 && at < min(32, left)) g.hit[row] = pick(z[j], (int)at);
#pragma unroll
                        for (int i = 0; i < 32; ++i) part[i & 3] += exp2_fast(fmaf(z[j][i], LOG2E, -from));
                        sum = (part[0] + part[1]) + (part[2] + part[3]);
                        top = m;
                    }
                } else if (R == Role::Grad) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int col = n * TILE + first(2 * x);       // of the piece
                        if (col >= g.held) break;
                        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                        __syncwarp();
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int left = g.cols - (g.v0 + col + 32 * h);
                            const int64_t at = target - (g.v0 + col + 32 * h);
                            float (&v)[32] = z[2 * x + h];
                            column(2 * x + h);
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] = exp2_fast((v[i] - lse) * LOG2E);
                            if (at >= 0 && at < 32) {
#pragma unroll
                                for (int i = 0; i < 32; ++i) v[i] -= i == (int)at ? 1.0f : 0.0f;
                            }
                            __syncwarp();
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] = skip || i >= left ? 0.0f : v[i] * weight;
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                sts128(stg + (u32)(lane * 128 + (((4 * h + j) ^ (lane & 7)) << 4)),
                                       make_uint4(pack2<T>(v[8 * j], v[8 * j + 1]), pack2<T>(v[8 * j + 2], v[8 * j + 3]),
                                                  pack2<T>(v[8 * j + 4], v[8 * j + 5]), pack2<T>(v[8 * j + 6], v[8 * j + 7])));
                        }
                        fence_async_smem();
                        __syncwarp();
                        if (lane == 0 && row0 < g.rows) {
                            asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];"
                                         ::"l"(&g.c), "r"(col), "r"(row0), "r"(0), "r"(stg) : "memory");
                            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                        }
                    }
                } else if (R == Role::Acc) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int col = n * TILE + first(x);
                        if (col >= g.cols) break;
                        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                        __syncwarp();
                        const float (&v)[32] = z[x];
                        column(x);
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            sts128(stg + (u32)(lane * 128 + ((j ^ (lane & 7)) << 4)),
                                   make_uint4(__float_as_uint(v[4 * j] * unscale), __float_as_uint(v[4 * j + 1] * unscale),
                                              __float_as_uint(v[4 * j + 2] * unscale), __float_as_uint(v[4 * j + 3] * unscale)));
                        fence_async_smem();
                        __syncwarp();
                        if (lane == 0 && row0 < g.rows) {
                            // one addition per element and launch: the order of the pieces
                            if (g.add)
                                asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.bulk_group [%0, {%1, %2, %3}], [%4];"
                                             ::"l"(&g.c), "r"(col), "r"(row0), "r"(t.split), "r"(stg) : "memory");
                            else
                                asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];"
                                             ::"l"(&g.c), "r"(col), "r"(row0), "r"(t.split), "r"(stg) : "memory");
                            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                        }
                    }
                } else {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int col = n * TILE + first(2 * x);
                        if (col >= g.cols) break;
                        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                        __syncwarp();
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float (&v)[32] = z[2 * x + h];
                            column(2 * x + h);
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] *= unscale;
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                sts128(stg + (u32)(lane * 128 + (((4 * h + j) ^ (lane & 7)) << 4)),
                                       make_uint4(pack2<T>(v[8 * j], v[8 * j + 1]), pack2<T>(v[8 * j + 2], v[8 * j + 3]),
                                                  pack2<T>(v[8 * j + 4], v[8 * j + 5]), pack2<T>(v[8 * j + 6], v[8 * j + 7])));
                        }
                        if (g.tma_out) {
                            fence_async_smem();
                            __syncwarp();
                            if (lane == 0 && row0 < g.rows) {
                                asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];"
                                             ::"l"(&g.c), "r"(col), "r"(g.out_row + row0), "r"(0), "r"(stg) : "memory");
                                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                            }
                        } else {
                            // a row of 64 columns at a time, two a lane
                            __syncwarp();
                            const bool words = ((reinterpret_cast<uintptr_t>(g.out) | (uintptr_t)(g.out_ld * 2)) & 3) == 0;
                            const int left = g.cols - col - 2 * lane;
                            T* out = static_cast<T*>(g.out) + (g.out_row + (int64_t)row0) * g.out_ld + col + 2 * lane;
                            const int rows = min(32, g.rows - row0);
                            for (int r = 0; r < rows; ++r) {
                                u32 w;
                                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w)
                                             : "r"(stg + (u32)(r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4)) : "memory");
                                if (words && left > 1) {
                                    *reinterpret_cast<u32*>(out) = w;
                                } else {
                                    if (left > 0) reinterpret_cast<unsigned short*>(out)[0] = (unsigned short)w;
                                    if (left > 1) reinterpret_cast<unsigned short*>(out)[1] = (unsigned short)(w >> 16);
                                }
                                out += g.out_ld;
                            }
                            __syncwarp();
                        }
                    }
                }
                if (!PARTS) taken();
            }
            if (R == Role::Lse && ok && mine) g.part[(int64_t)(t.run * 2 + half) * g.rows + row] = make_float2(top, sum);
        }
        if (R != Role::Lse && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
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

// The same products the other way round, for up to 128 rows: features (words
// of the vocabulary; dx: its columns) on the instruction's M side, all rows,
// rounded up to 32, on its N side.  The weights' bytes bound these calls, so
// what a stage of the ring holds of rows, and what the instruction spends on
// rows that are not there, goes to weights: two k-blocks a stage.  Lane and
// column have changed places, so Lse sums over lanes, and g and dx leave as 32
// neighbours of a row.  (16 x 4096 x 32768: 61.9 -> 52.5 us, 128 rows 61.8 ->
// 56.  With more rows, in tiles that fit them better than 256, the sums over lanes
// took longer than what was saved: 777 x 1150 x 50001 167 -> 216 us.)
template <int ROWS> struct Turned {
    static constexpr int KPS = 2;                                      // k-blocks per stage
    static constexpr u32 B_BYTES = ROWS / 2 * 128, STAGE_BYTES = KPS * (A_BYTES + B_BYTES);
    static constexpr int STAGES = ROWS == 128 ? 4 : 5;
    static constexpr int SMEM_BYTES = 1024 + STAGES * (int)STAGE_BYTES + 512;
    static_assert(SMEM_BYTES <= 227 * 1024, "shared memory");
};

// 16 values a lane to sums over the lanes: lanes 2 c and 2 c + 1 get column c's.
__device__ __forceinline__ float sum_columns(float (&v)[16], int lane) {
#pragma unroll
    for (int o = 16, n = 8; n; o >>= 1, n >>= 1)
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const bool up = lane & o;
            const float keep = up ? v[i + n] : v[i], give = up ? v[i] : v[i + n];
            v[i] = keep + __shfl_xor_sync(0xFFFFFFFFu, give, o);
        }
    return v[0] + __shfl_xor_sync(0xFFFFFFFFu, v[0], 1);
}
// Largest of the lanes' values (NaN counts for nothing).
__device__ __forceinline__ float largest(float v) {
    u32 b = __float_as_uint(fmaxf(v, -INFINITY));
    b ^= (u32)((int)b >> 31) | 0x80000000u;
    b = __reduce_max_sync(0xFFFFFFFFu, b);
    b ^= b & 0x80000000u ? 0x80000000u : 0xFFFFFFFFu;
    return __uint_as_float(b);
}

template <class T, Role R, bool PARTS, bool A_MN, int ROWS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1) turned_kernel(const __grid_constant__ CeArgs g) {
    using namespace bafe::tc;
    constexpr int PART = PARTS ? CHUNK<T, R> : 1 << 30;
    second_may_start();
    constexpr int ST = Turned<ROWS>::STAGES, KPS = Turned<ROWS>::KPS, BLOCKS = ROWS / 32;
    constexpr u32 BB = Turned<ROWS>::B_BYTES, SB = Turned<ROWS>::STAGE_BYTES;
    extern __shared__ unsigned char smem_raw[];
    const u32 raw_addr = smem_u32(smem_raw);
    const u32 base = (raw_addr + 1023u) & ~1023u;
    unsigned char* smem = smem_raw + (base - raw_addr);
    const u32 bars = base + ST * SB;
    auto FULL = [&](int s) { return bars + 8u * s; };
    auto EMPTY = [&](int s) { return bars + 8u * (ST + s); };
    auto TFULL = [&](int b) { return bars + 8u * (2 * ST + b); };
    auto TEMPTY = [&](int b) { return bars + 8u * (2 * ST + 2 + b); };
    const u32 DRAIN = bars + 8u * (2 * ST + 4);
    volatile Shared* sh = reinterpret_cast<volatile Shared*>(smem + ST * SB + 8 * (2 * ST + 5));
    volatile float* part = reinterpret_cast<volatile float*>(sh + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const u32 cta = cluster_rank();
    const int pair = (int)(blockIdx.x >> 1), num_pairs = (int)(gridDim.x >> 1);

    if (threadIdx.x == 0) {
        for (int s = 0; s < ST; ++s) {
            mbar_init(FULL(s), 1);
            mbar_init(EMPTY(s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(TFULL(b), 1);
            mbar_init(TEMPTY(b), 16);                    // the 8 epilogue warps of both CTAs
        }
        mbar_init(DRAIN, 1);
        sh->abort = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32((const void*)&sh->tmem_base)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();                                      // both CTAs' barriers exist
    tc_fence_after();
    const u32 tmem = sh->tmem_base;
    first_is_done();

    // A unit: a tile of features; Lse: `run` of them; Acc: a part of its contraction.
    auto unit_at = [&](int u) {
        Unit t;
        t.n = 0;
        t.split = R == Role::Acc ? u / g.m_tiles : 0;
        t.run = R == Role::Acc ? u % g.m_tiles : u;
        t.m = R == Role::Lse ? t.run * g.run : t.run;    // first feature tile
        t.count = R == Role::Lse ? min(g.run, g.m_tiles - t.m) : 1;
        return t;
    };
    // in stages of KPS k-blocks; what is behind the last is read as 0
    const int all = (g.kblocks + KPS - 1) / KPS;
    auto k_first = [&](const Unit& t) { return R == Role::Acc ? (int)((int64_t)all * t.split / g.splits) : 0; };
    auto k_end = [&](const Unit& t) { return R == Role::Acc ? (int)((int64_t)all * (t.split + 1) / g.splits) : all; };

    if (warp == 0) {
        // ---------------------------------------- TMA producer (both CTAs) --
        int s = 0;
        u32 phase = 0;
        bool ok = true;
        u32 armed[ST];
#pragma unroll
        for (int i = 0; i < ST; ++i) armed[i] = 0xFFFFFFFFu;
        const u32 both = KPS * (2 * A_BYTES + (u32)g.tile_n * 128u);   // bytes of both CTAs
        for (int u = pair; lane == 0 && ok && u < g.units; u += num_pairs) {
            const Unit t = unit_at(u);
            const int rb = (int)cta * (g.tile_n / 2), k1 = k_end(t);
            for (int m = t.m; m < t.m + t.count && ok; ++m) {
                const int fa = m * TILE + (int)cta * (TILE / 2);
                for (int ks = k_first(t); ks < k1; ++ks) {
                    if (!wait<false>(EMPTY(s), phase ^ 1u, sh, g, 1u)) { ok = false; break; }
                    const u32 a_dst = base + s * SB, b_dst = a_dst + KPS * A_BYTES;
                    if (cta == 0) mbar_expect_tx(FULL(s), both);
#pragma unroll
                    for (int h = 0; h < KPS; ++h) {
                        const int k = (ks * KPS + h) * BK;
                        if (A_MN) {
#pragma unroll
                            for (int j = 0; j < 2; ++j)
                                tma_load_3d_pair(a_dst + h * A_BYTES + j * MN_BOX, &g.a, FULL(s), fa + 64 * j, g.b_row + k, 0);
                        } else {
                            tma_load_3d_pair(a_dst + h * A_BYTES, &g.a, FULL(s), k, g.b_row + fa, 0);
                        }
                        tma_load_3d_pair(b_dst + h * BB, &g.b, FULL(s), k, rb, 0);
                    }
                    armed[s] = phase;
                    if (++s == ST) { s = 0; phase ^= 1u; }
                }
            }
        }
        // Drain (bounded): copies in flight, both CTAs' on the leader's barriers.
        if (lane == 0 && cta == 0) {
#pragma unroll
            for (int i = 0; i < ST; ++i) {
                const u64 t0 = now_ns();
                if (armed[i] != 0xFFFFFFFFu)
                    while (!mbar_try(FULL(i), armed[i]) && now_ns() - t0 < drain_ns(g)) {}
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // --------------------------------------- MMA issuer (leader CTA) --
        if (lane == 0 && cta == 0) {
            constexpr u32 FMT = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
            constexpr u32 A_LBO = A_MN ? MN_BOX : 16u, A_KK = (A_MN ? 2048u : 32u) >> 4, B_KK = 32u >> 4;
            const u64 a_first = smem_desc(base, A_LBO, 1024u, 2u), b_first = smem_desc(base + KPS * A_BYTES, 16u, 1024u, 2u);
            const u32 idesc = instr_desc(A_MN, 0, g.tile_n, 256, FMT);
            u64 a = a_first, b = b_first;
            int s = 0;
            u32 phase = 0, count = 0;
            bool ok = true;
            for (int u = pair; ok && u < g.units; u += num_pairs) {
                const Unit t = unit_at(u);
                for (int m = 0; m < t.count && ok; ++m) {
                    const int first = k_first(t), last = k_end(t);
                    for (int k0 = first, k1; k0 < last; k0 = k1) {
                        k1 = last - k0 > PART / KPS ? k0 + PART / KPS : last;
                        const u32 buf = count & 1u;
                        if (!wait<true>(TEMPTY(buf), ((count >> 1) & 1u) ^ 1u, sh, g, 2u)) { ok = false; break; }
                        tc_fence_after();
                        const u32 d = tmem + buf * 256u;
                        for (int ks = k0; ks < k1; ++ks) {
                            if (!wait<true>(FULL(s), phase, sh, g, 3u)) { ok = false; break; }
                            tc_fence_after();
#pragma unroll
                            for (int kk = 0; kk < 4 * KPS; ++kk)
                                tc_mma_f16kind_pair(d, a + (kk >> 2) * (A_BYTES >> 4) + (kk & 3) * A_KK, b + (kk >> 2) * (BB >> 4) + (kk & 3) * B_KK,
                                                    idesc, ks > k0 || kk > 0 ? 1u : 0u);
                            tc_commit_pair(EMPTY(s));    // both CTAs' stage s is free
                            a += SB >> 4;
                            b += SB >> 4;
                            if (++s == ST) { s = 0; phase ^= 1u; a = a_first; b = b_first; }
                        }
                        if (!ok) break;
                        tc_commit_pair(TFULL(buf));
                        ++count;
                    }
                }
            }
            tc_commit_pair(DRAIN);
            const u64 t0 = now_ns();
            while (!mbar_try(DRAIN, 0u) && now_ns() - t0 < drain_ns(g)) {}
        }
        __syncwarp();
    } else {
        // ---------------------------------- epilogue (both CTAs, 8 warps) --
        // A thread has one feature of the tile (TMEM's lane); the two warps of
        // a lane quarter take turns along the rows, 16 at a time: column c of
        // part i is row 32 i + 16 half + c.
        const int q = warp & 3, half = (warp - 2) >> 2;
        float2 scale = make_float2(1.0f, 1.0f);
        if (R != Role::Lse) scale = scales_of(g, part);
        const float unscale = scale.y;
        u32 count = 0;
        bool ok = true;
        for (int u = pair; ok && u < g.units; u += num_pairs) {
            const Unit t = unit_at(u);
            const int row0 = half * 16;
            float top[BLOCKS], sum[BLOCKS];                // Lse: of column lane / 2 of each part
#pragma unroll
            for (int i = 0; i < BLOCKS; ++i) {
                top[i] = -INFINITY;
                sum[i] = 0.0f;
            }
            const int k0 = k_first(t), k1 = k_end(t);
            for (int m = t.m; m < t.m + t.count; ++m) {
                const int f0 = m * TILE + (int)cta * (TILE / 2) + q * 32, f = f0 + lane;
                float z[BLOCKS][16];                      // the sums of the contraction's parts
                u32 src = 0u;
                auto next = [&]() {                      // the next sums are there
                    const u32 buf = count & 1u;
                    const bool ready = wait<false>(TFULL(buf), (count >> 1) & 1u, sh, g, 4u);
                    if (!__all_sync(0xFFFFFFFFu, ready)) return false;
                    tc_fence_after();
                    src = tmem + ((u32)(q * 32) << 16) + buf * 256u + (u32)half * 16u;
                    return true;
                };
                auto taken = [&]() {                     // their columns may be written again
                    const u32 buf = count & 1u;
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        if (cta == 0) mbar_arrive(TEMPTY(buf));
                        else mbar_arrive_cluster(TEMPTY(buf), 0u);
                    }
                    ++count;
                };
                for (int ks = k0; PARTS && ks < k1; ks += PART / KPS) {
                    if (!next()) { ok = false; break; }
#pragma unroll
                    for (int i = 0; i < BLOCKS; ++i) {
                        if (32 * i >= g.tile_n) break;
                        u32 v[16];
                        tmem_ld16(src + 32u * i, v);
                        if (ks == k0) {
#pragma unroll
                            for (int c = 0; c < 16; ++c) z[i][c] = __uint_as_float(v[c]);
                        } else {
#pragma unroll
                            for (int c = 0; c < 16; c += 2) bafe::fadd2_rn(z[i][c], z[i][c + 1], v[c], v[c + 1]);
                        }
                    }
                    taken();
                }
                if (!PARTS) ok = next();
                if (!ok) break;
                if (R != Role::Lse) {
#pragma unroll (PARTS ? BLOCKS : 1)
                    for (int i = 0; i < BLOCKS; ++i) {
                        const int part0 = row0 + 32 * i;
                        if (32 * i >= g.tile_n || part0 >= g.rows) break;
                        float v[16];
                        if (!PARTS) tmem_ld16(src + 32u * i, reinterpret_cast<u32 (&)[16]>(v));
#pragma unroll
                        for (int c = 0; PARTS && c < 16; ++c) v[c] = z[i][c];
                        if (R == Role::Grad) {
                            // what this lane knows of column lane % 16: its target (-1: none, -2:
                            // ignored, where nothing that lse and z hold counts), dloss and lse
                            int target = -1;
                            float weight = 0.0f, lse = 0.0f;
                            const int row = part0 + (lane & 15);
                            if (row < g.rows) {
                                const int64_t word = target_of(g, row);
                                const bool in = word >= 0 && word < g.cols;
                                target = word == g.ignore ? -2 : in ? (int)word : -1;
                                lse = g.lse[row];
                                weight = in ? g.dloss[row * g.dloss_stride] * scale.x : NAN;
                            }
                            T* out = static_cast<T*>(g.out) + (int64_t)part0 * g.out_ld + f;
                            const int word = g.v0 + f;
#pragma unroll
                            for (int c = 0; c < 16; ++c) {
                                const int aim = __shfl_sync(0xFFFFFFFFu, target, c);
                                const float by = __shfl_sync(0xFFFFFFFFu, weight, c), from = __shfl_sync(0xFFFFFFFFu, lse, c);
                                float p = exp2_fast((v[c] - from) * LOG2E);
                                p -= aim == word ? 1.0f : 0.0f;
                                p = aim == -2 || word >= g.cols ? 0.0f : p * by;
                                if (part0 + c < g.rows && f < g.held) out[c * g.out_ld] = from_f32<T>(p);
                            }
                        } else if (R == Role::Acc) {
                            float* out = g.acc + t.split * g.acc_stride + (int64_t)part0 * g.out_ld + f;
                            float old[16];
#pragma unroll
                            for (int c = 0; c < 16; ++c)     // one addition per element and launch: the order of the pieces
                                old[c] = g.add && part0 + c < g.rows && f < g.cols ? out[c * g.out_ld] : 0.0f;
#pragma unroll
                            for (int c = 0; c < 16; ++c)
                                if (part0 + c < g.rows && f < g.cols) out[c * g.out_ld] = fmaf(v[c], unscale, old[c]);
                        } else {
                            T* out = static_cast<T*>(g.out) + (int64_t)part0 * g.out_ld + f;
#pragma unroll
                            for (int c = 0; c < 16; ++c)
                                if (part0 + c < g.rows && f < g.cols) out[c * g.out_ld] = from_f32<T>(v[c] * unscale);
                        }
                        __syncwarp();
                    }
                    if (!PARTS) taken();
                    continue;
                }
#pragma unroll
                for (int i = 0; i < BLOCKS; ++i) {
                    if (32 * i >= g.tile_n) break;
                    const int part0 = row0 + 32 * i;
                    int target = -1;
                    if (lane < 16 && part0 + lane < g.rows) {
                        const int64_t word = target_of(g, part0 + lane);
                        if (word >= f0 && word < f0 + 32 && word < g.cols) target = (int)word;
                    }
                    for (u32 mine = __ballot_sync(0xFFFFFFFFu, target >= 0); mine; mine &= mine - 1) {   // rare
                        const int c = __ffs(mine) - 1, word = __shfl_sync(0xFFFFFFFFu, target, c);
                        const float h = pick(z[i], c);
                        if (f == word) g.hit[part0 + c] = h;
                    }
                    float own = -INFINITY;               // the largest of column lane / 2, times log2 e
#pragma unroll
                    for (int c = 0; c < 16; ++c) {
                        const float v = f < g.cols ? z[i][c] : -INFINITY;
                        const float high = largest(v) * LOG2E, from = high > -INFINITY ? high : 0.0f;
                        z[i][c] = exp2_fast(fmaf(v, LOG2E, -from));
                        own = lane >> 1 == c ? high : own;
                    }
                    const float s = sum_columns(z[i], lane);
                    const float high = fmaxf(top[i], own), from = high > -INFINITY ? high : 0.0f;
                    sum[i] = sum[i] * exp2_fast(top[i] - from) + s * exp2_fast(own - from);
                    top[i] = high;
                }
            }
            if (R == Role::Lse && ok) {
#pragma unroll
                for (int i = 0; i < BLOCKS; ++i) {
                    const int row = row0 + 32 * i + (lane >> 1);
                    if (32 * i < g.tile_n && row < g.rows && !(lane & 1))
                        g.part[((int64_t)t.run * 8 + cta * 4 + q) * g.rows + row] = make_float2(top[i], sum[i]);
                }
            }
        }
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

// Joins the runs' maxima and sums of JOIN_ROWS rows: 128 threads a row, so
// that few rows with many runs do not wait for one another's exponentials.
constexpr int JOIN_ROWS = 8;
__device__ __forceinline__ float2 join(float2 a, float2 b) {
    const float m = fmaxf(a.x, b.x), from = m == -INFINITY ? 0.0f : m;
    return make_float2(m, a.y * exp2_fast(a.x - from) + b.y * exp2_fast(b.x - from));
}
__global__ void __launch_bounds__(1024) join_kernel(const float2* part, const float* hit, const void* target, int target_bytes,
                                                    int64_t ignore, float* loss, float* lse, int slots, int rows, int vocab) {
    __shared__ float2 all[JOIN_ROWS][33];
    first_is_done();
    const int x = threadIdx.x % JOIN_ROWS, y = threadIdx.x / JOIN_ROWS, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row = (int)blockIdx.x * JOIN_ROWS + x;
    float2 v = make_float2(-INFINITY, 0.0f);
    if (row < rows)
#pragma unroll 4
        for (int i = y; i < slots; i += 1024 / JOIN_ROWS) v = join(v, __ldcg(&part[(int64_t)i * rows + row]));
    // a fixed order: the lanes of a row in a warp, then the warps
#pragma unroll
    for (int o = JOIN_ROWS; o < 32; o <<= 1) v = join(v, make_float2(__shfl_xor_sync(0xFFFFFFFFu, v.x, o), __shfl_xor_sync(0xFFFFFFFFu, v.y, o)));
    if (lane < JOIN_ROWS) all[lane][warp] = v;
    __syncthreads();
    if (warp >= JOIN_ROWS) return;
    v = all[warp][lane];
    const int r = (int)blockIdx.x * JOIN_ROWS + warp;
    float m = v.x;
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    const float from = m == -INFINITY ? 0.0f : m;
    const float s = warp_sum(v.y * exp2_fast(v.x - from));
    if (lane == 0 && r < rows) {
        const float l = (float)(((double)m + (double)log2f(s)) / (double)LOG2E);
        lse[r] = l;
        const int64_t t = target_bytes == 8 ? static_cast<const int64_t*>(target)[r] : (int64_t)static_cast<const int*>(target)[r];
        loss[r] = t == ignore ? 0.0f : t >= 0 && t < vocab ? l - __ldcg(&hit[r]) : NAN;
    }
}

// range over the largest counted |dloss|, and its inverse.
__global__ void __launch_bounds__(1024) scale_kernel(const __grid_constant__ CeArgs g, float* scale) {
    __shared__ float top[32];
    second_may_start();
    float m = 0.0f;
#pragma unroll 8
    for (int i = threadIdx.x; i < g.losses; i += 1024) m = fmaxf(m, counted(g, i));
    m = warp_max_nan(m);
    if ((threadIdx.x & 31) == 0) top[threadIdx.x >> 5] = m;
    __syncthreads();
    if (threadIdx.x < 32) {
        m = warp_max_nan(top[threadIdx.x]);
        if (threadIdx.x == 0) {
            const float2 s = scales_of(m, g.range);
            scale[0] = s.x;
            scale[1] = s.y;
        }
    }
}

// Sums of the splits, rounded, four columns a thread; acc rows are acc_ld
// long, `stride` apart from split to split.
template <class T> __global__ void __launch_bounds__(256) round_kernel(const float* acc, int64_t acc_ld, int64_t stride, int splits, T* out,
                                                                       int64_t out_ld, int64_t rows, int width) {
    const int units = (width + 3) / 4, u = blockIdx.y * blockDim.x + threadIdx.x;
    const int64_t r = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    second_may_start();
    first_is_done();
    if (r >= rows || u >= units) return;
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int i = 0; i < splits; ++i) {
        const float4 v = __ldcg(reinterpret_cast<const float4*>(acc + i * stride + r * acc_ld + 4 * u));
        s.x += v.x;
        s.y += v.y;
        s.z += v.z;
        s.w += v.w;
    }
    T* o = out + r * out_ld + 4 * u;
    const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (4 * u + i < width) o[i] = from_f32<T>(v[i]);
}

// ------------------------------------------------------------- host side --

constexpr int64_t PIECE_BYTES = int64_t(1) << 29;       // of g at a time, where that holds MIN_PIECE words
constexpr int64_t MIN_PIECE = 4096;
constexpr int64_t OWN_SCALES = 8192;                    // rows whose largest |dloss| every CTA finds itself
constexpr int64_t PART_BYTES = int64_t(1) << 27;        // of the forward pass's sums

int64_t tiles_of(int64_t n, int64_t tile) { return (n + tile - 1) / tile; }
int64_t round256(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// Rows of a turned kernel's tile, a multiple of 32; 0 where rows are too many.
int turned_rows(int64_t rows) { return rows <= 128 ? (int)tiles_of(rows, 32) * 32 : 0; }

// Forward: tiles of the vocabulary, of a run of them, and the sums that a row's runs leave.
struct LsePlan {
    int turned, n_tiles, run, runs, slots;
};
LsePlan lse_plan(int64_t rows, int64_t vocab, int pairs) {
    const int64_t m = tiles_of(rows, TILE);
    LsePlan p;
    p.turned = turned_rows(rows);
    p.n_tiles = (int)tiles_of(vocab, TILE);
    // Turned: a run to a pair.  Else single tiles, as long as their sums fit into
    // PART_BYTES: pairs that walk along the vocabulary share less of the weights
    // (8192 x 4096 x 131072: runs of 16 7.0 ms, single tiles 6.5).
    const int64_t run = p.turned ? tiles_of(p.n_tiles, pairs) : tiles_of(2 * p.n_tiles * rows * 8, PART_BYTES);
    p.run = (int)(run < 1 ? 1 : run < p.n_tiles ? run : p.n_tiles);
    p.runs = (p.n_tiles + p.run - 1) / p.run;
    p.slots = p.runs * (p.turned ? 8 : 2);
    return p;
}

// Gradient: words of a piece, splits of dx's contraction, whether dx's sums
// need 32-bit memory.
struct GradPlan {
    int64_t piece, ld, acc_ld;
    int pieces, splits, turned;
    bool direct;
};
GradPlan grad_plan(int64_t rows, int64_t vocab, int64_t width, int pairs) {
    GradPlan p;
    p.turned = turned_rows(rows);
    int64_t most = PIECE_BYTES / 2 / (rows > 0 ? rows : 1) / TILE * TILE;
    if (most < MIN_PIECE) most = MIN_PIECE;
    p.pieces = (int)tiles_of(vocab, most);
    p.piece = tiles_of(tiles_of(vocab, p.pieces), TILE) * TILE;
    p.pieces = (int)tiles_of(vocab, p.piece);
    if (p.pieces == 1) p.piece = vocab;
    p.ld = tiles_of(p.piece, 64) * 64;
    const int64_t tiles = tiles_of(rows, TILE) * tiles_of(width, TILE), kblocks = tiles_of(p.piece, BK);
    // rounds of the pairs per whole contraction, and a little for each split's sums
    p.splits = 1;
    double best = (double)tiles_of(tiles, pairs);
    for (int s = 2; s <= 32 && tiles < 4 * pairs && 8 * s <= kblocks; ++s) {
        const double cost = (double)tiles_of(tiles * s, pairs) / s + 0.005 * s;
        if (cost < best) {
            best = cost;
            p.splits = s;
        }
    }
    p.direct = p.pieces == 1 && p.splits == 1;
    p.acc_ld = (width + 3) / 4 * 4;
    return p;
}

int check_sizes(const char* what, int64_t rows, int64_t vocab, int64_t width) {
    if (rows < 0 || rows > (int64_t(1) << 24) || vocab < 1 || vocab > (int64_t(1) << 24) || width < 1 || width > (int64_t(1) << 20))
        return fail(8, std::string(what) + ": sizes out of range (0 <= rows <= 2^24, 1 <= vocab <= 2^24, 1 <= width <= 2^20)");
    if (tiles_of(rows, TILE) * tiles_of(vocab, 128) > (int64_t(1) << 30)) return fail(8, std::string(what) + ": too many tiles");
    return 0;
}

struct Operands {
    Matrix x, w;
    int64_t copies;                    // workspace bytes of their aligned forms
};
Operands operands(const void* x, int64_t x_ld, const void* w, int64_t w_ld, int64_t rows, int64_t vocab, int64_t width) {
    Operands o;
    o.x = {x, rows > 1 ? x_ld : (width + 7) / 8 * 8, 0, rows, width, 1};
    o.w = {w, vocab > 1 ? w_ld : (width + 7) / 8 * 8, 0, vocab, width, 1};
    o.copies = copy_bytes(o.x, 2) + copy_bytes(o.w, 2);
    return o;
}

// after: the launch before is one of this file's too, on the same stream, and
// this one may be made ready while it ends (every kernel here waits for the one
// before, so all before that are done as well).
template <class K> int launch_pairs(const char* what, K kernel, const CeArgs& a, int pairs, int smem, bool after, cudaStream_t st) {
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = 2u * (unsigned)(a.units < pairs ? a.units : pairs);
    cfg.blockDim = THREADS;
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = after ? 1 : 0;
    cudaLaunchKernelEx(&cfg, kernel, a);                 // its error is read by launched
    return launched(what);
}

template <class T, Role R, bool PARTS, bool A_MN, bool B_MN>
int launch_parts(const char* what, const CeArgs& a, int pairs, int dev, cudaStream_t st, bool after) {
    auto k = ce_kernel<T, R, PARTS, A_MN, B_MN>;
    static bool ready[64] = {false};
    if (!ready[dev]) {
        if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES) != cudaSuccess) {
            cudaGetLastError();
            return fail(14, std::string(what) + ": cudaFuncSetAttribute");
        }
        ready[dev] = true;
    }
    return launch_pairs(what, k, a, pairs, SMEM_BYTES, after, st);
}
// The longest contraction of a unit, in k-blocks: splits are of whole ones, or of stages of two.
int longest(const CeArgs& a) { return a.splits == 1 ? a.kblocks : ((a.kblocks + 1) / 2 + a.splits - 1) / a.splits * 2; }
// PARTS: sums in parts, where the contraction is longer than one.
template <class T, Role R, bool A_MN, bool B_MN>
int launch(const char* what, const CeArgs& a, int pairs, int dev, cudaStream_t st, bool after = false) {
    if constexpr (R != Role::Lse)
        if (longest(a) <= CHUNK<T, R>) return launch_parts<T, R, false, A_MN, B_MN>(what, a, pairs, dev, st, after);
    return launch_parts<T, R, true, A_MN, B_MN>(what, a, pairs, dev, st, after);
}

template <class T, Role R, bool PARTS, bool A_MN, int ROWS>
int launch_turned_rows(const char* what, const CeArgs& a, int pairs, int dev, cudaStream_t st, bool after) {
    auto k = turned_kernel<T, R, PARTS, A_MN, ROWS>;
    static bool ready[64] = {false};
    if (!ready[dev]) {
        if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, Turned<ROWS>::SMEM_BYTES) != cudaSuccess) {
            cudaGetLastError();
            return fail(14, std::string(what) + ": cudaFuncSetAttribute");
        }
        ready[dev] = true;
    }
    return launch_pairs(what, k, a, pairs, Turned<ROWS>::SMEM_BYTES, after, st);
}
template <class T, Role R, bool PARTS, bool A_MN>
int launch_turned_parts(const char* what, const CeArgs& a, int pairs, int dev, cudaStream_t st, bool after) {
    if (a.tile_n <= 32) return launch_turned_rows<T, R, PARTS, A_MN, 32>(what, a, pairs, dev, st, after);
    return launch_turned_rows<T, R, PARTS, A_MN, 128>(what, a, pairs, dev, st, after);
}
template <class T, Role R, bool A_MN>
int launch_turned(const char* what, const CeArgs& a, int pairs, int dev, cudaStream_t st, bool after = false) {
    if constexpr (R != Role::Lse)
        if (longest(a) <= CHUNK<T, R>) return launch_turned_parts<T, R, false, A_MN>(what, a, pairs, dev, st, after);
    return launch_turned_parts<T, R, true, A_MN>(what, a, pairs, dev, st, after);
}
// Turns a launch's shape: its columns become the features.
void turn(CeArgs& a, int tile_rows) {
    a.tile_n = tile_rows;
    a.m_tiles = a.units = a.n_tiles;
    a.n_tiles = 1;
}

// Shape of a launch's result and contraction.
void shape(CeArgs& a, int64_t rows, int64_t cols, int64_t contraction, int group_m, unsigned long long limit) {
    a.rows = (int)rows;
    a.cols = (int)cols;
    a.m_tiles = (int)tiles_of(rows, TILE);
    a.n_tiles = (int)tiles_of(cols, TILE);
    a.group_m = group_m < a.m_tiles ? group_m : a.m_tiles;
    a.units = a.m_tiles * a.n_tiles;
    a.splits = 1;
    a.kblocks = (int)tiles_of(contraction, BK);
    a.timeout_ns = limit + contraction_ns(contraction);
}

// Tensor map of a result: 32 rows of 128 bytes.
int encode_result(TmaDesc* d, void* p, int es, int64_t ld, int64_t rows, int64_t cols, int64_t count, std::string& err) {
    uint64_t dims[3] = {(uint64_t)cols, (uint64_t)rows, (uint64_t)count};
    uint64_t strides[2] = {(uint64_t)(ld * es), (uint64_t)(rows * ld * es)};
    uint32_t box[3] = {(uint32_t)(128 / es), 32, 1};
    return tc_encode_tensor_map(d, es == 4 ? 1 : 2, 3, p, dims, strides, box, 1, err);
}

int start(CeArgs& a, int& dev, int& sms) {
    if (int rc = current_device(dev, sms)) return rc;
    memset(&a, 0, sizeof(a));
    a.err = device_error_word(dev);
    if (!a.err) return fail(6, "cannot allocate the device error word");
    return 0;
}

// Row tiles that pairs work on at a time, and share through L2: of the logits
// (8192 x 4096 x 131072: 8 6.59 ms, 12 6.52, 16 6.41, 24 6.53), and of dx and dw
// (4, 8 and 16 alike).
constexpr int GROUP_LOGITS = 16, GROUP_GRAD = 8;

template <class T>
int forward(CeArgs& a, const Operands& o, const LsePlan& p, float* loss, float* lse, int pairs, int dev, cudaStream_t st) {
    std::string err;
    int rc = encode(p.turned ? &a.b : &a.a, o.x, 2, (uint32_t)(p.turned ? p.turned / 2 : 128), err);
    if (!rc) rc = encode(p.turned ? &a.a : &a.b, o.w, 2, 128, err);
    if (rc) return fail(rc, err);
    shape(a, o.x.rows, o.w.rows, o.x.cols, GROUP_LOGITS, timeout_ns());
    a.run = p.run;
    a.runs = p.runs;
    if (p.turned) {
        turn(a, p.turned);
        a.units = p.runs;
        if (int rc2 = launch_turned<T, Role::Lse, false>("linear_cross_entropy", a, pairs, dev, st)) return rc2;
    } else {
        a.units = a.m_tiles * p.runs;
        if (int rc2 = launch<T, Role::Lse, false, false>("linear_cross_entropy", a, pairs, dev, st)) return rc2;
    }
    return launch_second("linear_cross_entropy: join", join_kernel, dim3((unsigned)tiles_of(a.rows, JOIN_ROWS)), dim3(1024), st, a.part,
                         a.hit, a.target, a.target_bytes, a.ignore, loss, lse, p.slots, a.rows, a.cols);
}

template <class T>
int backward(CeArgs a, const Operands& o, const GradPlan& p, void* g, float* acc, void* dx, int64_t dx_ld, void* dw, int64_t dw_ld,
             int pairs, int dev, cudaStream_t st) {
    const char* what = "linear_cross_entropy_grad";
    const int64_t rows = o.x.rows, vocab = o.w.rows, width = o.x.cols;
    const unsigned long long limit = timeout_ns();
    std::string err;
    for (int i = 0; i < p.pieces; ++i) {
        const int64_t v0 = i * p.piece, words = vocab - v0 < p.piece ? vocab - v0 : p.piece, held = tiles_of(words, 64) * 64;
        Matrix mg = {g, p.ld, 0, rows, held, 1};
        a.v0 = (int)v0;
        // g of the piece
        CeArgs s = a;
        int rc = encode(p.turned ? &s.b : &s.a, o.x, 2, (uint32_t)(p.turned ? p.turned / 2 : 128), err);
        if (!rc) rc = encode(p.turned ? &s.a : &s.b, o.w, 2, 128, err);
        if (!rc && !p.turned) rc = encode_result(&s.c, g, 2, p.ld, rows, held, 1, err);
        if (rc) return fail(rc, err);
        shape(s, rows, words, width, GROUP_LOGITS, limit);
        s.cols = (int)vocab;
        s.held = (int)held;
        s.b_row = (int)v0;
        if (p.turned) {
            turn(s, p.turned);
            s.out = g;
            s.out_ld = p.ld;
            if (int rc2 = launch_turned<T, Role::Grad, false>(what, s, pairs, dev, st, i > 0 || a.scale)) return rc2;
        } else if (int rc2 = launch<T, Role::Grad, false, false>(what, s, pairs, dev, st, i > 0 || a.scale)) {
            return rc2;
        }
        // dx, over the piece's words
        s = a;
        rc = encode(p.turned ? &s.b : &s.a, mg, 2, (uint32_t)(p.turned ? p.turned / 2 : 128), err);
        if (!rc) rc = encode(p.turned ? &s.a : &s.b, o.w, 2, 64, err);
        shape(s, rows, width, words, GROUP_GRAD, limit);
        s.b_row = (int)v0;
        if (p.turned) turn(s, p.turned);
        if (p.direct) {
            s.out = dx;
            s.out_ld = dx_ld;
            s.tma_out = !p.turned && aligned16(dx) && dx_ld % 8 == 0;
            if (!rc && s.tma_out) rc = encode_result(&s.c, dx, 2, dx_ld, rows, width, 1, err);
            if (rc) return fail(rc, err);
            if (int rc2 = p.turned ? launch_turned<T, Role::Out, true>(what, s, pairs, dev, st, true)
                                   : launch<T, Role::Out, false, true>(what, s, pairs, dev, st, true)) return rc2;
        } else {
            if (!rc && !p.turned) rc = encode_result(&s.c, acc, 4, p.acc_ld, rows, width, p.splits, err);
            if (rc) return fail(rc, err);
            s.acc = acc;
            s.acc_stride = rows * p.acc_ld;
            if (p.turned) s.out_ld = p.acc_ld;
            const int stages = (s.kblocks + 1) / 2;      // turned: two k-blocks each, one at least for every split
            s.splits = p.splits < stages ? p.splits : stages;
            s.units *= s.splits;
            s.add = i > 0;
            if (int rc2 = p.turned ? launch_turned<T, Role::Acc, true>(what, s, pairs, dev, st, true)
                                   : launch<T, Role::Acc, false, true>(what, s, pairs, dev, st, true)) return rc2;
            if (i + 1 == p.pieces) {
                const int units = (int)tiles_of(width, 4), x = units >= 128 ? 128 : units > 32 ? 64 : 32;
                if (int rc2 = launch_second(what, round_kernel<T>, dim3((unsigned)tiles_of(rows, 256 / x), (unsigned)tiles_of(units, x)),
                                            dim3(x, 256 / x), st, acc, p.acc_ld, rows * p.acc_ld, p.splits, static_cast<T*>(dx), dx_ld, rows,
                                            (int)width)) return rc2;
            }
        }
        // dw of the piece, over all rows
        s = a;
        rc = encode(&s.a, mg, 2, 64, err);
        if (!rc) rc = encode(&s.b, o.x, 2, 64, err);
        s.out = dw;
        s.out_ld = dw_ld;
        s.tma_out = aligned16(dw) && dw_ld % 8 == 0;
        if (!rc && s.tma_out) rc = encode_result(&s.c, dw, 2, dw_ld, v0 + words, width, 1, err);
        if (rc) return fail(rc, err);
        shape(s, words, width, rows, GROUP_GRAD, limit);
        s.out_row = (int)v0;
        if (int rc2 = launch<T, Role::Out, true, true>(what, s, pairs, dev, st, true)) return rc2;
    }
    return 0;
}

int check_call(const char* what, const void* x, int64_t x_ld, const void* w, int64_t w_ld, const void* target, int target_bytes,
               int64_t rows, int64_t vocab, int64_t width, int dtype) {
    if (dtype != BAFE_DTYPE_F16 && dtype != BAFE_DTYPE_BF16) return fail(8, std::string(what) + ": x and w must be f16 or bf16");
    if (target_bytes != 4 && target_bytes != 8) return fail(8, std::string(what) + ": targets must have 4 or 8 bytes");
    if (rows && (!x || !w || !target)) return fail(8, std::string(what) + ": null operand");
    if ((rows > 1 && x_ld < width) || (vocab > 1 && w_ld < width))
        return fail(8, std::string(what) + ": strides must be at least the rows' lengths");
    if (!element_aligned(2, {x, w}) || !element_aligned(target_bytes, {target}))
        return fail(8, std::string(what) + ": operands must start on a multiple of their element's size");
    return 0;
}

int64_t lse_bytes(const LsePlan& p, int64_t rows) { return round256((int64_t)p.slots * rows * 8) + round256(rows * 4); }
int64_t grad_bytes(const GradPlan& p, int64_t rows) {
    return 256 + round256(rows * p.ld * 2) + (p.direct ? 0 : round256(p.splits * rows * p.acc_ld * 4));
}

}  // namespace
}  // namespace lm
}  // namespace bafe_cuda

#define BAFE_API extern "C" __attribute__((visibility("default")))

using namespace bafe_cuda;
using namespace bafe_cuda::lm;

BAFE_API int64_t bafe_cuda_linear_cross_entropy_workspace(const void* x, int64_t x_ld, const void* w, int64_t w_ld, int64_t rows,
                                                          int64_t vocab, int64_t width, int gradient) {
    const char* what = gradient ? "linear_cross_entropy_grad" : "linear_cross_entropy";
    if (check_sizes(what, rows, vocab, width)) return -1;
    if (rows == 0) return 0;
    int dev = 0, sms = 0;
    if (current_device(dev, sms)) return -1;
    const int64_t copies = operands(x, x_ld, w, w_ld, rows, vocab, width).copies;
    return copies + (gradient ? grad_bytes(grad_plan(rows, vocab, width, sms / 2), rows) : lse_bytes(lse_plan(rows, vocab, sms / 2), rows));
}

BAFE_API int bafe_cuda_linear_cross_entropy(const void* x, int64_t x_ld, const void* w, int64_t w_ld, const void* target,
                                            int target_bytes, float* loss, float* lse, int64_t rows, int64_t vocab, int64_t width,
                                            int64_t ignore_index, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* what = "linear_cross_entropy";
    if (int rc = check_sizes(what, rows, vocab, width)) return rc;
    if (int rc = check_call(what, x, x_ld, w, w_ld, target, target_bytes, rows, vocab, width, dtype)) return rc;
    if (rows == 0) return 0;
    if (!loss || !lse) return fail(8, "linear_cross_entropy: null operand");
    if (!element_aligned(4, {loss, lse})) return fail(8, "linear_cross_entropy: operands must start on a multiple of their element's size");
    CeArgs a;
    int dev = 0, sms = 0;
    if (int rc = start(a, dev, sms)) return rc;
    Operands o = operands(x, x_ld, w, w_ld, rows, vocab, width);
    const LsePlan p = lse_plan(rows, vocab, sms / 2);
    if (!workspace || workspace_bytes < o.copies + lse_bytes(p, rows) || !aligned16(workspace))
        return fail(8, "linear_cross_entropy: workspace too small or unaligned (see bafe_cuda_linear_cross_entropy_workspace)");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    char* ws = static_cast<char*>(workspace);
    if (int rc = make_ready(what, o.x, 2, ws, sms, st)) return rc;
    if (int rc = make_ready(what, o.w, 2, ws, sms, st)) return rc;
    a.part = reinterpret_cast<float2*>(ws);
    a.hit = reinterpret_cast<float*>(ws + round256((int64_t)p.slots * rows * 8));
    a.target = target;
    a.target_bytes = target_bytes;
    a.ignore = ignore_index;
    return dtype == BAFE_DTYPE_BF16 ? forward<__nv_bfloat16>(a, o, p, loss, lse, sms / 2, dev, st)
                                    : forward<__half>(a, o, p, loss, lse, sms / 2, dev, st);
}

BAFE_API int bafe_cuda_linear_cross_entropy_grad(const float* dloss, int64_t dloss_stride, const void* x, int64_t x_ld, const void* w,
                                                 int64_t w_ld, const void* target, int target_bytes, const float* lse, void* dx,
                                                 int64_t dx_ld, void* dw, int64_t dw_ld, int64_t rows, int64_t vocab, int64_t width,
                                                 int64_t ignore_index, int dtype, void* workspace, int64_t workspace_bytes,
                                                 void* stream) {
    const char* what = "linear_cross_entropy_grad";
    if (int rc = check_sizes(what, rows, vocab, width)) return rc;
    if (int rc = check_call(what, x, x_ld, w, w_ld, target, target_bytes, rows, vocab, width, dtype)) return rc;
    if (!dw || (rows && (!dloss || !lse || !dx))) return fail(8, "linear_cross_entropy_grad: null operand");
    if ((rows > 1 && (dx_ld < width || dloss_stride < 0)) || (vocab > 1 && dw_ld < width))
        return fail(8, "linear_cross_entropy_grad: strides must be at least the rows' lengths");
    if (!element_aligned(2, {dx, dw}) || !element_aligned(4, {dloss, lse}))
        return fail(8, "linear_cross_entropy_grad: operands must start on a multiple of their element's size");
    CeArgs a;
    int dev = 0, sms = 0;
    if (int rc = start(a, dev, sms)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (vocab == 1) dw_ld = (width + 7) / 8 * 8;
    if (rows == 0) {
        const cudaError_t e = cudaMemset2DAsync(dw, (size_t)dw_ld * 2, 0, (size_t)width * 2, (size_t)vocab, st);
        return e == cudaSuccess ? 0 : (cudaGetLastError(), fail(7, "linear_cross_entropy_grad: cudaMemset2DAsync"));
    }
    if (rows == 1) dx_ld = (width + 7) / 8 * 8;
    Operands o = operands(x, x_ld, w, w_ld, rows, vocab, width);
    const GradPlan p = grad_plan(rows, vocab, width, sms / 2);
    if (!workspace || workspace_bytes < o.copies + grad_bytes(p, rows) || !aligned16(workspace))
        return fail(8, "linear_cross_entropy_grad: workspace too small or unaligned (see bafe_cuda_linear_cross_entropy_workspace)");
    char* ws = static_cast<char*>(workspace);
    if (int rc = make_ready(what, o.x, 2, ws, sms, st)) return rc;
    if (int rc = make_ready(what, o.w, 2, ws, sms, st)) return rc;
    float* scale = reinterpret_cast<float*>(ws);
    void* g = ws + 256;
    float* acc = reinterpret_cast<float*>(ws + 256 + round256(rows * p.ld * 2));
    a.dloss = dloss;
    a.dloss_stride = dloss_stride;
    a.target = target;
    a.target_bytes = target_bytes;
    a.lse = lse;
    a.ignore = ignore_index;
    a.range = dtype == BAFE_DTYPE_BF16 ? 1.0f : 32768.0f;   // |p - onehot| is 1 at most
    a.losses = (int)rows;
    a.vocab = (int)vocab;
    if (rows > OWN_SCALES) {
        scale_kernel<<<1, 1024, 0, st>>>(a, scale);
        if (int rc = launched(what)) return rc;
        a.scale = scale;
    }
    if (dtype == BAFE_DTYPE_BF16) return backward<__nv_bfloat16>(a, o, p, g, acc, dx, dx_ld, dw, dw_ld, sms / 2, dev, st);
    return backward<__half>(a, o, p, g, acc, dx, dx_ld, dw, dw_ld, sms / 2, dev, st);
}
