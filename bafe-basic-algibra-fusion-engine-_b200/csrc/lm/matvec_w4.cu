// matvec_w4.cu -- a few rows of activations times 4-bit weights that have a
// scale, and optionally a zero point, for each group of columns:
//
//   y[m][n] = xs[m] * sum_g s[n][g] * sum_{k in g} (q[n][k] - z[n][g]) * x[m][k]
//
// (z = 8 without zero points; xs only for e4m3 rows).  Byte j of a weight
// row holds k = 2j in its low and k = 2j + 1 in its high four bits.
//
// Bound by memory: the weights are half a byte each and used for a handful
// of multiply-adds.  At full bandwidth a B200 SM takes in about 46 weights a
// clock, 2.8 lane-instructions each, so unpacking and multiplying have to
// stay well below that.  Both go through 8-bit integers: four weights come
// out of a 32-bit word with one logic operation (and a shift for the other
// four), and mma.sync m16n8k32 (u8 x s8 -> s32) multiplies them (weights as
// the 16 rows, tokens as the 8 columns).  Weights as 16-bit floats would take
// two to three operations for every two weights (exponent, subtraction of
// the zero point) and twice the instructions of a fused multiply-add per
// token.  tcgen05 has nothing to add here: its operands would have to be
// unpacked into shared memory first.
//
// The tokens are made 24-bit fixed-point numbers for it, once per block:
// each 128 consecutive k of a token share a power of two that brings the
// largest near 2^22, every value is rounded to the nearest integer X (e4m3
// values are integers then: no rounding; f16 and bf16 values within 2^-11 and
// 2^-14 of the largest one neither; smaller ones are off by at most 2^-22 of
// the largest, as in a 32-bit sum they would be), and X is cut into three
// signed bytes.  The sums of q times each byte over 128 k are exact 32-bit
// integers.  Each is freed of the zero point (z times the sum of those bytes)
// while everything is still exact, so that weights equal to their zero point
// give zeros; then they are joined and scaled in 32-bit floating point.  A row
// that holds an infinity or a NaN gives NaN.
//
// One or two tokens put their bytes side by side into the instruction's eight
// columns (column 3 token + byte) instead of using it once for each byte: a
// third of the multiplications, and the bytes' sums are only joined at a
// tile's end (1 x 32768 x 8192: 44 us without).
//
// The order of k inside an instruction is free as long as both operands
// agree, so the weights are used as they lie in memory: a lane takes whole
// words, k = 0 2 4 6 as one register and 1 3 5 7 as the other, and the tokens'
// bytes are laid out in that order.  All 32 k of one instruction must belong
// to one group, whose scale multiplies its sums: groups of a multiple of 128
// let each lane load 16 bytes (4 lanes: 128 k), groups of 64 8 bytes, other
// multiples of 32 4 bytes.
//
// A block's warps form teams.  A team walks tiles of 32 rows (two of the
// instruction's, so that the tokens' bytes, three for every half-byte weight
// and token tile, are read from shared memory half as often); each of its
// warps has a part of the tile's k-blocks of 128, and they add their sums
// through shared memory, behind a barrier of the team's own.
// Small teams wait less for one another, large ones spread few tiles over
// more warps: w4_shape weighs both.  The weights of the next steps travel into shared memory with
// asynchronous copies, each thread into slots of its own, so that no barrier
// guards them and the bytes in flight do not cost registers.  Scales and zero
// points come four at a time, one row a lane, and are made numbers once, in
// shared memory: fetched for each k-block by itself, every 2 bytes cost a
// sector of 32 and doubled the traffic into the SM (8 x 32768 x 8192: 73 us,
// 37 without them).  Where the tiles are too few for the SMs, or the tokens' bytes would crowd out the weights', k is
// also cut into slices over blocks, whose sums a second kernel adds in slice
// order.
#include "common.cuh"

namespace bafe_cuda {
namespace lm {
namespace {

constexpr int MAX_TOKENS = 32;         // per launch
constexpr int TILE = 32;               // weight rows
constexpr int ROWS = 4;                // of them per lane: r, r + 8, r + 16, r + 24
constexpr int DEPTH = 3;               // k-blocks of a warp in flight or in use
constexpr int SEG = 4;                 // scale units of a row that are fetched together
constexpr int LIMBS = 3;               // bytes of a token's value
constexpr int WARPS = 16;              // a block's, one block per SM

struct W4Args {
    const void* x;
    const float* x_scale;              // or null
    const uint8_t* q;
    const void* scales;
    const uint8_t* zeros;              // or null: 8
    void* y;
    float* part;                       // [slices][tokens][n], when sliced
    int64_t x_ld, q_ld, s_ld, z_ld, y_ld;
    int64_t n, k;
    int qbytes;                        // bytes of a weight row
    int tokens;
    uint64_t group_inv;                // ceil(2^40 / (group / 32)): block of 32 -> group
    int scale_type;                    // BAFE dtype
    int x_type;                        // BAFE dtype or e4m3
    int out_bf16;
    int kblocks;                       // of 128
    int slice_kb;                      // k-blocks per slice
    int tiles;
    int team;                          // warps that share a tile
    int per_member;                    // k-blocks of each
    int unit_groups;                   // a scale unit is a whole group
    int groups;
};

__device__ __forceinline__ void mma_u8s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Integers as floats without a conversion instruction (a quarter or less of
// the rate of an addition): 0x4B400000 + v, for |v| < 2^22, is the float
// 1.5 * 2^23 + v.  The sums start from that integer.
constexpr int BIAS_BITS = 0x4B400000;
constexpr float BIAS = 12582912.0f;
__device__ __forceinline__ float small_float(int biased) { return __int_as_float(biased) - BIAS; }
// The same from BIAS_BITS.
__device__ __forceinline__ void mma_u8s8_first(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(BIAS_BITS));
}
__device__ __forceinline__ uint32_t ldg32(const void* p) { return __ldg(static_cast<const uint32_t*>(p)); }
__device__ __forceinline__ uint32_t ldg16(const void* p) { return __ldg(static_cast<const unsigned short*>(p)); }
__device__ __forceinline__ uint32_t ldg8(const void* p) { return __ldg(static_cast<const uint8_t*>(p)); }

__device__ __forceinline__ float scale_f32(uint32_t raw, int type) {
    if (type == BAFE_DTYPE_F32) return __uint_as_float(raw);
    if (type == BAFE_DTYPE_BF16) return __uint_as_float(raw << 16);
    return __half2float(__ushort_as_half((unsigned short)raw));
}
__device__ __forceinline__ uint32_t load_scale(const void* row, int i, int type) {
    if (type == BAFE_DTYPE_F32) return ldg32(static_cast<const uint32_t*>(row) + i);
    return ldg16(static_cast<const unsigned short*>(row) + i);
}

template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src) {
    const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(d), "l"(src), "n"(BYTES) : "memory");
}

// Starts the copy of LW words (of 8 weights) from `src` into `dst`; `left`
// bytes of the row are there (none, where it is negative).  Wide: one copy of LW * 4 bytes (row starts and lengths are
// multiples of it).  Words: one word, copied where it lies inside the row,
// else put together byte by byte; Bytes: byte by byte.  Bytes behind the
// row's end become 0.
enum class Load { Wide, Words, Bytes };
template <int LW> struct alignas(4 * LW) WordsOf { uint32_t w[LW]; };
template <int LW, Load LD>
__device__ __forceinline__ void fetch_words(WordsOf<LW>* dst, const uint8_t* src, int left) {
    if constexpr (LD == Load::Wide) {
        if (left > 0) {
            copy_async<LW * 4>(dst, src);
        } else {
#pragma unroll
            for (int v = 0; v < LW; ++v) dst->w[v] = 0;
        }
    } else {
        static_assert(LW == 1, "one word at a time");
        if (LD == Load::Words && left >= 4) {
            copy_async<4>(dst, src);
        } else {
            uint32_t t = 0;
#pragma unroll
            for (int b = 0; b < 4; ++b)
                if (b < left) t |= ldg8(src + b) << (8 * b);
            dst->w[0] = t;
        }
    }
}

__device__ __forceinline__ void store_result(const W4Args& g, int tok, int64_t n, float v) {
    if (g.x_scale) v *= g.x_scale[tok];
    if (g.out_bf16) static_cast<__nv_bfloat16*>(g.y)[tok * g.y_ld + n] = __float2bfloat16_rn(v);
    else static_cast<__half*>(g.y)[tok * g.y_ld + n] = __float2half_rn(v);
}

template <class T>
__device__ __forceinline__ void load_tokens(const void* x, int64_t at, int64_t left, float (&f)[8]) {
    const T* p = static_cast<const T*>(x) + at;
    if (left >= 8 && (reinterpret_cast<uintptr_t>(p) & 15u) == 0) {
        unpack(*reinterpret_cast<const Pack<T, 8>*>(p), f);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = j < left ? to_f32(p[j]) : 0.0f;
    }
}

// e4m3: two values an instruction, eight bytes a load.
__device__ __forceinline__ void load_tokens_e4m3(const void* x, int64_t at, int64_t left, float (&f)[8]) {
    const uint8_t* p = static_cast<const uint8_t*>(x) + at;
    uint2 v = make_uint2(0u, 0u);                        // e4m3 0
    if (left >= 8 && (reinterpret_cast<uintptr_t>(p) & 7u) == 0) {
        v = *reinterpret_cast<const uint2*>(p);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < left) (j < 4 ? v.x : v.y) |= (uint32_t)p[j] << (8 * (j & 3));
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((j < 2 ? v.x : v.y) >> (16 * (j & 1))), __NV_E4M3);
        const float2 two = __half22float2(__half2(h));
        f[2 * j] = two.x;
        f[2 * j + 1] = two.y;
    }
}

template <int LW, int NT_, Load LD>
__global__ void __launch_bounds__(WARPS * 32, 1) matvec_w4_kernel(const W4Args g) {
    // NT token tiles of 8; 0: one or two tokens, bytes side by side
    constexpr bool NARROW = NT_ == 0;
    constexpr int NT = NARROW ? 1 : NT_, PASSES = NARROW ? 1 : LIMBS;
    constexpr int U = 4 / LW, TP = NT * 8;
    constexpr int E = ROWS * U;                          // pieces of LW words a thread holds per k-block
    extern __shared__ __align__(128) unsigned char smem[];
    constexpr int threads = WARPS * 32;
    if (g.part) second_may_start();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int team = warp / g.team, member = warp % g.team, teams = WARPS / g.team;
    const int r = lane >> 2, c = lane & 3;
    const int kb0 = blockIdx.y * g.slice_kb;
    const int nkb = min(g.kblocks - kb0, g.slice_kb);
    const int x_row = nkb * 128 + 16;                    // bytes per token and limb: 16 keep two tokens' reads apart
    // this thread's slots: [DEPTH][E][threads] pieces
    WordsOf<LW>* slots = reinterpret_cast<WordsOf<LW>*>(smem) + threadIdx.x;
    unsigned char* after = smem + (size_t)DEPTH * threads * E * LW * 4;
    // the warp's scales and zero points of SEG units: row i at (i % 8) * 4 + i / 8, a lane's four rows side by side
    float* seg_s = reinterpret_cast<float*>(after) + warp * (2 * SEG * TILE);
    float* seg_z = seg_s + SEG * TILE;
    unsigned char* xs = after + WARPS * 2 * SEG * TILE * 4;                     // [LIMBS][tokens][x_row]
    // Of each scale unit and column: the sums of the bytes that are multiplied
    // there (NARROW: one byte's), and the power of two of the k-block.  Two
    // columns' values lie side by side: {s0 s0' s1 s1' s2 s2' u u'}, {s s' u u'}.
    float* xt = reinterpret_cast<float*>(xs + ((LIMBS * g.tokens * x_row + 127) & ~127));
    constexpr int XT = NARROW ? 2 : LIMBS + 1;           // floats per column
    // the team's sums: [members but the first][lanes] of 8 NT floats
    float4* red = reinterpret_cast<float4*>(xt + nkb * U * TP * XT) + team * (g.team - 1) * 32 * 2 * NT;

    // this warp's k-blocks of a tile: [kb_from, kb_from + per_tile), as far as there are any
    const int per_tile = g.per_member, kb_from = member * per_tile;
    const int first_tile = team * gridDim.x + blockIdx.x, next_tile = gridDim.x * teams;   // blocks differ by one tile at most

    auto row_of = [&](int tile, int in) {
        const int64_t row = (int64_t)tile * TILE + in;
        return row < g.n ? row : g.n - 1;                // in bounds; its sums are not stored
    };
    // where the tile being fetched lies for this lane
    const uint8_t* f_q[ROWS];
    auto fetch = [&](int tile, int step, int d) {
        const int kbl = kb_from + step;
        if (tile < g.tiles && kbl < nkb) {               // the same for the whole warp
            if (step == 0) {
#pragma unroll
                for (int h = 0; h < ROWS; ++h) f_q[h] = g.q + row_of(tile, r + 8 * h) * g.q_ld + kb0 * 64 + c * (4 * LW);
            }
            WordsOf<LW>* dst = slots + d * E * threads;
#pragma unroll
            for (int h = 0; h < ROWS; ++h)
#pragma unroll
                for (int l = 0; l < U; ++l) {
                    const int at = kbl * 64 + l * (16 * LW);
                    fetch_words<LW, LD>(dst + (h * U + l) * threads, f_q[h] + at, g.qbytes - kb0 * 64 - c * (4 * LW) - at);
                }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // Scales and zero points of row `lane`, the SEG units from a step on:
    // asked for one segment ahead, put into shared memory as numbers at its
    // start.  wide: four of them in one load.
    uint32_t s_raw[SEG], z_raw[SEG];
    bool s_wide = false, z_wide = false;
    auto ask = [&](int tile, int step) {
        const int kbl = kb_from + step;
        if (tile >= g.tiles || kbl >= nkb) return;
        const int64_t row = row_of(tile, lane);
        const int unit = (kb0 + kbl) * U;                // of 32 LW k each
        const int first = g.unit_groups ? unit : 0;
        const int esize = g.scale_type == BAFE_DTYPE_F32 ? 4 : 2;
        const char* sr = static_cast<const char*>(g.scales) + (row * g.s_ld + first) * esize;
        const uint8_t* zr = g.zeros ? g.zeros + row * g.z_ld + first : nullptr;
        const bool four = g.unit_groups && first + SEG <= g.groups;
        s_wide = four && esize == 2 && (reinterpret_cast<uintptr_t>(sr) & 7u) == 0;
        z_wide = four && zr && (reinterpret_cast<uintptr_t>(zr) & 3u) == 0;
        if (s_wide) {
            const uint2 v = __ldg(reinterpret_cast<const uint2*>(sr));
            s_raw[0] = v.x;
            s_raw[1] = v.y;
        }
        if (z_wide) z_raw[0] = ldg32(zr);
        if (!s_wide || (zr && !z_wide)) {
#pragma unroll
            for (int o = 0; o < SEG; ++o) {
                // the unit's own group, or the one that it lies in
                const int group = g.unit_groups ? o : (int)(((uint64_t)((unit + o) * LW) * g.group_inv) >> 40);
                const bool there = first + group < g.groups;
                if (!s_wide) s_raw[o] = there ? load_scale(sr, group, g.scale_type) : 0u;
                if (zr && !z_wide) z_raw[o] = there ? ldg8(zr + group) : 0u;
            }
        }
    };
    auto put = [&]() {
        const int to = (lane & 7) * 4 + (lane >> 3);
#pragma unroll
        for (int o = 0; o < SEG; ++o) {
            const uint32_t s = s_wide ? (o & 1 ? s_raw[o / 2] >> 16 : s_raw[o / 2] & 0xFFFFu) : s_raw[o];
            const uint32_t z = !g.zeros ? 8u : z_wide ? (z_raw[0] >> (8 * o)) & 255u : z_raw[o];
            seg_s[o * TILE + to] = scale_f32(s, g.scale_type);
            seg_z[o * TILE + to] = small_float(BIAS_BITS + (int)z);
        }
    };

    // The first k-blocks are on their way while the tokens are laid out.
    int f_tile = first_tile, f_step = 0;
    auto fetch_next = [&](int d) {
        fetch(f_tile, f_step, d);
        if (++f_step == per_tile) { f_step = 0; f_tile += next_tile; }
    };
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) fetch_next(d);
    int tile = first_tile, at_step = 0;
    ask(tile, at_step);

    // Tokens: half a warp makes one k-block of one token, 8 k a lane; four
    // k-blocks' loads are in flight.
    constexpr int halves = threads / 16;
    const int jobs = g.tokens * nkb, in = lane & 15;
    for (int o0 = (int)(threadIdx.x >> 4); o0 < ((jobs + 1) & ~1); o0 += 4 * halves) {
        float f4[4][8];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int p = min(o0 + q * halves, jobs - 1), tok = p / nkb, kbl = p % nkb;
            const int64_t k = (int64_t)(kb0 + kbl) * 128 + in * 8, left = g.k - k;
            if (g.x_type == BAFE_DTYPE_BF16) load_tokens<__nv_bfloat16>(g.x, tok * g.x_ld + k, left, f4[q]);
            else if (g.x_type == BAFE_DTYPE_F16) load_tokens<__half>(g.x, tok * g.x_ld + k, left, f4[q]);
            else load_tokens_e4m3(g.x, tok * g.x_ld + k, left, f4[q]);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            // both halves of a warp stay together: the odd one out repeats the last
            if (o0 + q * halves >= ((jobs + 1) & ~1)) break;
            const int p = min(o0 + q * halves, jobs - 1), tok = p / nkb, kbl = p % nkb;
            const float (&f)[8] = f4[q];
            float top = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) top = max_nan(top, fabsf(f[j]));
#pragma unroll
            for (int d = 8; d; d >>= 1) top = max_nan(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
            // the largest in [2^e, 2^(e + 1)) becomes [2^21, 2^22); blocks
            // below 2^-103 keep that scale, which stays finite
            const int eb = max((int)(__float_as_uint(top) >> 23), 24);
            const bool finite = eb < 255;
            const float up = finite ? __uint_as_float((uint32_t)(275 - eb) << 23) : 0.0f;
            const float down = finite ? __uint_as_float((uint32_t)(eb - 21) << 23) : __uint_as_float(0x7FC00000u);
            uint32_t y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                // adding 1.5 * 2^23 leaves the rounded integer in the low bits
                const int v = __float_as_int(fmaf(finite ? f[j] : 0.0f, up, BIAS)) - BIAS_BITS;
                y[j] = (uint32_t)(v + 0x808080) ^ 0x808080u;  // three signed bytes
            }
            unsigned char* dst = xs + tok * x_row + kbl * 128 + in * 8;
            uint32_t even[LIMBS], odd[LIMBS];
            const uint32_t p0 = __byte_perm(y[0], y[2], 0x5140), p1 = __byte_perm(y[4], y[6], 0x5140);
            const uint32_t p2 = __byte_perm(y[1], y[3], 0x5140), p3 = __byte_perm(y[5], y[7], 0x5140);
            even[0] = __byte_perm(p0, p1, 0x5410);
            even[1] = __byte_perm(p0, p1, 0x7632);
            odd[0] = __byte_perm(p2, p3, 0x5410);
            odd[1] = __byte_perm(p2, p3, 0x7632);
            even[2] = __byte_perm(__byte_perm(y[0], y[2], 0x0062), __byte_perm(y[4], y[6], 0x0062), 0x5410);
            odd[2] = __byte_perm(__byte_perm(y[1], y[3], 0x0062), __byte_perm(y[5], y[7], 0x0062), 0x5410);
#pragma unroll
            for (int m = 0; m < LIMBS; ++m)
                *reinterpret_cast<uint2*>(dst + m * g.tokens * x_row) = make_uint2(even[m], odd[m]);
            // the bytes' sums over one unit's lanes, the first two (below 2^15) in one word
            auto bytes_of = [&](int m) { return __dp4a((int)even[m], 0x01010101, __dp4a((int)odd[m], 0x01010101, 0)); };
            int s01 = bytes_of(0) + bytes_of(1) * 65536, s2 = bytes_of(2);
#pragma unroll
            for (int d = 1; d < 4 * LW; d <<= 1) {
                s01 += __shfl_xor_sync(0xFFFFFFFFu, s01, d);
                s2 += __shfl_xor_sync(0xFFFFFFFFu, s2, d);
            }
            if (in % (4 * LW) == 0) {
                const int s0 = (short)s01, unit = kbl * U + in / (4 * LW);
                const float sum[LIMBS] = {(float)s0, (float)((s01 - s0) >> 16), (float)s2};
                if constexpr (NARROW) {
#pragma unroll
                    for (int m = 0; m < LIMBS; ++m) {
                        const int col = tok * LIMBS + m;
                        float* to = xt + (unit * TP + (col & ~1)) * XT + (col & 1);
                        to[0] = sum[m];
                        to[2] = down;
                    }
                } else {
                    float* to = xt + (unit * TP + (tok & ~1)) * XT + (tok & 1);
#pragma unroll
                    for (int m = 0; m < LIMBS; ++m) to[2 * m] = sum[m];
                    to[2 * LIMBS] = down;
                }
            }
        }
    }
    // columns behind the last token: finite, so that their sums are harmless
    const int used = NARROW ? LIMBS * g.tokens : g.tokens;
    for (int o = threadIdx.x; o < nkb * U * (TP - used); o += threads) {
        const int col = used + o % (TP - used);
        float* to = xt + (o / (TP - used) * TP + (col & ~1)) * XT + (col & 1);
#pragma unroll
        for (int m = 0; m < XT; ++m) to[2 * m] = 0.0f;
    }
    __syncthreads();

    // This lane's bytes of its token in each column tile.  Columns behind the
    // last token repeat it; their sums are not stored.
    const int x_limb = g.tokens * x_row;
    const unsigned char* xlane[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int tok = NARROW ? r / LIMBS : t * 8 + r;
        xlane[t] = xs + (NARROW ? r % LIMBS : 0) * x_limb + min(tok, g.tokens - 1) * x_row + c * (8 * LW);
    }
    // NARROW: what the bytes of this lane's columns 2c, 2c + 1 count
    float narrow_weight[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int limb = (2 * c + e) % LIMBS;
        narrow_weight[e] = limb == 0 ? 1.0f : limb == 1 ? 256.0f : 65536.0f;
    }
    float acc[NT][2 * ROWS];                             // [row h, token 2c + e] at 2 h + e
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 2 * ROWS; ++e) acc[t][e] = 0.0f;
    int d = 0;
    while (tile < g.tiles) {                             // the same for the whole team
        const int kbl = kb_from + at_step;
        asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory");
        int t1 = tile, next_step = at_step + 1;
        if (next_step == per_tile) { next_step = 0; t1 += next_tile; }
        // a segment is LW steps of U units
        if (at_step % LW == 0) {
            __syncwarp();                                // the last segment is read
            put();
            __syncwarp();
            if (at_step + LW < per_tile) ask(tile, at_step + LW);
            else ask(tile + next_tile, 0);
        }
        if (kbl < nkb) {
            float s[U][ROWS], z[U][ROWS];
#pragma unroll
            for (int l = 0; l < U; ++l) {
                const int o = (at_step % LW) * U + l;
                const float4 s4 = *reinterpret_cast<const float4*>(seg_s + o * TILE + 4 * r);
                const float4 z4 = *reinterpret_cast<const float4*>(seg_z + o * TILE + 4 * r);
                s[l][0] = s4.x; s[l][1] = s4.y; s[l][2] = s4.z; s[l][3] = s4.w;
                z[l][0] = z4.x; z[l][1] = z4.y; z[l][2] = z4.z; z[l][3] = z4.w;
            }
            const WordsOf<LW>* src = slots + d * E * threads;
#pragma unroll
            for (int l = 0; l < U; ++l) {
                WordsOf<LW> w[ROWS];
#pragma unroll
                for (int h = 0; h < ROWS; ++h) w[h] = src[(h * U + l) * threads];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    int sum[2][PASSES][4];
                    uint32_t xb[PASSES][2 * LW];         // this lane's LW units of 8 bytes of its token
#pragma unroll
                    for (int m = 0; m < PASSES; ++m) {
                        const unsigned char* p = xlane[t] + m * x_limb + kbl * 128 + l * (32 * LW);
                        if constexpr (LW == 1) {
                            const uint2 v = *reinterpret_cast<const uint2*>(p);
                            xb[m][0] = v.x; xb[m][1] = v.y;
                        } else {
#pragma unroll
                            for (int v = 0; v < LW / 2; ++v) {
                                const uint4 q = *reinterpret_cast<const uint4*>(p + 16 * v);
                                xb[m][4 * v] = q.x; xb[m][4 * v + 1] = q.y; xb[m][4 * v + 2] = q.z; xb[m][4 * v + 3] = q.w;
                            }
                        }
                    }
#pragma unroll
                    for (int v = 0; v < LW; ++v)
#pragma unroll
                        for (int p = 0; p < 2; ++p) {
                            const uint32_t lo = w[2 * p].w[v], hi = w[2 * p + 1].w[v];
                            const uint32_t a0 = lo & 0x0F0F0F0Fu, a1 = hi & 0x0F0F0F0Fu;
                            const uint32_t a2 = (lo >> 4) & 0x0F0F0F0Fu, a3 = (hi >> 4) & 0x0F0F0F0Fu;
#pragma unroll
                            for (int m = 0; m < PASSES; ++m) {
                                if (v == 0) mma_u8s8_first(sum[p][m], a0, a1, a2, a3, xb[m][0], xb[m][1]);
                                else mma_u8s8(sum[p][m], a0, a1, a2, a3, xb[m][2 * v], xb[m][2 * v + 1]);
                            }
                        }
                    // the byte sums and the power of two of this lane's two columns
                    Pair x_sum[PASSES], x_unit;
                    const float4* xv = reinterpret_cast<const float4*>(xt + ((kbl * U + l) * TP + t * 8 + 2 * c) * XT);
                    if constexpr (NARROW) {
                        const float4 v = xv[0];
                        x_sum[0] = pair(v.x, v.y);
                        x_unit = pair(v.z, v.w);
                    } else {
                        const float4 v = xv[0], w = xv[1];
                        x_sum[0] = pair(v.x, v.y);
                        x_sum[1] = pair(v.z, v.w);
                        x_sum[2] = pair(w.x, w.y);
                        x_unit = pair(w.z, w.w);
                    }
                    const Pair bias = pair(-BIAS, -BIAS);
#pragma unroll
                    for (int h = 0; h < ROWS; ++h) {
                        // both columns at once; each byte's sum is below 15 *
                        // 128 * 128 < 2^18, the zero point's share below 2^22
                        const int (&q)[PASSES][4] = sum[h >> 1];
                        const int i = (h & 1) * 2;
                        const Pair zero = pair(-z[l][h], -z[l][h]);
                        auto freed = [&](int m) {
                            return fma2(zero, x_sum[m], add2(pair(__int_as_float(q[m][i]), __int_as_float(q[m][i + 1])), bias));
                        };
                        Pair v = freed(0);
                        if constexpr (!NARROW) {
                            v = fma2(freed(1), pair(256.0f, 256.0f), v);
                            v = fma2(freed(2), pair(65536.0f, 65536.0f), v);
                        }
                        const Pair to = pair(acc[t][2 * h], acc[t][2 * h + 1]);
                        split(fma2(mul2(pair(s[l][h], s[l][h]), x_unit), v, to), acc[t][2 * h], acc[t][2 * h + 1]);
                    }
                }
            }
        }
        fetch_next(d);                                   // into the slots just read
        if (++d == DEPTH) d = 0;
        if (next_step == 0) {
            if constexpr (NARROW) {
                // Columns 0 1 | 2 3 | 4 5 of lanes c = 0, 1, 2 are the bytes
                // 0 1 | 2 0 | 1 2 of tokens 0 0 | 0 1 | 1 1: token c ends up
                // in lane c = 0, 1.
#pragma unroll
                for (int h = 0; h < ROWS; ++h) {
                    float a0 = acc[0][2 * h] * narrow_weight[0], a1 = acc[0][2 * h + 1] * narrow_weight[1];
                    const float give = c == 1 ? a0 : a0 + a1;
                    const float got = __shfl_down_sync(0xFFFFFFFFu, give, 1);
                    acc[0][2 * h] = (c == 0 ? a0 + a1 : a1) + got;
                    acc[0][2 * h + 1] = 0.0f;
                }
            }
            // The first warp of the team adds the others' sums, in warp order,
            // and stores; the leading barrier is for its reading of the last
            // tile's.
            if (g.team > 1) {
                asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(g.team * 32) : "memory");
                if (member)
#pragma unroll
                    for (int t = 0; t < 2 * NT; ++t)
                        red[((member - 1) * 2 * NT + t) * 32 + lane] =
                            make_float4(acc[t / 2][t % 2 * 4], acc[t / 2][t % 2 * 4 + 1], acc[t / 2][t % 2 * 4 + 2], acc[t / 2][t % 2 * 4 + 3]);
                asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(g.team * 32) : "memory");
            }
            if (member == 0) {
                for (int m = 0; m < g.team - 1; ++m)
#pragma unroll
                    for (int t = 0; t < 2 * NT; ++t) {
                        const float4 v = red[(m * 2 * NT + t) * 32 + lane];
                        acc[t / 2][t % 2 * 4] += v.x;
                        acc[t / 2][t % 2 * 4 + 1] += v.y;
                        acc[t / 2][t % 2 * 4 + 2] += v.z;
                        acc[t / 2][t % 2 * 4 + 3] += v.w;
                    }
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int h = 0; h < ROWS; ++h)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int tok = NARROW ? (e ? g.tokens : c) : t * 8 + 2 * c + e;
                            const int64_t n = (int64_t)tile * TILE + r + 8 * h;
                            if (tok < g.tokens && n < g.n) {
                                const float v = acc[t][2 * h + e];
                                if (g.part) g.part[((int64_t)blockIdx.y * g.tokens + tok) * g.n + n] = v;
                                else store_result(g, tok, n, v);
                            }
                        }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 2 * ROWS; ++e) acc[t][e] = 0.0f;
        }
        tile = t1;
        at_step = next_step;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// The slices' sums, added in slice order.
__global__ void __launch_bounds__(256) matvec_w4_sum_kernel(const W4Args g, int slices) {
    const int64_t o = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (o >= (int64_t)g.tokens * g.n) return;
    const int tok = (int)(o / g.n);
    const int64_t n = o % g.n;
    float v = 0.0f;
    first_is_done();
    for (int s = 0; s < slices; ++s) v += __ldcg(g.part + (int64_t)s * g.tokens * g.n + o);
    store_result(g, tok, n, v);
}

// How a launch is cut: warps per team, slices of k, blocks per slice.
struct W4Shape { int team, per_member, slices, slice_kb, tiles, kblocks, smem, grid; };

constexpr int SMEM_MAX = 227 * 1024;
int w4_smem(int tokens, int slice_kb, int units, int team) {
    const int tp = tokens <= 8 ? 8 : tokens <= 16 ? 16 : 32;
    return DEPTH * WARPS * 32 * ROWS * 16 + WARPS * 2 * SEG * TILE * 4 + ((LIMBS * tokens * (slice_kb * 128 + 16) + 127) & ~127) +
           slice_kb * units * tp * (tokens <= 2 ? 8 : 16) + (WARPS - WARPS / team) * 32 * tp * 4;
}

// units: scale units of a k-block.  Of the cuts that fit shared memory, the
// one with the fewest steps: those of the busiest warp (one for each k-block
// and one for the end of each tile: what latency costs), those of the busiest
// SM over its warps (what throughput costs), and, measured, about six for a
// second kernel.
W4Shape w4_shape(int64_t tokens, int64_t n, int64_t k, int units, int sms) {
    W4Shape best;
    best.tiles = (int)((n + TILE - 1) / TILE);
    best.kblocks = (int)((k + 127) / 128);
    best.team = 0;
    int64_t least = 0;
    for (int slices = 1; slices <= best.kblocks; slices *= 2) {
        int kb = (best.kblocks + slices - 1) / slices;
        if (slices > 1) kb = (kb + SEG - 1) / SEG * SEG;
        const int real = (best.kblocks + kb - 1) / kb;
        const int64_t per_slice = real < sms ? sms / real : 1;
        for (int team = 1; team <= WARPS; team *= 2) {
            const int smem = w4_smem((int)tokens, kb, units, team);
            if (smem > SMEM_MAX) continue;
            const int64_t teams = per_slice * (WARPS / team);
            const int64_t waves = (real + sms - 1) / sms;
            // whole segments of scales where there are any
            int per = (kb + team - 1) / team;
            if (per > SEG / units) per = (per + SEG / units - 1) / (SEG / units) * (SEG / units);
            const int64_t blocks = (best.tiles + WARPS / team - 1) / (WARPS / team);
            const int64_t grid = blocks < per_slice ? blocks : per_slice;
            const int64_t steps = waves * ((best.tiles + teams - 1) / teams * (per + 1) + (best.tiles + grid - 1) / grid * kb / WARPS) +
                                  (real > 1 ? 6 : 0);
            if (best.team && steps >= least) continue;
            least = steps;
            best.team = team;
            best.per_member = per;
            best.slices = real;
            best.slice_kb = kb;
            best.smem = smem;
            best.grid = (int)grid;
        }
    }
    return best;
}

template <int LW, int NT, Load LD>
int w4_launch(const W4Args& a, const W4Shape& s, int dev, cudaStream_t st) {
    auto k = matvec_w4_kernel<LW, NT, LD>;
    static bool ready[64] = {false};
    if (!ready[dev]) {
        if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX) != cudaSuccess) {
            cudaGetLastError();
            return fail(14, "matvec_w4: cudaFuncSetAttribute");
        }
        ready[dev] = true;
    }
    k<<<dim3(s.grid, s.slices), WARPS * 32, s.smem, st>>>(a);
    return launched("matvec_w4");
}

template <int LW, Load LD>
int w4_tokens(const W4Args& a, const W4Shape& s, int dev, cudaStream_t st) {
    if (a.tokens <= 2) return w4_launch<LW, 0, LD>(a, s, dev, st);
    if (a.tokens <= 8) return w4_launch<LW, 1, LD>(a, s, dev, st);
    if (a.tokens <= 16) return w4_launch<LW, 2, LD>(a, s, dev, st);
    return w4_launch<LW, 4, LD>(a, s, dev, st);
}

// Scale units of a k-block: what one load of a lane's weights spans (4, 2 or
// 1 words) has to stay inside a group, and inside the row.
int w4_units(const void* q, int64_t q_ld, int64_t k, int64_t group) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(q) | (uintptr_t)q_ld | (uintptr_t)((k + 1) / 2);
    if (group % 128 == 0 && at % 16 == 0) return 1;
    if (group % 64 == 0 && at % 8 == 0) return 2;
    return 4;
}

// Tokens of the next launch.  Four tiles of tokens spill; where the weights
// are many enough to hide a second launch, 16 at a time are faster with groups
// of 128 (32768 x 8192: 32 tokens 177 -> 140 us, 17 tokens 167 -> 103; 8192 x
// 8192, 32 tokens 58 -> 48), elsewhere not (32 tokens, 8192 x 4096: 31 against
// 30; 24 tokens, 32768 x 8192, groups of 64: 183 against 176).
int64_t w4_step(int64_t left, int64_t n, int64_t k, int units) {
    const int64_t most = left > 16 && units == 1 && n * k >= (int64_t(1) << 26) ? 16 : MAX_TOKENS;
    return left < most ? left : most;
}

int w4_typed(const W4Args& a, const W4Shape& s, int64_t group, int dev, cudaStream_t st) {
    const int units = w4_units(a.q, a.q_ld, a.k, group);
    if (units == 1) return w4_tokens<4, Load::Wide>(a, s, dev, st);
    if (units == 2) return w4_tokens<2, Load::Wide>(a, s, dev, st);
    if ((reinterpret_cast<uintptr_t>(a.q) | (uintptr_t)a.q_ld) % 4 == 0) return w4_tokens<1, Load::Words>(a, s, dev, st);
    return w4_tokens<1, Load::Bytes>(a, s, dev, st);
}

int w4_check(int64_t tokens, int64_t n, int64_t k, int64_t group) {
    if (tokens < 0 || n < 0 || k < 1 || n > (int64_t(1) << 30) || k > (int64_t(1) << 22))
        return fail(8, "matvec_w4: sizes out of range (tokens >= 0, 0 <= n <= 2^30, 1 <= k <= 2^22)");
    if (group < 32 || group % 32 || group > (int64_t(1) << 30))
        return fail(8, "matvec_w4: the group size must be a positive multiple of 32");
    return 0;
}

}  // namespace
}  // namespace lm
}  // namespace bafe_cuda

#define BAFE_API extern "C" __attribute__((visibility("default")))

using namespace bafe_cuda;
using namespace bafe_cuda::lm;

BAFE_API int64_t bafe_cuda_matvec_w4_workspace(int64_t tokens, int64_t n, int64_t k, int64_t group) {
    if (w4_check(tokens, n, k, group)) return -1;
    int dev = 0, sms = 0;
    if (current_device(dev, sms)) return -1;
    // whichever way the weights turn out to lie; the first launch and those of what may be left
    int64_t need = 0;
    for (int units = 1; n && units <= 4; units *= 2)
        for (int64_t left = tokens < MAX_TOKENS ? tokens : MAX_TOKENS; left > 0; --left) {
            const int64_t m = w4_step(left, n, k, units);
            const W4Shape s = w4_shape(m, n, k, units, sms);
            if (s.slices > 1 && s.slices * m * n * 4 > need) need = s.slices * m * n * 4;
            if (left == tokens && m == tokens) break;    // one launch
        }
    return need;
}

BAFE_API int bafe_cuda_matvec_w4(const void* x, int64_t x_ld, const float* x_scale, const void* qweight, int64_t q_ld,
                                 const void* scales, int64_t s_ld, const void* zeros, int64_t z_ld, void* y,
                                 int64_t y_ld, int64_t tokens, int64_t n, int64_t k, int64_t group, int x_dtype,
                                 int scale_dtype, int y_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
    if (int rc = w4_check(tokens, n, k, group)) return rc;
    const bool x8 = x_dtype == DTYPE_E4M3;
    if (!x8 && x_dtype != BAFE_DTYPE_F16 && x_dtype != BAFE_DTYPE_BF16)
        return fail(8, "matvec_w4: x must be f16, bf16 or e4m3");
    if (y_dtype != BAFE_DTYPE_F16 && y_dtype != BAFE_DTYPE_BF16) return fail(8, "matvec_w4: y must be f16 or bf16");
    if (!is_float_type(scale_dtype)) return fail(8, "matvec_w4: the scales must be f32, f16 or bf16");
    if (tokens == 0 || n == 0) return 0;
    if (!x || !qweight || !scales || !y) return fail(8, "matvec_w4: null operand");
    const int64_t groups = (k + group - 1) / group;
    if (x_ld < k || q_ld < (k + 1) / 2 || s_ld < groups || (zeros && z_ld < groups) || y_ld < n)
        return fail(8, "matvec_w4: row strides must be at least the rows' lengths");
    if (!element_aligned(2, {y, x8 ? nullptr : x}) || !element_aligned(scale_dtype == BAFE_DTYPE_F32 ? 4 : 2, {scales}) ||
        !element_aligned(4, {x_scale}))
        return fail(8, "matvec_w4: operands must start on a multiple of their element's size");
    int dev = 0, sms = 0;
    if (int rc = current_device(dev, sms)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int units = w4_units(qweight, q_ld, k, group);
    for (int64_t done = 0, m; done < tokens; done += m) {
        m = w4_step(tokens - done, n, k, units);
        const W4Shape s = w4_shape(m, n, k, units, sms);
        if (s.slices > 1 && (!workspace || workspace_bytes < s.slices * m * n * 4 ||
                             (reinterpret_cast<uintptr_t>(workspace) & 3u)))
            return fail(8, "matvec_w4: workspace too small (see bafe_cuda_matvec_w4_workspace)");
        W4Args a;
        a.x = static_cast<const char*>(x) + done * x_ld * (x8 ? 1 : 2);
        a.x_scale = x_scale ? x_scale + done : nullptr;
        a.q = static_cast<const uint8_t*>(qweight);
        a.scales = scales;
        a.zeros = static_cast<const uint8_t*>(zeros);
        a.y = static_cast<char*>(y) + done * y_ld * 2;
        a.part = s.slices > 1 ? static_cast<float*>(workspace) : nullptr;
        a.x_ld = x_ld; a.q_ld = q_ld; a.s_ld = s_ld; a.z_ld = z_ld; a.y_ld = y_ld;
        a.n = n; a.k = k;
        a.qbytes = (int)((k + 1) / 2);
        a.tokens = (int)m;
        a.group_inv = ((uint64_t(1) << 40) + group / 32 - 1) / (group / 32);   // exact for blocks below 2^17
        a.scale_type = scale_dtype;
        a.x_type = x_dtype;
        a.out_bf16 = y_dtype == BAFE_DTYPE_BF16;
        a.kblocks = s.kblocks;
        a.slice_kb = s.slice_kb;
        a.tiles = s.tiles;
        a.team = s.team;
        a.per_member = s.per_member;
        a.unit_groups = group == 128 / units;
        a.groups = (int)groups;
        if (int rc = w4_typed(a, s, group, dev, st)) return rc;
        if (s.slices > 1) {
            if (int rc = launch_second("matvec_w4 slice sum", matvec_w4_sum_kernel, dim3((unsigned)((m * n + 255) / 256)), dim3(256), st,
                                       a, s.slices))
                return rc;
        }
    }
    return 0;
}
