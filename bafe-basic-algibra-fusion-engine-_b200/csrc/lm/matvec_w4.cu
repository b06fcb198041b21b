// matvec_w4.cu -- a few rows of activations times 4-bit weights that have a
// scale, and optionally a zero point, for each group of columns:
//
//   y[m][n] = xs[m] * sum_g s[n][g] * sum_{k in g} (q[n][k] - z[n][g]) * x[m][k]
//
// (z = 8 without zero points; xs only for e4m3 rows).  Byte j of a weight
// row holds k = 2j in its low and k = 2j + 1 in its high four bits.
//
// The products are exact.  q - z is a whole number of at most 8 significant
// bits, which f16 and bf16 hold; the tokens are multiplied in their own type
// (e4m3 as f16, which holds all of its values); mma.sync m16n8k16 takes the
// weights as its 16 rows, the tokens as its 8 columns, and adds in 32 bits.
// A unit of up to 128 k of one group is summed that way, then multiplied by
// its scale and added to the result's sum in 32 bits.  So a weight at its zero
// point counts for nothing, however large the token it meets, and what a large
// token hides in a sum is no more than in any 32-bit sum.  (Tokens as 24-bit
// fixed point with a power of two per 128 k, multiplied as three bytes by the
// integer instruction, lost the small ones beside a large one even where that
// one's weight was the zero point.  Against that form, one and two tokens take
// longer now, 3 and more mostly less: 1 x 32768 x 8192 f16 34 -> 41 us and bf16
// 34 -> 46, 8 f16 50 -> 43, 16 bf16 71 -> 56, 32 140 -> 110.)  An infinity in a
// token is made a NaN: its row gives NaN throughout.
//
// The floor is the weights' bytes (8 x 32768 x 8192 with zero points: 21.5
// us); what bounds it is instructions: a step of 32 rows x 128 k takes about
// 390 of them a warp (370 in f16), 112 for taking out the half-bytes (a shift and one logic
// operation for a pair, at half the issue rate; f16 has room for two of the
// four pairs without a shift: 80), 64 for the zero points and 16 products, with
// the issue slots 57 to 59 % busy and four warps a scheduler.  Shifting by means of
// the multiplier's upper half took longer (46 -> 54 us).
//
// The order of k inside an instruction is free as long as both operands
// agree, so the weights are used as they lie in memory: a lane takes whole
// words; the half-bytes 0 4 | 1 5 | 2 6 | 3 7 of each come out as pairs of
// 16-bit numbers, and the tokens are laid out in that order.  All k of a unit
// must belong to one group: groups of a multiple of 128 let each lane load 16
// bytes (4 lanes: 128 k), groups of 64 8 bytes, other multiples of 32 4 bytes.
//
// A block's warps form teams.  A team walks tiles of 32 rows (two of the
// instruction's, so that the tokens are read from shared memory half as
// often); each of its warps has a part of the tile's k-blocks of 128, and they
// add their sums through shared memory, behind a barrier of the team's own.
// Small teams wait less for one another, large ones spread few tiles over
// more warps: w4_shape weighs both.  The weights of the next steps travel into shared memory with
// asynchronous copies, each thread into slots of its own, so that no barrier
// guards them and the bytes in flight do not cost registers.  Scales and zero
// points come four at a time, one row a lane, and are put into shared memory:
// fetched for each k-block by itself, every 2 bytes cost a sector of 32 and
// doubled the traffic into the SM.  Where the tiles are too few for the SMs, or the tokens would crowd out the weights, k is
// also cut into slices over blocks, whose sums a second kernel adds in slice
// order.
#include "common.cuh"

#include <type_traits>

namespace bafe_cuda {
namespace lm {
namespace {

constexpr int MAX_TOKENS = 32;         // per launch (two of 16 for 17 to 32 are slower or even nearly everywhere: 32 x 8192 x 8192 41 against 34 us)
constexpr int TILE = 32;               // weight rows
constexpr int ROWS = 4;                // of them per lane: r, r + 8, r + 16, r + 24
constexpr int DEPTH = 3;               // k-blocks of a warp in flight or in use
constexpr int SEG = 4;                 // scale units of a row that are fetched together
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

// Of the multiplied type T: the instruction that adds 16 products to a sum in
// 32 bits, and the 16-bit pairs around it.
template <class T> struct Mul;
template <> struct Mul<__half> {
    // 1024 in both halves: a four-bit q in the low bits makes it 1024 + q
    static constexpr uint32_t MAGIC = 0x64006400u;
    static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ uint32_t add(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ uint32_t sixteenth(uint32_t a, uint32_t b) {      // a / 16 + b
        uint32_t r;
        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(0x2C002C00u), "r"(b));
        return r;
    }
};
template <> struct Mul<__nv_bfloat16> {
    static constexpr uint32_t MAGIC = 0x43004300u;       // 128
    static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ uint32_t add(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
};
// The bits of `of` and `magic` together, in one instruction while both are registers.
__device__ __forceinline__ uint32_t pick(uint32_t from, uint32_t of, uint32_t magic) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(from), "r"(of), "r"(magic));
    return r;
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

// Eight values of a token; those behind the row's end are 0.
template <class T>
__device__ __forceinline__ Pack<T, 8> load_tokens(const void* x, int64_t at, int64_t left) {
    const T* p = static_cast<const T*>(x) + at;
    if (left >= 8 && (reinterpret_cast<uintptr_t>(p) & 15u) == 0) return *reinterpret_cast<const Pack<T, 8>*>(p);
    Pack<T, 8> v;
    const unsigned short* bits = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j)
        v.w[j] = (2 * j < left ? (uint32_t)bits[2 * j] : 0u) | (2 * j + 1 < left ? (uint32_t)bits[2 * j + 1] << 16 : 0u);
    return v;
}

// e4m3, as f16 (exact): two values an instruction, eight bytes a load.
__device__ __forceinline__ Pack<__half, 8> load_tokens_e4m3(const void* x, int64_t at, int64_t left) {
    const uint8_t* p = static_cast<const uint8_t*>(x) + at;
    uint2 b = make_uint2(0u, 0u);
    if (left >= 8 && (reinterpret_cast<uintptr_t>(p) & 7u) == 0) {
        b = *reinterpret_cast<const uint2*>(p);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < left) (j < 4 ? b.x : b.y) |= (uint32_t)p[j] << (8 * (j & 3));
    }
    Pack<__half, 8> v;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((j < 2 ? b.x : b.y) >> (16 * (j & 1))), __NV_E4M3);
        v.w[j] = (uint32_t)h.x | (uint32_t)h.y << 16;
    }
    return v;
}

// bf16 rows that hold a value of 2^96 or more are multiplied by 2^-32, and
// their results by 2^32: q x summed over a scale unit then stays in range
// (f16 and e4m3 cannot leave it).
constexpr uint32_t FAR = (127 + 96) << 7;                // bf16 bits of 2^96
__device__ __forceinline__ bool any_far(const uint4& v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    bool far = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) far |= (w[j] & 0x7F80u) >= FAR || (w[j] >> 16 & 0x7F80u) >= FAR;
    return far;
}

template <class T, int LW, int NT, Load LD>              // T: what is multiplied; NT: token tiles of 8
__global__ void __launch_bounds__(WARPS * 32, 1) matvec_w4_kernel(const W4Args g) {
    constexpr bool BF16 = sizeof(T) == 2 && Mul<T>::MAGIC == Mul<__nv_bfloat16>::MAGIC;
    constexpr int U = 4 / LW;
    constexpr int E = ROWS * U;                          // pieces of LW words a thread holds per k-block
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ uint32_t far_rows;
    constexpr int threads = WARPS * 32;
    if (g.part) second_may_start();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int team = warp / g.team, member = warp % g.team, teams = WARPS / g.team;
    const int r = lane >> 2, c = lane & 3;
    const int kb0 = blockIdx.y * g.slice_kb;
    const int nkb = min(g.kblocks - kb0, g.slice_kb);
    const int x_row = nkb * 256 + 64;                    // bytes per token: 64 keep two tokens' reads apart
    // this thread's slots: [DEPTH][E][threads] pieces
    WordsOf<LW>* slots = reinterpret_cast<WordsOf<LW>*>(smem) + threadIdx.x;
    unsigned char* after = smem + (size_t)DEPTH * threads * E * LW * 4;
    // the warp's scales and zero points of SEG units: row i at (i % 8) * 4 + i / 8, a lane's four rows side by side
    float* seg_s = reinterpret_cast<float*>(after) + warp * (2 * SEG * TILE);
    uint32_t* seg_z = reinterpret_cast<uint32_t*>(seg_s + SEG * TILE);
    unsigned char* xs = after + WARPS * 2 * SEG * TILE * 4;                     // [tokens][x_row]
    // the team's sums: [members but the first][lanes] of 8 NT floats
    float4* red = reinterpret_cast<float4*>(xs + g.tokens * x_row) + team * (g.team - 1) * 32 * 2 * NT;

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
    // asked for one segment ahead, put into shared memory at its start, the
    // scale as a number and the zero point z as what is taken off MAGIC + q:
    // MAGIC + z in both halves.  bf16 holds 128 + z up to 127 only; 128 more
    // are marked in the sign and taken off by a second subtraction, where the
    // warp's segment has any (big).  wide: four of them in one load.
    uint32_t s_raw[SEG], z_raw[SEG];
    bool big = false;
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
        uint32_t any = 0;
#pragma unroll
        for (int o = 0; o < SEG; ++o) {
            const uint32_t s = s_wide ? (o & 1 ? s_raw[o / 2] >> 16 : s_raw[o / 2] & 0xFFFFu) : s_raw[o];
            const uint32_t z = !g.zeros ? 8u : z_wide ? (z_raw[0] >> (8 * o)) & 255u : z_raw[o];
            seg_s[o * TILE + to] = scale_f32(s, g.scale_type);
            seg_z[o * TILE + to] = Mul<T>::MAGIC + (BF16 ? (z & 127u) | (z & 128u) << 8 : z) * 0x00010001u;
            any |= z;
        }
        if (BF16) big = __any_sync(0xFFFFFFFFu, any & 128u);
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

    // Tokens: 8 k a thread, four loads in flight.  They are laid down in the
    // order in which a lane's weight words use them: word v of lane c in unit l
    // at 16 (4 (l LW + v) + c), its values as the pairs k = 0 4 | 1 5 | 2 6 | 3 7
    // that the weights' half-bytes come out in.  An infinity is made NaN here
    // (v + (v - v)), which reaches every output of its row.
    const int pieces = g.tokens * nkb * 16;
    bool far = false;
    for (int o0 = threadIdx.x; o0 < pieces; o0 += 4 * threads) {
        Pack<T, 8> p[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int o = min(o0 + q * threads, pieces - 1), tok = (o >> 4) / nkb, kbl = (o >> 4) % nkb;
            const int64_t k = (int64_t)(kb0 + kbl) * 128 + (o & 15) * 8, left = g.k - k;
            if constexpr (BF16) p[q] = load_tokens<T>(g.x, tok * g.x_ld + k, left);
            else if (g.x_type == DTYPE_E4M3) p[q] = load_tokens_e4m3(g.x, tok * g.x_ld + k, left);
            else p[q] = load_tokens<T>(g.x, tok * g.x_ld + k, left);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int o = o0 + q * threads;
            if (o >= pieces) break;
            const int tok = (o >> 4) / nkb, kbl = (o >> 4) % nkb, j = o & 15;
            const int l = j / (4 * LW), c_of = j % (4 * LW) / LW, v = j % LW;
            uint32_t (&w)[4] = p[q].w;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = Mul<T>::add(w[i], Mul<T>::sub(w[i], w[i]));
            const uint4 to = make_uint4(__byte_perm(w[0], w[2], 0x5410), __byte_perm(w[0], w[2], 0x7632),
                                        __byte_perm(w[1], w[3], 0x5410), __byte_perm(w[1], w[3], 0x7632));
            if (BF16) far |= any_far(to);
            *reinterpret_cast<uint4*>(xs + tok * x_row + kbl * 256 + ((l * LW + v) * 4 + c_of) * 16) = to;
        }
    }
    uint32_t far_mask = 0;                               // bit t: token t's values were multiplied by 2^-32
    if (!BF16) {
        __syncthreads();
    } else if (__syncthreads_or(far)) {                  // rare
        if (threadIdx.x == 0) far_rows = 0;
        __syncthreads();
        for (int o = threadIdx.x; o < pieces; o += threads) {
            const int tok = (o >> 4) / nkb, at = (o >> 4) % nkb * 256 + (o & 15) * 16;
            if (any_far(*reinterpret_cast<const uint4*>(xs + tok * x_row + at))) atomicOr(&far_rows, 1u << tok);
        }
        __syncthreads();
        far_mask = far_rows;
        for (int o = threadIdx.x; o < pieces; o += threads) {
            const int tok = (o >> 4) / nkb, at = (o >> 4) % nkb * 256 + (o & 15) * 16;
            if (!(far_mask >> tok & 1u)) continue;
            Pack<T, 8>& p = *reinterpret_cast<Pack<T, 8>*>(xs + tok * x_row + at);
            float f[8];
            unpack(p, f);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] *= 2.3283064365386963e-10f;        // 2^-32
            pack(f, p);
        }
        __syncthreads();
    }

    // This lane's values of its token in each column tile.  Columns behind the
    // last token repeat it; their sums are not stored.
    const unsigned char* xlane[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) xlane[t] = xs + min(t * 8 + r, g.tokens - 1) * x_row + c * 16;
    uint32_t low = 0x000F000Fu, magic = Mul<T>::MAGIC;   // kept in registers
    asm volatile("" : "+r"(low), "+r"(magic));
    uint32_t low4 = low << 4;
    asm volatile("" : "+r"(low4));
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
            const WordsOf<LW>* src = slots + d * E * threads;
#pragma unroll
            for (int l = 0; l < U; ++l) {
                const int o = (at_step % LW) * U + l;
                const float4 s4 = *reinterpret_cast<const float4*>(seg_s + o * TILE + 4 * r);
                const uint4 z4 = *reinterpret_cast<const uint4*>(seg_z + o * TILE + 4 * r);
                const float s[ROWS] = {s4.x, s4.y, s4.z, s4.w};
                const uint32_t z[ROWS] = {z4.x, z4.y, z4.z, z4.w};
                WordsOf<LW> w[ROWS];
#pragma unroll
                for (int h = 0; h < ROWS; ++h) w[h] = src[(h * U + l) * threads];
                float sum[NT][2][4];                     // of 16 rows by 8 tokens each
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 8; ++i) sum[t][i >> 2][i & 3] = 0.0f;
                auto multiply = [&](auto second) {
#pragma unroll
                    for (int v = 0; v < LW; ++v) {
                        uint32_t a[ROWS][4];             // q - z of k = 0 4 | 1 5 | 2 6 | 3 7
#pragma unroll
                        for (int h = 0; h < ROWS; ++h) {
                            const uint32_t q = w[h].w[v];
                            if constexpr (BF16) {
                                auto off = [&](uint32_t u) {
                                    if constexpr (decltype(second)::value)
                                        return Mul<T>::sub(Mul<T>::sub(u, z[h] & 0x7FFF7FFFu), z[h] & 0x8000u ? Mul<T>::MAGIC : 0u);
                                    else
                                        return Mul<T>::sub(u, z[h]);
                                };
#pragma unroll
                                for (int i = 0; i < 4; ++i) a[h][i] = off(pick(q >> (4 * i), low, magic));
                            } else {
                                // f16 has room for the upper half-bytes where they are: 1024 + 16 q
                                const uint32_t z16 = Mul<T>::sub(0x63806380u, z[h]);      // 960 - (1024 + z) = -(64 + z)
                                a[h][0] = Mul<T>::sub(pick(q, low, magic), z[h]);
                                a[h][1] = Mul<T>::sixteenth(pick(q, low4, magic), z16);
                                a[h][2] = Mul<T>::sub(pick(q >> 8, low, magic), z[h]);
                                a[h][3] = Mul<T>::sixteenth(pick(q >> 8, low4, magic), z16);
                            }
                        }
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            const uint4 x = *reinterpret_cast<const uint4*>(xlane[t] + kbl * 256 + (l * LW + v) * 64);
#pragma unroll
                            for (int p = 0; p < 2; ++p) {
                                Mul<T>::mma(sum[t][p], a[2 * p][0], a[2 * p + 1][0], a[2 * p][1], a[2 * p + 1][1], x.x, x.y);
                                Mul<T>::mma(sum[t][p], a[2 * p][2], a[2 * p + 1][2], a[2 * p][3], a[2 * p + 1][3], x.z, x.w);
                            }
                        }
                    }
                };
                if (BF16 && big) multiply(std::true_type());
                else multiply(std::false_type());
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int h = 0; h < ROWS; ++h) {     // both columns at once
                        const Pair v = pair(sum[t][h >> 1][(h & 1) * 2], sum[t][h >> 1][(h & 1) * 2 + 1]);
                        const Pair to = pair(acc[t][2 * h], acc[t][2 * h + 1]);
                        split(fma2(pair(s[h], s[h]), v, to), acc[t][2 * h], acc[t][2 * h + 1]);
                    }
            }
        }
        fetch_next(d);                                   // into the slots just read
        if (++d == DEPTH) d = 0;
        if (next_step == 0) {
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
                            const int tok = t * 8 + 2 * c + e;
                            const int64_t n = (int64_t)tile * TILE + r + 8 * h;
                            if (tok < g.tokens && n < g.n) {
                                float v = acc[t][2 * h + e];
                                if (BF16 && far_mask >> tok & 1u) v *= 4294967296.0f;
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

constexpr int SMEM_MAX = 227 * 1024 - 128;              // beside the static far_rows
int w4_smem(int tokens, int slice_kb, int team) {
    const int tp = tokens <= 8 ? 8 : tokens <= 16 ? 16 : 32;
    return DEPTH * WARPS * 32 * ROWS * 16 + WARPS * 2 * SEG * TILE * 4 + tokens * (slice_kb * 256 + 64) +
           (WARPS - WARPS / team) * 32 * tp * 4;
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
            const int smem = w4_smem((int)tokens, kb, team);
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

template <class T, int LW, int NT, Load LD>
int w4_launch(const W4Args& a, const W4Shape& s, int dev, cudaStream_t st) {
    auto k = matvec_w4_kernel<T, LW, NT, LD>;
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

template <class T, int LW, Load LD>
int w4_tokens(const W4Args& a, const W4Shape& s, int dev, cudaStream_t st) {
    if (a.tokens <= 8) return w4_launch<T, LW, 1, LD>(a, s, dev, st);
    if (a.tokens <= 16) return w4_launch<T, LW, 2, LD>(a, s, dev, st);
    return w4_launch<T, LW, 4, LD>(a, s, dev, st);
}

// Scale units of a k-block: what one load of a lane's weights spans (4, 2 or
// 1 words) has to stay inside a group, and inside the row.
int w4_units(const void* q, int64_t q_ld, int64_t k, int64_t group) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(q) | (uintptr_t)q_ld | (uintptr_t)((k + 1) / 2);
    if (group % 128 == 0 && at % 16 == 0) return 1;
    if (group % 64 == 0 && at % 8 == 0) return 2;
    return 4;
}

template <class T>
int w4_typed(const W4Args& a, const W4Shape& s, int units, int dev, cudaStream_t st) {
    if (units == 1) return w4_tokens<T, 4, Load::Wide>(a, s, dev, st);
    if (units == 2) return w4_tokens<T, 2, Load::Wide>(a, s, dev, st);
    if ((reinterpret_cast<uintptr_t>(a.q) | (uintptr_t)a.q_ld) % 4 == 0) return w4_tokens<T, 1, Load::Words>(a, s, dev, st);
    return w4_tokens<T, 1, Load::Bytes>(a, s, dev, st);
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
    // whichever way the weights turn out to lie; whole launches and the last
    int64_t need = 0;
    for (int units = 1; n && units <= 4; units *= 2)
        for (const int64_t m : {tokens < MAX_TOKENS ? tokens : MAX_TOKENS, tokens % MAX_TOKENS}) {
            if (m == 0) continue;
            const W4Shape s = w4_shape(m, n, k, units, sms);
            if (s.slices > 1 && s.slices * m * n * 4 > need) need = s.slices * m * n * 4;
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
        m = tokens - done < MAX_TOKENS ? tokens - done : MAX_TOKENS;
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
        if (int rc = x_dtype == BAFE_DTYPE_BF16 ? w4_typed<__nv_bfloat16>(a, s, units, dev, st) : w4_typed<__half>(a, s, units, dev, st))
            return rc;
        if (s.slices > 1) {
            if (int rc = launch_second("matvec_w4 slice sum", matvec_w4_sum_kernel, dim3((unsigned)((m * n + 255) / 256)), dim3(256), st,
                                       a, s.slices))
                return rc;
        }
    }
    return 0;
}
