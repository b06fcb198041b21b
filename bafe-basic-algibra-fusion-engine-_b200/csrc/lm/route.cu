// route.cu -- routing to experts: scores, the k best experts of each row,
// their weights, the rows' order by expert, and the gradient.
//
//   s = softmax or sigmoid of a row's logits
//   c = s + bias where the logit is above -inf (an open expert); else shut
//   groups of consecutive experts are worth the sum of their group_top
//   largest open c; the keep best groups' experts stay open
//   experts = the k open ones of largest c, in this order (the lowest index of
//   equals; -1 where none is left), weights = s of them, over their sum with
//   renorm, times scale
//   offsets[e] = first place of expert e when all choices are sorted by
//   expert (equal ones in their own order), place[t][j] = that of choice j of
//   row t: what grouped_matmul takes.
//
// What bounds this is instructions, not bytes.  LPR lanes share a row -- 8 up
// to 256 experts, so that a warp has four rows and what is done once per lane
// or round counts for four -- with up to 32 scores each in registers, in
// quads.  The k-th largest of the 8 largest-of-a-few of every lane is a lower
// bound of the k-th largest of all; the few experts above it (k and some) go
// into a list, whose members are ranked by comparing all with all.  (A warp a
// row, the largest picked k + 1 times: 1900 instructions a row of 256, 60.7 us for
// 16384 rows, 8 of 256 in groups; with the list 1250, 53.3; eight lanes a row 640,
// 31: 23 in this kernel, at 36 % of the issue slots, and 7 in the second.)
// Rows with more than 32 such experts take the long way, one expert a round.
//
// Without a bias the order of the experts is that of the logits, which is the
// scores' and goes on where those are equal in any number of bits (a sigmoid's 1
// above 37); without groups nothing else is computed for the choice.  With a
// bias, and for the groups' worths, the order is that of c in 64 bits (scores below
// e^-700 count as 0): two f32 scores nearer to one another than their errors
// could be the other way round.  Experts that near are among the few; where
// there are any, the few scores are made again in 64 bits, and so are the
// groups' worths where two are near at the border (if a group's own largest are
// near to one another too, the whole row).
//
// The order by expert is a counting sort in two kernels: each block numbers
// the choices of its rows, expert by expert, and leaves their counts; the
// second kernel adds the counts of the blocks before.  Warps and lanes go in order,
// no atomics whose order matters: the same places every run.  Few rows take
// one block and one kernel.
#include "common.cuh"

#include <cmath>

namespace bafe_cuda {
namespace lm {
namespace {

typedef unsigned int u32;
constexpr u32 ALL = 0xFFFFFFFFu;
constexpr int MAX_EXPERTS = 1024;
constexpr int MAX_K = 31;              // a list of 32 holds them and one more
constexpr int MAX_GROUPS = 32;
constexpr int SMALL_ROWS = 64;         // rows that one block routes and sorts

struct RouteArgs {
    const void* logits;
    const float* bias;                 // [experts], or null
    float* weights;                    // [rows][k]
    int* experts;                      // [rows][k]
    int* offsets;                      // [n + 1]
    int* place;                        // [rows][k]
    void* counts;                      // [chunks][counts_ld]: choices of each block's rows per expert, bytes or ints
    int64_t ld, rows, chunk_rows;
    int n, k, groups, keep, group_size, group_top, chunks;
    int dtype, sigmoid, renorm;
    int vec;                           // rows of quads on their boundaries
    int byte_counts, counts_ld;
    u32 group_inverse;                 // 2^32 / group_size, rounded up
    float scale;
};
__device__ __forceinline__ int group_of(const RouteArgs& g, int e) {   // exact for e < 2^16
    return g.group_size == 1 ? e & 31 : (int)__umulhi((u32)e, g.group_inverse) & 31;
}

__device__ __forceinline__ float load_one(const void* p, int dtype, int64_t at) {
    if (dtype == BAFE_DTYPE_F32) return static_cast<const float*>(p)[at];
    if (dtype == BAFE_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]);
    return __half2float(static_cast<const __half*>(p)[at]);
}

// Approximate exponential and reciprocal: both within 2^-22, the exponent
// rounded to 2^-24 of itself.
__device__ __forceinline__ float exp2_fast(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float inverse_fast(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
constexpr float LOG2E = 1.4426950408889634f;

// e^x in 64 bits, 0 below e^-700, to a few 2^-53: 2^n e^r with n the nearest
// whole number to x / ln 2, r from x in two steps (Cody and Waite: ln 2 as a
// part of 32 bits, whose products with n are exact, and the rest), |r| <= 0.35, and e^r
// by its Taylor polynomial, whose first left-out term is r^14 / 14! < 2^-57.
// Short, for the reason given at choose_long.
__device__ __forceinline__ double exp64(double x) {
    x = fmin(fmax(x, -700.0), 700.0);
    const double n = rint(x * 1.4426950408889634074);
    const double high = 0x1.62e42feep-1, low = 0x1.a39ef35793c76p-33;
    const double r = fma(-n, low, fma(-n, high, x));
    double p = 1.0 / 6227020800.0;                       // 1 / 13!
    p = fma(p, r, 1.0 / 479001600.0);
    p = fma(p, r, 1.0 / 39916800.0);
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return x <= -700.0 ? 0.0 : p * __hiloint2double((1023 + (int)n) << 20, 0);
}
// 1 / x for x from 1 to 2^1020, by Newton's iteration from the 32-bit one.
__device__ __forceinline__ double inverse64(double x) {
    const int up = __double2hiint(x) >> 20;              // x's exponent: the start is made for 1 <= x < 2
    const double m = __hiloint2double((__double2hiint(x) & 0xFFFFF) | 0x3FF00000, __double2loint(x));
    double y = (double)(1.0f / (float)m);
    y = fma(y, fma(-m, y, 1.0), y);
    y = fma(y, fma(-m, y, 1.0), y);
    return y * __hiloint2double((2046 - up) << 20, 0);
}
// A score in 64 bits; softmax: m is the row's largest logit and inv the
// inverse of the row's sum.
__device__ __noinline__ double score64(bool sigmoid, double l, double m, double inv) {
    const double x = exp64(sigmoid ? -l : l - m);
    return sigmoid ? inverse64(1.0 + x) : x * inv;
}
// That inverse, by the LPR lanes of a row, lane r of them.
template <int LPR> __device__ __noinline__ double inverse_sum64(const RouteArgs& g, int64_t row, int r, double m) {
    double z = 0.0;
#pragma unroll 2
    for (int e = r; e < g.n; e += LPR) z += exp64((double)load_one(g.logits, g.dtype, row * g.ld + e) - m);
#pragma unroll 1
    for (int o = LPR / 2; o; o >>= 1) z += __shfl_xor_sync(ALL, z, o);
    return inverse64(z);                                 // at least 1: the largest's own; a shut row's is used nowhere
}

// A row's choice in 64 bits, by a warp, one expert a round; d: n doubles.
// Rare, and so in loops that are not unrolled and without CUDA's exp and
// division: code that an SM has not run yet comes in from L2 line by line, some
// 50 ns an instruction, and one such row holds up the whole call (unrolled 10 us).
__device__ __noinline__ void choose_long(const RouteArgs& g, int64_t row, int lane, double* d, int* choice) {
    const double shut = -INFINITY;
    const bool scored = g.bias || g.groups > 1;
    double m = shut, inv = 1.0;
    if (scored && !g.sigmoid) {
#pragma unroll 1
        for (int e = lane; e < g.n; e += 32) m = fmax(m, (double)load_one(g.logits, g.dtype, row * g.ld + e));
#pragma unroll 1
        for (int o = 16; o; o >>= 1) m = fmax(m, __shfl_xor_sync(ALL, m, o));
        if (!(m > shut)) m = 0.0;
        inv = inverse_sum64<32>(g, row, lane, m);
    }
#pragma unroll 1
    for (int e = lane; e < g.n; e += 32) {
        const double l = load_one(g.logits, g.dtype, row * g.ld + e);
        double x = l;
        if (scored) x = score64(g.sigmoid, l, m, inv) + (g.bias ? (double)g.bias[e] : 0.0);
        d[e] = l > shut ? x : shut;
    }
    __syncwarp();
    if (g.groups > 1) {
        double worth = shut;                             // of group `lane`
        const double* group = d + min(lane, g.groups - 1) * g.group_size;
        double a = shut, b = shut;
#pragma unroll 1
        for (int i = 0; i < g.group_size; ++i) {
            b = fmax(b, fmin(a, group[i]));
            a = fmax(a, group[i]);
        }
        worth = g.group_top > 1 && b > shut ? a + b : a;
        int better = 0;
#pragma unroll 1
        for (int h = 0; h < g.groups; ++h) {
            const double w = __shfl_sync(ALL, worth, h);
            better += w > worth || (w == worth && h < lane);
        }
        const u32 stay = __ballot_sync(ALL, better < g.keep && lane < g.groups);
#pragma unroll 1
        for (int e = lane; e < g.n; e += 32) {
            if (!(stay >> group_of(g, e) & 1u)) d[e] = shut;
            else if (!g.bias && d[e] > shut) d[e] = load_one(g.logits, g.dtype, row * g.ld + e);     // the same order, finer
        }
    }
    choice[lane] = -1;
    __syncwarp();
#pragma unroll 1
    for (int j = 0; j < g.k; ++j) {
        double best = shut;
        int at = g.n;
#pragma unroll 1
        for (int e = lane; e < g.n; e += 32)
            if (d[e] > best) {
                best = d[e];
                at = e;
            }
#pragma unroll 1
        for (int o = 16; o; o >>= 1) {
            const double other = __shfl_xor_sync(ALL, best, o);
            const int its = __shfl_xor_sync(ALL, at, o);
            if (other > best || (other == best && its < at)) {
                best = other;
                at = its;
            }
        }
        if (at >= g.n) break;                            // no open expert left
        if (lane == (at & 31)) {
            choice[j] = at;
            d[at] = shut;
        }
        __syncwarp();
    }
}

struct Few {                           // an expert that may be chosen
    float c;
    int e;
};

template <int LPR> __device__ __forceinline__ float row_max(float v) {
#pragma unroll
    for (int o = LPR / 2; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(ALL, v, o));
    return v;
}
template <int LPR> __device__ __forceinline__ float row_sum(float v) {
#pragma unroll
    for (int o = LPR / 2; o; o >>= 1) v += __shfl_xor_sync(ALL, v, o);
    return v;
}

// Slot i of lane r of a row is expert (i / 4 * LPR + r) * 4 + i % 4: quads of
// neighbouring lanes lie side by side.
template <int LPR, int V> __device__ __forceinline__ void load_quads(const RouteArgs& g, int64_t at, int r, float (&l)[V]) {
    auto all = [&](auto* src) {
        typedef typename std::remove_const<typename std::remove_pointer<decltype(src)>::type>::type T;
        src += at;
#pragma unroll
        for (int q = 0; q < V / 4; ++q) {
            const int e = (q * LPR + r) * 4;
            if (g.vec) {
                Pack<T, 4> p;
                float f[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                if (e < g.n) {
                    p = *reinterpret_cast<const Pack<T, 4>*>(src + e);
                    unpack<4>(p, f);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) l[4 * q + j] = f[j];
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) l[4 * q + j] = e + j < g.n ? to_f32(src[e + j]) : -INFINITY;
            }
        }
    };
    if (g.dtype == BAFE_DTYPE_F32) all(static_cast<const float*>(g.logits));
    else if (g.dtype == BAFE_DTYPE_BF16) all(static_cast<const __nv_bfloat16*>(g.logits));
    else all(static_cast<const __half*>(g.logits));
}

// s sorted, the largest first: 1, 2, 4 or 8 values, by a fixed network.
template <int S> __device__ __forceinline__ void sort_down(float (&s)[S]) {
    auto cx = [&](int a, int b) {
        const float hi = fmaxf(s[a], s[b]);
        s[b] = fminf(s[a], s[b]);
        s[a] = hi;
    };
    if constexpr (S == 4) {
        cx(0, 1), cx(2, 3), cx(0, 2), cx(1, 3), cx(1, 2);
    } else if constexpr (S == 8) {
        cx(0, 1), cx(2, 3), cx(4, 5), cx(6, 7), cx(0, 2), cx(1, 3), cx(4, 6), cx(5, 7), cx(1, 2), cx(5, 6);
        cx(0, 4), cx(1, 5), cx(2, 6), cx(3, 7), cx(2, 4), cx(3, 5), cx(1, 2), cx(3, 4), cx(5, 6);
    }
}

constexpr int MAX_FEW = 32, FEW_LD = MAX_FEW + 1;       // one more, so that rows start in other banks

// A warp's shared memory: a list, its 64-bit scores, the choice and the
// groups' worths for each of its rows; the rows' scores.
template <int LPR, int V> struct WarpMem {
    static constexpr int ROWS = 32 / LPR, WIDE = LPR * V;
    static constexpr int LIST = 0, EXACT = LIST + ROWS * FEW_LD * 8, WORTH = EXACT + ROWS * FEW_LD * 8;
    static constexpr int CHOICE = WORTH + ROWS * FEW_LD * 4, SCORES = (CHOICE + ROWS * 32 * 4 + 15) & ~15;
    static constexpr int SCORE_BYTES = ROWS * WIDE * 4 > WIDE * 8 ? ROWS * WIDE * 4 : WIDE * 8;      // or one row in 64 bits
    static constexpr int BYTES = SCORES + SCORE_BYTES;
};

// Routes rows [first, first + 32 / LPR) below `end`; their choices go to
// list and masks, counted from row `from`, too.
template <int LPR, int V>
__device__ __forceinline__ void route_rows(const RouteArgs& g, int64_t first, int64_t end, int lane, const float* bias, bool bad_bias, float high_bias,
                                           unsigned char* mem, int* list, u32* masks, int64_t from) {
    typedef WarpMem<LPR, V> M;
    constexpr int TURNS = 32 / LPR;                      // of a row's lanes over 32 entries
    const int sub = lane / LPR, r = lane % LPR;
    const bool live = first + sub < end;
    const int64_t row = live ? first + sub : end - 1;    // the rows behind the last are routed as the last, and not stored
    Few* few = reinterpret_cast<Few*>(mem + M::LIST) + sub * FEW_LD;
    int* choice = reinterpret_cast<int*>(mem + M::CHOICE) + sub * 32;
    float c[V];
    load_quads<LPR, V>(g, row * g.ld, r, c);
#pragma unroll
    for (int t = 0; t < TURNS; ++t) {
        few[t * LPR + r] = {-INFINITY, -1};
        choice[t * LPR + r] = -1;
    }
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < V; ++i) m = max_nan(m, c[i]);
#pragma unroll
    for (int o = LPR / 2; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(ALL, m, o));
    const bool bad = !(m == m) || bad_bias || (!g.sigmoid && m == INFINITY);     // a softmax of infinities has no value
    if (!(m > -INFINITY)) m = 0.0f;
    const bool scored = g.bias || g.groups > 1;          // else the logits have the scores' order
    float inv = 1.0f;                                    // of the softmax's sum
    if (!g.sigmoid && (scored || !g.renorm)) {
        float z = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) z += exp2_fast((c[i] - m) * LOG2E);
        inv = inverse_fast(fmaxf(row_sum<LPR>(z), 1e-30f));
    }
    // Errors of the f32 scores.  Sigmoid, in half ulps of 1: the exponent's
    // rounding counts as 1.25 |l| s (1 - s) <= 0.3, the exponential's as s (1 - s) 4
    // <= 1, the addition's as 1, the reciprocal's as 2: below 4.5, 8 (2^-21) are
    // allowed.  Softmax, relative to the largest score: the exponent's as up to
    // |l - m| e^-|l - m|, the sum's roundings as up to 36, the others as a few: 2^-17 is allowed.
    const float tell = g.sigmoid ? 0x1p-21f : 0x1p-17f * inv;
    bool longer = false;
    if (scored) {
#pragma unroll
        for (int q = 0; q < V / 4; ++q) {
            const float4 b4 = *reinterpret_cast<const float4*>(bias + (q * LPR + r) * 4);
            const float b[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float l = c[4 * q + j];
                const float s = g.sigmoid ? inverse_fast(1.0f + exp2_fast(-LOG2E * l)) : exp2_fast((l - m) * LOG2E) * inv;
                c[4 * q + j] = l > -INFINITY ? s + b[j] : -INFINITY;
            }
        }
        if (g.groups > 1) {
            float* scores = reinterpret_cast<float*>(mem + M::SCORES) + sub * M::WIDE;
            float* worths = reinterpret_cast<float*>(mem + M::WORTH) + sub * FEW_LD;
#pragma unroll
            for (int q = 0; q < V / 4; ++q)
                *reinterpret_cast<float4*>(scores + (q * LPR + r) * 4) = make_float4(c[4 * q], c[4 * q + 1], c[4 * q + 2], c[4 * q + 3]);
            __syncwarp();
            for (int h = r; h < g.groups; h += LPR) {
                // from another element in every group: other banks
                float a = -INFINITY, b = -INFINITY;
                int at = h % g.group_size;
                const float* group = scores + h * g.group_size;
#pragma unroll 4
                for (int i = 0; i < g.group_size; ++i) {
                    const float v = group[at];
                    b = fmaxf(b, fminf(a, v));
                    a = fmaxf(a, v);
                    if (++at == g.group_size) at = 0;
                }
                // half of it, which does not leave f32's range where biases are beyond half of that
                worths[h] = g.group_top > 1 && b > -INFINITY ? 0.5f * a + 0.5f * b : 0.5f * a;
            }
            __syncwarp();
            u32 stay = 0;
            float in = INFINITY, out = -INFINITY;        // the worst kept, the best other
            for (int h = r; h < g.groups; h += LPR) {
                const float worth = worths[h];
                int better = 0;
#pragma unroll 4
                for (int x = 0; x < g.groups; ++x) {
                    const float w = worths[x];
                    better += w > worth || (w == worth && x < h);
                }
                if (better < g.keep) {
                    stay |= 1u << h;
                    in = fminf(in, worth);
                } else {
                    out = fmaxf(out, worth);
                }
            }
#pragma unroll
            for (int o = LPR / 2; o; o >>= 1) {
                stay |= __shfl_xor_sync(ALL, stay, o);
                in = fminf(in, __shfl_xor_sync(ALL, in, o));
                out = fmaxf(out, __shfl_xor_sync(ALL, out, o));
            }
            // Half a worth's error: half of two scores', and three roundings of
            // numbers up to the largest score and |bias| (their sum may be small).
            const bool border = out > -INFINITY && in - out <= 2.0f * tell + 0x1p-21f * (1.0f + high_bias);
            if (__any_sync(ALL, border)) {
                // The worths in 64 bits, of each group's largest by the f32
                // scores (the long way, if those are not clear).
                double* exact = reinterpret_cast<double*>(mem + M::EXACT) + sub * FEW_LD;
                const double whole = g.sigmoid ? 1.0 : inverse_sum64<LPR>(g, row, r, m);
                bool unclear = false;
#pragma unroll 1
                for (int h = r; h < g.groups; h += LPR) {
                    float a = -INFINITY, b = -INFINITY, d = -INFINITY;
                    int ea = 0, eb = 0;
#pragma unroll 1
                    for (int e = h * g.group_size; e < (h + 1) * g.group_size; ++e) {
                        const float v = scores[e];
                        if (v > a) {
                            d = b, b = a, eb = ea;
                            a = v, ea = e;
                        } else if (v > b) {
                            d = b, b = v, eb = e;
                        } else {
                            d = fmaxf(d, v);
                        }
                    }
                    const bool two = g.group_top > 1 && b > -INFINITY;
                    const float last = two ? b : a, next = two ? d : b;
                    unclear |= last - next <= 2.0f * tell + 0x1p-21f * fabsf(last);
                    double w = -INFINITY;
                    if (a > -INFINITY) {
                        w = score64(g.sigmoid, load_one(g.logits, g.dtype, row * g.ld + ea), m, whole) + (double)bias[ea];
                        if (two) w += score64(g.sigmoid, load_one(g.logits, g.dtype, row * g.ld + eb), m, whole) + (double)bias[eb];
                    }
                    exact[h] = w;
                }
                __syncwarp();
                u32 keep = 0;
#pragma unroll 1
                for (int h = r; h < g.groups; h += LPR) {
                    int better = 0;
#pragma unroll 1
                    for (int x = 0; x < g.groups; ++x) better += exact[x] > exact[h] || (exact[x] == exact[h] && x < h);
                    if (better < g.keep) keep |= 1u << h;
                }
#pragma unroll 1
                for (int o = LPR / 2; o; o >>= 1) {
                    keep |= __shfl_xor_sync(ALL, keep, o);
                    unclear |= __shfl_xor_sync(ALL, (int)unclear, o) != 0;
                }
                if (border && !unclear) stay = keep;
                longer = border && unclear;
                __syncwarp();                            // exact is read
            }
            if (!g.bias) {                               // the order of the logits, among those that stay
                float l[V];
                load_quads<LPR, V>(g, row * g.ld, r, l);
#pragma unroll
                for (int i = 0; i < V; ++i) c[i] = l[i];
            }
#pragma unroll
            for (int q = 0; q < V / 4; ++q) {
                const int e = (q * LPR + r) * 4;
                if (g.group_size % 4 == 0) {
                    const bool kept = stay >> group_of(g, e) & 1u;
#pragma unroll
                    for (int j = 0; j < 4; ++j) c[4 * q + j] = kept ? c[4 * q + j] : -INFINITY;
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) c[4 * q + j] = stay >> group_of(g, e + j) & 1u ? c[4 * q + j] : -INFINITY;
                }
            }
        }
    }
    // The k-th largest of the lanes' largest-of-a-few (equal heads as one: no higher).
    constexpr int S = V < 8 ? V : 8, B = V / S;
    float s[S];
#pragma unroll
    for (int j = 0; j < S; ++j) {
        s[j] = c[j * B];
#pragma unroll
        for (int i = 1; i < B; ++i) s[j] = fmaxf(s[j], c[j * B + i]);
    }
    sort_down<S>(s);
    float bound = -INFINITY;
    for (int j = 0; j < g.k; ++j) {
        bound = row_max<LPR>(s[0]);
        const bool mine = s[0] == bound;
#pragma unroll
        for (int i = 0; i + 1 < S; ++i) s[i] = mine ? s[i + 1] : s[i];
        s[S - 1] = mine ? -INFINITY : s[S - 1];
    }
    if (g.bias) bound -= 4.0f * tell + 0x1p-20f * fabsf(bound);        // and all that may be as large in 64 bits
    if (!(bound > -INFINITY)) bound = -3.4028235e38f;    // shut ones stay out
    int n = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) n += c[i] >= bound;
    int at = n;                                          // places before this lane's
#pragma unroll
    for (int o = 1; o < LPR; o <<= 1) {
        const int u = __shfl_up_sync(ALL, at, o, LPR);
        if (r >= o) at += u;
    }
    const int total = __shfl_sync(ALL, at, sub * LPR + LPR - 1);
    at -= n;
    __syncwarp();                                        // few is cleared
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (c[i] >= bound) {
            if (at < MAX_FEW) few[at] = {c[i], (i / 4 * LPR + r) * 4 + i % 4};
            ++at;
        }
    __syncwarp();
    longer |= total > MAX_FEW;
    const int most_few = (int)__reduce_max_sync(ALL, longer ? 0u : (u32)total);
    const float slack = 2.0f * tell;
    bool near = false;
    for (int p = r; p - r < most_few; p += LPR) {
        const Few own = few[p];
        const float off = own.e < 0 ? -1.0f : slack + 0x1p-21f * fabsf(own.c);     // none behind the list's end
        int rank = 0;
        for (int q = 0; q < most_few; ++q) {
            const Few f = few[q];
            rank += f.c > own.c || (f.c == own.c && f.e < own.e);
            near |= q != p && fabsf(f.c - own.c) <= off;
        }
        if (own.e >= 0 && rank < g.k) choice[rank] = own.e;
    }
    if (g.bias && __any_sync(ALL, near && !longer)) {
        double* exact = reinterpret_cast<double*>(mem + M::EXACT) + sub * FEW_LD;
        const double whole = g.sigmoid ? 1.0 : inverse_sum64<LPR>(g, row, r, m);
#pragma unroll 1
        for (int p = r; p - r < most_few; p += LPR) {
            const int e = few[p].e;
            exact[p] = e >= 0 ? score64(g.sigmoid, load_one(g.logits, g.dtype, row * g.ld + e), m, whole) + (double)bias[e] : -INFINITY;
        }
        __syncwarp();
#pragma unroll 1
        for (int p = r; p - r < most_few; p += LPR) {
            const int e = few[p].e;
            const double own = exact[p];
            int rank = 0;
#pragma unroll 1
            for (int q = 0; q < most_few; ++q) rank += exact[q] > own || (exact[q] == own && few[q].e < e);
            if (e >= 0 && rank < g.k) choice[rank] = e;
        }
    }
    const u32 slow = __ballot_sync(ALL, longer && live && !bad && r == 0);
    for (u32 left = slow; left; left &= left - 1) {
        const int x = __ffs(left) - 1;
        __syncwarp();
        choose_long(g, first + x / LPR, lane, reinterpret_cast<double*>(mem + M::SCORES), reinterpret_cast<int*>(mem + M::CHOICE) + x / LPR * 32);
    }
    __syncwarp();
    // Weights.  Renormalised ones are made relative to the largest chosen, so
    // that they hold where all scores are tiny.
    int e[TURNS];
    float z[TURNS], high = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int t = 0; t < TURNS; ++t) {
        e[t] = -1;
        z[t] = 0.0f;
        const int j = t * LPR + r;
        if (t * LPR < g.k && j < g.k) {
            e[t] = bad ? j : choice[j];
            if (e[t] >= 0) {
                z[t] = load_one(g.logits, g.dtype, row * g.ld + e[t]);
                high = fmaxf(high, z[t]);
            }
        }
    }
    if (g.renorm) {
        high = row_max<LPR>(high);
#pragma unroll
        for (int t = 0; t < TURNS; ++t)
            if (t * LPR < g.k) {
                if (e[t] >= 0) z[t] = g.sigmoid ? expf(fminf(z[t], 0.0f) - fminf(high, 0.0f)) / (1.0f + expf(-fabsf(z[t]))) : expf(z[t] - high);
                sum += z[t];
            }
        sum = row_sum<LPR>(sum);
    }
#pragma unroll
    for (int t = 0; t < TURNS; ++t) {
        const int j = t * LPR + r;
        if (t * LPR < g.k && j < g.k && live) {
            float w = 0.0f;
            if (bad) w = NAN;
            else if (e[t] >= 0) w = (g.renorm ? z[t] / sum : g.sigmoid ? 1.0f / (1.0f + expf(-z[t])) : expf(z[t] - m) * inv) * g.scale;
            g.weights[row * g.k + j] = w;
            g.experts[row * g.k + j] = e[t];
            const int x = (int)(row - from);
            list[x * g.k + j] = e[t];
            if (e[t] >= 0) atomicOr(&masks[(x >> 5) * g.n + e[t]], 1u << (x & 31));
        }
    }
    __syncwarp();                                        // the list and the choice are read
}

// Exclusive sums of total[0 .. n) into first[0 .. n], by all threads; part: 32 words.
__device__ __forceinline__ void scan_counts(const int* total, int* first, int* part, int n) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    for (int w = warp; w * 32 < n; w += warps) {
        const int e = w * 32 + lane, t = e < n ? total[e] : 0;
        int v = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(ALL, v, o);
            if (lane >= o) v += u;
        }
        if (e < n) first[e] = v - t;
        if (lane == 31) part[w] = v;
    }
    __syncthreads();
    if (warp == 0) {
        int v = lane * 32 < n ? part[lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(ALL, v, o);
            if (lane >= o) v += u;
        }
        part[lane] = v;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < n; e += blockDim.x)
        if (e >= 32) first[e] += part[e / 32 - 1];
    if (threadIdx.x == 0) first[n] = part[31];
    __syncthreads();
}

// 128 registers a thread, for 32 scores and their sorted maxima.  (1024 threads
// of 64 registers, 16 lanes a row: 16384 x 256 30.6 us instead of 31.3, but
// every call of few rows 2 us longer.  256 threads: one row 0.7 us shorter than 7.5,
// 16 rows 2.4 longer than 8.5.)
constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
constexpr int BATCH = 128;             // rows whose choices a block numbers at a time
constexpr int WORDS = BATCH / 32;

// Shared memory of route_kernel, in bytes.
template <int LPR, int V> struct Layout {
    int bias, total, first, part, high, masks, list, warps, bytes;
    __host__ __device__ Layout(int n, int k) {
        bias = 0;
        total = bias + 4 * LPR * V;
        first = total + 4 * n;
        part = first + 4 * (n + 1);
        high = part + 128;
        masks = high + 4;
        list = masks + 4 * WORDS * n;
        warps = (list + 4 * BATCH * k + 15) & ~15;
        bytes = warps + WARPS * WarpMem<LPR, V>::BYTES;
    }
};

// Each block routes chunk_rows rows and numbers their choices, expert by
// expert; alone (FEW: one block, all rows) it makes the places of them.  A row
// has an expert once at most, so a choice's number is that of the earlier
// rows with its expert: a bit per row in the expert's mask.  (Numbering by
// matching lanes' experts took 400 clocks for 32 choices.)
template <int LPR, int V, bool FEW> __global__ void __launch_bounds__(THREADS, 1) route_kernel(const RouteArgs g) {
    extern __shared__ __align__(16) unsigned char smem[];
    if (!FEW) second_may_start();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Layout<LPR, V> at(g.n, g.k);
    float* bias = reinterpret_cast<float*>(smem + at.bias);
    int *total = reinterpret_cast<int*>(smem + at.total), *first = reinterpret_cast<int*>(smem + at.first);
    int *part = reinterpret_cast<int*>(smem + at.part), *list = reinterpret_cast<int*>(smem + at.list);
    u32* masks = reinterpret_cast<u32*>(smem + at.masks);              // [WORDS][n]
    int* high = reinterpret_cast<int*>(smem + at.high);                // bits of the largest finite |bias|
    if (threadIdx.x == 0) *high = 0;
    __syncthreads();
    bool bad = false;
    for (int e = threadIdx.x; e < LPR * V; e += THREADS) {
        const float b = g.bias && e < g.n ? g.bias[e] : 0.0f;
        bias[e] = b;
        bad |= !(b == b);
        if (g.groups > 1 && b != 0.0f && fabsf(b) < INFINITY) atomicMax(high, __float_as_int(fabsf(b)));
    }
    for (int e = threadIdx.x; e < g.n; e += THREADS) total[e] = 0;
    for (int i = threadIdx.x; i < WORDS * g.n; i += THREADS) masks[i] = 0u;
    bad = __syncthreads_or(bad);
    const int64_t a = blockIdx.x * g.chunk_rows, b = a + g.chunk_rows < g.rows ? a + g.chunk_rows : g.rows;
    constexpr int ROWS = WarpMem<LPR, V>::ROWS;
    unsigned char* mem = smem + at.warps + warp * WarpMem<LPR, V>::BYTES;
    for (int64_t from = a; from < b; from += BATCH) {
        const int64_t to = from + BATCH < b ? from + BATCH : b;
        for (int64_t row = from + warp * ROWS; row < to; row += WARPS * ROWS) route_rows<LPR, V>(g, row, to, lane, bias, bad, __int_as_float(*high), mem, list, masks, from);
        __syncthreads();
        if (FEW) {
            for (int e = threadIdx.x; e < g.n; e += THREADS) {
                int count = 0;
#pragma unroll
                for (int w = 0; w < WORDS; ++w) count += __popc(masks[w * g.n + e]);
                total[e] = count;
            }
            __syncthreads();
            scan_counts(total, first, part, g.n);
        }
        const int entries = (int)(to - from) * g.k;
        for (int i = threadIdx.x; i < entries; i += THREADS) {
            const int e = list[i], r = i / g.k;
            int p = -1;
            if (e >= 0) {
                p = FEW ? first[e] : total[e];
#pragma unroll
                for (int w = 0; w < WORDS; ++w) {
                    const u32 m = masks[w * g.n + e];
                    p += __popc(w < r >> 5 ? m : w == r >> 5 ? m & ((1u << (r & 31)) - 1u) : 0u);
                }
            }
            g.place[from * g.k + i] = p;
        }
        __syncthreads();
        if (!FEW) {
            for (int e = threadIdx.x; e < g.n; e += THREADS) {
                int count = total[e];
#pragma unroll
                for (int w = 0; w < WORDS; ++w) {
                    count += __popc(masks[w * g.n + e]);
                    masks[w * g.n + e] = 0u;
                }
                total[e] = count;
            }
            __syncthreads();
        }
    }
    if (FEW) {
        if (g.rows == 0) scan_counts(total, first, part, g.n);
        for (int e = threadIdx.x; e <= g.n; e += THREADS) g.offsets[e] = first[e];
    } else if (g.byte_counts) {
        unsigned char* counts = static_cast<unsigned char*>(g.counts) + (int64_t)blockIdx.x * g.counts_ld;
        for (int e = threadIdx.x; e < g.counts_ld; e += THREADS) counts[e] = e < g.n ? (unsigned char)total[e] : 0;
    } else {
        int* counts = static_cast<int*>(g.counts) + (int64_t)blockIdx.x * g.counts_ld;
        for (int e = threadIdx.x; e < g.counts_ld; e += THREADS) counts[e] = e < g.n ? total[e] : 0;
    }
}

// Adds the counts of the experts before, and of the blocks before.  Every block
// reads all counts, which is what it takes time for (148 blocks x 256 experts
// in 32 bits: 22 MB through L2, 9 us); up to 255 rows a block's are bytes.
constexpr int PLACE_THREADS = 1024;
__global__ void __launch_bounds__(PLACE_THREADS, 1) place_kernel(const RouteArgs g) {
    __shared__ int total[MAX_EXPERTS + 16], first[MAX_EXPERTS + 1], before[MAX_EXPERTS + 16], part[32];
    for (int e = threadIdx.x; e < MAX_EXPERTS + 16; e += PLACE_THREADS) total[e] = before[e] = 0;
    __syncthreads();
    first_is_done();
    const int64_t a = blockIdx.x * g.chunk_rows * g.k, all = g.rows * g.k;
    const int64_t b = a + g.chunk_rows * g.k < all ? a + g.chunk_rows * g.k : all;
    // this thread's first choice, on its way while the counts are summed
    const int64_t i0 = a + threadIdx.x;
    const int e0 = i0 < b ? __ldcg(&g.experts[i0]) : -1, p0 = i0 < b ? __ldcg(&g.place[i0]) : -1;
    if (g.byte_counts) {
        // eight experts a thread, as pairs of 16 bits: at most 255 x 256 blocks
        const int units = g.counts_ld / 8, parts = PLACE_THREADS / units, turn = threadIdx.x / units, mine = threadIdx.x % units;
        if (turn < parts) {
            u32 sum[4] = {0, 0, 0, 0}, early[4] = {0, 0, 0, 0};
#pragma unroll 8
            for (int c = turn; c < g.chunks; c += parts) {
                const uint2 v = __ldcg(reinterpret_cast<const uint2*>(static_cast<const unsigned char*>(g.counts) + (int64_t)c * g.counts_ld) + mine);
                const u32 h[4] = {v.x & 0x00FF00FFu, v.x >> 8 & 0x00FF00FFu, v.y & 0x00FF00FFu, v.y >> 8 & 0x00FF00FFu};
                const u32 keep = c < (int)blockIdx.x ? ALL : 0u;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sum[i] += h[i];
                    early[i] += h[i] & keep;
                }
            }
            // Few experts: a warp's lanes have the same ones, and their sums
            // would wait for one another (8 experts: 15.8 us for the call, 64 10.5).
            const bool alike = units < 32 && !(units & (units - 1));
            if (alike)
                for (int o = 16; o >= units; o >>= 1)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        sum[i] += __shfl_xor_sync(ALL, sum[i], o);
                        early[i] += __shfl_xor_sync(ALL, early[i], o);
                    }
            if (!alike || (threadIdx.x & 31) < units)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int word = i / 4 * 2 + (i & 1), up = (i >> 1 & 1) * 16;      // bytes 0, 2 and 1, 3 of a word
                atomicAdd(&total[mine * 8 + i], (int)(sum[word] >> up & 0xFFFFu));
                atomicAdd(&before[mine * 8 + i], (int)(early[word] >> up & 0xFFFFu));
            }
        }
    } else {
        const int parts = PLACE_THREADS / g.n;           // at least 1: n <= 1024
        const int turn = threadIdx.x / g.n, mine = threadIdx.x % g.n;
        if (turn < parts) {
            int sum = 0, early = 0;
#pragma unroll 16
            for (int c = turn; c < g.chunks; c += parts) {
                const int v = __ldcg(static_cast<const int*>(g.counts) + (int64_t)c * g.counts_ld + mine);
                sum += v;
                early += c < (int)blockIdx.x ? v : 0;
            }
            atomicAdd(&total[mine], sum);
            atomicAdd(&before[mine], early);
        }
    }
    __syncthreads();
    scan_counts(total, first, part, g.n);
    if (blockIdx.x == 0)
        for (int e = threadIdx.x; e <= g.n; e += PLACE_THREADS) g.offsets[e] = first[e];
    if (e0 >= 0) g.place[i0] = p0 + first[e0] + before[e0];
    for (int64_t i = i0 + PLACE_THREADS; i < b; i += PLACE_THREADS) {
        const int e = __ldcg(&g.experts[i]);
        if (e >= 0) g.place[i] = __ldcg(&g.place[i]) + first[e] + before[e];
    }
}

struct RouteGradArgs {
    const float* dweights;
    const void* logits;
    const int* experts;
    void* dlogits;
    int64_t dw_ld, ld, e_ld, out_ld, rows;
    int n, k, dtype, sigmoid, renorm;
    float scale;
};

// Gradient, a warp a row.  With g = scale * dweights at the chosen experts:
//   softmax                  dz_i = p_i (g_i - sum_j p_j g_j)
//   softmax, renormalised    dz_i = q_i (g_i - sum_j q_j g_j), q = softmax over the chosen
//   sigmoid                  dz_i = g_i s_i (1 - s_i)
//   sigmoid, renormalised    dz_i = (1 - s_i) q_i (g_i - sum_j q_j g_j), q = s over the chosen ones' sum
// Only the first reads the whole row.  Lane j computes choice j, from the
// logit it loads again, and stores it over what the row's lanes stored.
template <int V> __device__ __forceinline__ void load_row(const void* p, int dtype, int64_t at, int n, int lane, float (&l)[V]) {
    auto all = [&](auto* src) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int e = i * 32 + lane;
            l[i] = e < n ? to_f32(src[at + e]) : -INFINITY;
        }
    };
    if (dtype == BAFE_DTYPE_F32) all(static_cast<const float*>(p));
    else if (dtype == BAFE_DTYPE_BF16) all(static_cast<const __nv_bfloat16*>(p));
    else all(static_cast<const __half*>(p));
}

template <int V> __global__ void __launch_bounds__(256) route_grad_kernel(const RouteGradArgs g) {
    const int lane = threadIdx.x & 31;
    for (int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); row < g.rows; row += (int64_t)gridDim.x * 8) {
        int e = lane < g.k ? g.experts[row * g.e_ld + lane] : -1;
        if (e >= g.n) e = -1;
        const float dw = e >= 0 ? g.dweights[row * g.dw_ld + lane] * g.scale : 0.0f;
        const float z = e >= 0 ? load_one(g.logits, g.dtype, row * g.ld + e) : -INFINITY;
        float p[V], dz = 0.0f, dot = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) p[i] = 0.0f;
        if (!g.sigmoid && !g.renorm) {
            load_row<V>(g.logits, g.dtype, row * g.ld, g.n, lane, p);
            float m = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) m = max_nan(m, p[i]);
            m = warp_max_nan(m);
            if (m == -INFINITY) m = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                p[i] = expf(p[i] - m);
                sum += p[i];
            }
            sum = lm::warp_sum(sum);
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            const float mine = e >= 0 ? expf(z - m) * inv : 0.0f;
            dot = lm::warp_sum(mine * dw);
            dz = mine * (dw - dot);
#pragma unroll
            for (int i = 0; i < V; ++i) p[i] *= -dot * inv;
        } else {
            const float tail = expf(-fabsf(z));          // s = 1 / (1 + tail) or tail / (1 + tail)
            if (g.renorm) {
                const float top = warp_max_nan(z);
                float num = 0.0f;
                if (e >= 0) num = g.sigmoid ? expf(fminf(z, 0.0f) - fminf(top, 0.0f)) / (1.0f + tail) : expf(z - top);
                const float sum = lm::warp_sum(num);
                const float q = e >= 0 ? num / sum : 0.0f;
                dot = lm::warp_sum(q * dw);
                dz = q * (dw - dot);
                if (g.sigmoid) dz *= (z > 0.0f ? tail : 1.0f) / (1.0f + tail);
            } else {
                dz = dw * (tail / (1.0f + tail)) / (1.0f + tail);
            }
        }
        auto store = [&](auto* out) {
            typedef typename std::remove_pointer<decltype(out)>::type T;
            out += row * g.out_ld;
            __syncwarp();                                // the logits may lie there: all lanes have read theirs
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i * 32 + lane < g.n) out[i * 32 + lane] = from_f32<T>(p[i]);
            __syncwarp();
            if (e >= 0) out[e] = from_f32<T>(dz);
        };
        if (g.dtype == BAFE_DTYPE_F32) store(static_cast<float*>(g.dlogits));
        else if (g.dtype == BAFE_DTYPE_BF16) store(static_cast<__nv_bfloat16*>(g.dlogits));
        else store(static_cast<__half*>(g.dlogits));
    }
}

// Chunks of the rows: a block each.
int64_t chunks_of(int64_t rows, int sms) {
    const int64_t most = (rows + 31) / 32;
    return most < sms ? (most < 1 ? 1 : most) : sms;
}

// Whether a block's counts fit into bytes, and the second kernel's sums of them into 16 bits.
bool bytes_suffice(int64_t rows, int sms) {
    const int64_t chunks = chunks_of(rows, sms);
    return chunks <= 256 && (rows + chunks - 1) / chunks <= 255;
}
int64_t counts_bytes(int64_t rows, int64_t n, int sms) { return (n + 7) / 8 * 8 * (bytes_suffice(rows, sms) ? 1 : 4); }

// Lets a kernel have more than 48 KB of shared memory.
template <auto KERNEL> int more_smem(int bytes, int dev) {
    static bool ready[64] = {false};
    if (bytes <= 48 * 1024 || ready[dev]) return 0;
    if (cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) != cudaSuccess) {
        cudaGetLastError();
        return fail(14, "route: cudaFuncSetAttribute");
    }
    ready[dev] = true;
    return 0;
}

template <int LPR, int V> int launch_few(RouteArgs& g, int dev, cudaStream_t st) {
    const int bytes = Layout<LPR, V>(g.n, g.k).bytes;
    if (int rc = more_smem<route_kernel<LPR, V, true>>(bytes, dev)) return rc;
    g.chunk_rows = g.rows;
    route_kernel<LPR, V, true><<<1, THREADS, bytes, st>>>(g);
    return launched("route");
}
template <int LPR, int V> int launch_route(RouteArgs& g, int dev, cudaStream_t st) {
    if (g.rows <= SMALL_ROWS) return launch_few<LPR, V>(g, dev, st);
    const int bytes = Layout<LPR, V>(g.n, g.k).bytes;
    if (int rc = more_smem<route_kernel<LPR, V, false>>(bytes, dev)) return rc;
    route_kernel<LPR, V, false><<<g.chunks, THREADS, bytes, st>>>(g);
    if (int rc = launched("route")) return rc;
    return launch_second("route: places", place_kernel, dim3((unsigned)g.chunks), dim3(PLACE_THREADS), st, g);
}

int check_sizes(const char* what, int64_t rows, int64_t n, int64_t k) {
    if (rows < 0 || n < 1 || n > MAX_EXPERTS || k < 1 || k > MAX_K || k > n || rows > (int64_t(1) << 30) / k)
        return fail(8, std::string(what) + ": sizes out of range (1 <= k <= min(experts, 31), experts <= 1024, 0 <= rows * k <= 2^30)");
    return 0;
}

template <class F> int with_slots(int n, F f) {
    const int v = (n + 31) / 32;
    if (v <= 1) return f(std::integral_constant<int, 1>());
    if (v <= 2) return f(std::integral_constant<int, 2>());
    if (v <= 4) return f(std::integral_constant<int, 4>());
    if (v <= 8) return f(std::integral_constant<int, 8>());
    if (v <= 16) return f(std::integral_constant<int, 16>());
    return f(std::integral_constant<int, 32>());
}

}  // namespace
}  // namespace lm
}  // namespace bafe_cuda

#define BAFE_API extern "C" __attribute__((visibility("default")))

using namespace bafe_cuda;
using namespace bafe_cuda::lm;

BAFE_API int64_t bafe_cuda_route_workspace(int64_t rows, int64_t experts, int64_t k) {
    if (check_sizes("route", rows, experts, k)) return -1;
    if (rows <= SMALL_ROWS) return 0;
    int dev = 0, sms = 0;
    if (current_device(dev, sms)) return -1;
    return chunks_of(rows, sms) * counts_bytes(rows, experts, sms);
}

BAFE_API int bafe_cuda_route(const void* logits, int64_t ld, const float* bias, float* weights, int* experts, int* offsets,
                             int* place, int64_t rows, int64_t n, int64_t k, int64_t groups, int64_t keep_groups,
                             int group_top, int score, int renormalize, double scale, int dtype, void* workspace,
                             int64_t workspace_bytes, void* stream) {
    if (int rc = check_sizes("route", rows, n, k)) return rc;
    if (!is_float_type(dtype)) return fail(8, "route: logits must be f32, f16 or bf16");
    if (score != BAFE_CUDA_SCORE_SOFTMAX && score != BAFE_CUDA_SCORE_SIGMOID) return fail(8, "route: unknown score");
    if (groups < 1 || groups > MAX_GROUPS || n % groups || keep_groups < 1 || keep_groups > groups ||
        k > n / groups * keep_groups || group_top < 1 || group_top > 2)
        return fail(8, "route: groups must divide the experts (at most 32), the kept ones hold k experts, group_top be 1 or 2");
    if (!offsets || (rows && (!logits || !weights || !experts || !place))) return fail(8, "route: null operand");
    if (rows > 1 && ld < n) return fail(8, "route: strides must be at least the rows' lengths");
    if (!element_aligned(dtype == BAFE_DTYPE_F32 ? 4 : 2, {logits}) || !element_aligned(4, {bias, weights, experts, offsets, place}))
        return fail(8, "route: operands must start on a multiple of their element's size");
    const float fscale = (float)scale;
    if (!std::isfinite(fscale)) return fail(8, "route: scale must be finite");
    int dev = 0, sms = 0;
    if (int rc = current_device(dev, sms)) return rc;
    RouteArgs g = {};
    g.logits = logits;
    g.bias = bias;
    g.weights = weights;
    g.experts = experts;
    g.offsets = offsets;
    g.place = place;
    g.ld = ld;
    g.rows = rows;
    g.n = (int)n;
    g.k = (int)k;
    g.groups = (int)(keep_groups == groups ? 1 : groups);             // nothing to leave out
    g.keep = (int)keep_groups;
    g.group_size = (int)(n / groups);
    g.group_top = group_top;
    g.group_inverse = (u32)((0x100000000ull + (u32)g.group_size - 1) / (u32)g.group_size);
    g.dtype = dtype;
    g.sigmoid = score == BAFE_CUDA_SCORE_SIGMOID;
    g.renorm = renormalize != 0;
    g.scale = fscale;
    if (rows > SMALL_ROWS) {
        const int64_t chunks = chunks_of(rows, sms);
        if (!workspace || workspace_bytes < chunks * counts_bytes(rows, n, sms) || !element_aligned(8, {workspace}))
            return fail(8, "route: workspace too small or unaligned (see bafe_cuda_route_workspace)");
        g.counts = workspace;
        g.chunk_rows = (rows + chunks - 1) / chunks;
        g.byte_counts = bytes_suffice(rows, sms);
        g.counts_ld = (int)((n + 7) / 8 * 8);
        g.chunks = (int)((rows + g.chunk_rows - 1) / g.chunk_rows);
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int es = dtype == BAFE_DTYPE_F32 ? 4 : 2;
    g.vec = n % 4 == 0 && ((uintptr_t)logits | (uintptr_t)(rows > 1 ? ld * es : 0)) % (4 * es) == 0;
    // A row a warp: whole warps share a row, whose code is a quarter as long
    // (one row of 256 experts 7.5 us, 10.1 with eight lanes; 64 rows 13.8 so, in
    // four turns).
    if (rows <= WARPS) {
        if (n <= 128) return launch_few<32, 4>(g, dev, st);
        if (n <= 256) return launch_few<32, 8>(g, dev, st);
        if (n <= 512) return launch_few<32, 16>(g, dev, st);
    }
    if (n <= 32) return launch_route<8, 4>(g, dev, st);
    if (n <= 64) return launch_route<8, 8>(g, dev, st);
    if (n <= 128) return launch_route<8, 16>(g, dev, st);
    if (n <= 256) return launch_route<8, 32>(g, dev, st);
    if (n <= 512) return launch_route<16, 32>(g, dev, st);
    return launch_route<32, 32>(g, dev, st);
}

BAFE_API int bafe_cuda_route_grad(const float* dweights, int64_t dweights_ld, const void* logits, int64_t ld,
                                  const int* experts, int64_t experts_ld, void* dlogits, int64_t dlogits_ld, int64_t rows,
                                  int64_t n, int64_t k, int score, int renormalize, double scale, int dtype, void* stream) {
    if (int rc = check_sizes("route_grad", rows, n, k)) return rc;
    if (!is_float_type(dtype)) return fail(8, "route_grad: logits must be f32, f16 or bf16");
    if (score != BAFE_CUDA_SCORE_SOFTMAX && score != BAFE_CUDA_SCORE_SIGMOID) return fail(8, "route_grad: unknown score");
    if (rows == 0) return 0;
    if (!dweights || !logits || !experts || !dlogits) return fail(8, "route_grad: null operand");
    if (rows > 1 && (ld < n || dlogits_ld < n || dweights_ld < 0 || experts_ld < k))
        return fail(8, "route_grad: strides must be at least the rows' lengths");
    if (!element_aligned(dtype == BAFE_DTYPE_F32 ? 4 : 2, {logits, dlogits}) || !element_aligned(4, {dweights, experts}))
        return fail(8, "route_grad: operands must start on a multiple of their element's size");
    const float fscale = (float)scale;
    if (!std::isfinite(fscale)) return fail(8, "route_grad: scale must be finite");
    int dev = 0, sms = 0;
    if (int rc = current_device(dev, sms)) return rc;
    RouteGradArgs g = {};
    g.dweights = dweights;
    g.logits = logits;
    g.experts = experts;
    g.dlogits = dlogits;
    g.dw_ld = dweights_ld;
    g.ld = ld;
    g.e_ld = experts_ld;
    g.out_ld = dlogits_ld;
    g.rows = rows;
    g.n = (int)n;
    g.k = (int)k;
    g.dtype = dtype;
    g.sigmoid = score == BAFE_CUDA_SCORE_SIGMOID;
    g.renorm = renormalize != 0;
    g.scale = fscale;
    const int64_t blocks = (rows + 7) / 8, most = (int64_t)sms * 8;
    const unsigned grid = (unsigned)(blocks < most ? blocks : most);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return with_slots(g.n, [&](auto v) {
        route_grad_kernel<decltype(v)::value><<<grid, 256, 0, st>>>(g);
        return launched("route_grad");
    });
}
