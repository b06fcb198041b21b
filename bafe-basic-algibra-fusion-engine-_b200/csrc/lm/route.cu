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
// A warp takes a row, expert i * 32 + lane in slot i of a lane's registers.
// The k-th largest of the 32 lanes' largest is a lower bound of the k-th
// largest of all; the few experts above it (k and some) move into one lane
// each, and every lane counts those that come before its own.  (Picking the
// largest k + 1 times in turn took 1900 instructions a row of 256, this 600.)
// Rows with more than 32 such experts take the long way, one expert a round.
//
// The order is the one of the scores in 64 bits: two f32 scores nearer to one
// another than their errors could be the other way round.  Experts that near
// are among the few; where there are any, the few scores are made again in 64
// bits (sigmoid), or the whole row is (softmax, and groups near to one another at the
// border).  Without bias and groups the logits themselves have the scores'
// order, and nothing is computed for the choice.
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
constexpr int MAX_K = 31;              // the 32nd lane holds the runner-up
constexpr int MAX_GROUPS = 32;
constexpr int SMALL_ROWS = 64;         // rows that one block routes and sorts

struct RouteArgs {
    const void* logits;
    const float* bias;                 // [experts], or null
    float* weights;                    // [rows][k]
    int* experts;                      // [rows][k]
    int* offsets;                      // [n + 1]
    int* place;                        // [rows][k]
    int* counts;                       // [chunks][n]: choices of each block's rows per expert
    int64_t ld, rows, chunk_rows;
    int n, k, groups, keep, group_size, group_top, chunks;
    int dtype, sigmoid, renorm;
    float scale;
};

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
__device__ __forceinline__ float load_one(const void* p, int dtype, int64_t at) {
    if (dtype == BAFE_DTYPE_F32) return static_cast<const float*>(p)[at];
    if (dtype == BAFE_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]);
    return __half2float(static_cast<const __half*>(p)[at]);
}

// Largest of the lanes' values (no NaN among them): as unsigned numbers of the same
// order, which one instruction reduces.
__device__ __forceinline__ float warp_max(float v) {
    u32 b = __float_as_uint(v);
    b ^= (u32)((int)b >> 31) | 0x80000000u;
    b = __reduce_max_sync(ALL, b);
    b ^= b & 0x80000000u ? 0x80000000u : ALL;
    return __uint_as_float(b);
}
__device__ __forceinline__ double warp_max(double v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmax(v, __shfl_xor_sync(ALL, v, o));
    return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(ALL, v, o);
    return v;
}

// The `rounds` largest of c (shut ones are -inf): lane r gets the index and
// value of the r-th, -1 and -inf if there are no more.
template <class F, int V> __device__ __forceinline__ void choose(F (&c)[V], int rounds, int lane, int& my_e, F& my_c) {
    const F shut = -INFINITY;
    F top = shut;
    int slot = 0;
    auto look = [&]() {
        top = c[0];
        slot = 0;
#pragma unroll
        for (int i = 1; i < V; ++i)
            if (c[i] > top) {
                top = c[i];
                slot = i;
            }
    };
    look();
    my_e = -1;
    my_c = shut;
    for (int r = 0; r < rounds; ++r) {
        const F best = warp_max(top);
        if (!(best > shut)) break;
        const u32 who = __ballot_sync(ALL, top == best);
        int e = slot * 32 + lane;
        if (who & (who - 1)) e = (int)__reduce_min_sync(ALL, top == best ? (u32)e : ALL);
        else e = __shfl_sync(ALL, e, __ffs(who) - 1);
        if (lane == r) {
            my_e = e;
            my_c = best;
        }
        if (lane == (e & 31)) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i == e >> 5) c[i] = shut;
            look();
        }
    }
}

// Groups have 2^shift lanes each (32 over the next power of two of their
// number), and bit[i] is the first lane of the group of slot i's expert.
__device__ __forceinline__ int group_shift(const RouteArgs& g) { return g.groups > 1 ? __clz(g.groups - 1) - 27 : 5; }
template <int V> __device__ __forceinline__ void group_bits(const RouteArgs& g, int lane, u32 (&bit)[V]) {
    const int shift = group_shift(g);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int e = i * 32 + lane;
        bit[i] = g.groups > 1 && e < g.n ? 1u << (e / g.group_size << shift) : 1u;
    }
}

// Shuts the experts of the groups that are not kept; buf: n values.  Returns
// whether the worst kept and the best other group differ by no more than
// `slack` (the errors of four scores).
template <class F, int V>
__device__ __forceinline__ bool keep_groups(const RouteArgs& g, F (&c)[V], const u32 (&bit)[V], F* buf, int lane, F slack) {
    const F shut = -INFINITY;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (i * 32 + lane < g.n) buf[i * 32 + lane] = c[i];
    __syncwarp();
    // lanes per group: a power of two
    const int shift = group_shift(g), per = 1 << shift, mine = lane >> shift;
    F a = shut, b = shut;
    if (mine < g.groups)
        for (int i = lane & (per - 1); i < g.group_size; i += per) {
            const F v = buf[mine * g.group_size + i];
            b = fmax(b, fmin(a, v));
            a = fmax(a, v);
        }
    for (int o = per >> 1; o; o >>= 1) {
        const F a2 = __shfl_xor_sync(ALL, a, o), b2 = __shfl_xor_sync(ALL, b, o);
        b = fmax(fmax(b, b2), fmin(a, a2));
        a = fmax(a, a2);
    }
    const F worth = g.group_top > 1 && b > shut ? a + b : a;
    int better = 0;
    for (int h = 0; h < g.groups; ++h) {
        const F w = __shfl_sync(ALL, worth, h << shift);
        better += w > worth || (w == worth && h < mine);
    }
    const bool kept = mine < g.groups && better < g.keep;
    const u32 stay = __ballot_sync(ALL, kept);
    const F in = -warp_max(kept ? -worth : shut), out = warp_max(mine < g.groups && !kept ? worth : shut);
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (!(stay & bit[i])) c[i] = shut;
    return out > shut && in - out <= slack + F(0x1p-21) * (fabs(in) + fabs(out));
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

// A row's choice in 64 bits, one expert a round: lane j < k returns choice j.
template <int V> __device__ __noinline__ int choose_long(const RouteArgs& g, int64_t row, int lane, double* buf) {
    float l[V];
    load_row<V>(g.logits, g.dtype, row * g.ld, g.n, lane, l);
    double d[V], unused;
    if (g.bias || g.groups > 1) {
        if (g.sigmoid) {
#pragma unroll
            for (int i = 0; i < V; ++i) d[i] = 1.0 / (1.0 + exp(-(double)l[i]));
        } else {
            float m = -INFINITY;
#pragma unroll
            for (int i = 0; i < V; ++i) m = fmaxf(m, l[i]);
            m = warp_max(m);
            if (!(m > -INFINITY)) m = 0.0f;
            double z = 0.0;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                d[i] = exp((double)l[i] - (double)m);
                z += d[i];
            }
            z = warp_sum(z);
#pragma unroll
            for (int i = 0; i < V; ++i) d[i] /= z;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (g.bias && i * 32 + lane < g.n) d[i] += (double)g.bias[i * 32 + lane];
            if (!(l[i] > -INFINITY)) d[i] = -INFINITY;
        }
        if (g.groups > 1) {
            u32 bit[V];
            group_bits<V>(g, lane, bit);
            keep_groups<double, V>(g, d, bit, buf, lane, 0.0);
        }
    }
    if (!g.bias) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (g.groups <= 1 || d[i] > -INFINITY) d[i] = l[i];
    }
    int e;
    choose<double, V>(d, g.k, lane, e, unused);
    return e;
}

struct Few {                           // an expert that may be chosen
    float c;
    int e;
};

// Routes a row; few: 32 entries, buf: 8 bytes per expert where there are groups.
template <int V>
__device__ __forceinline__ void route_row(const RouteArgs& g, int64_t row, int lane, const float (&bias)[V], const u32 (&bit)[V],
                                          bool bad_bias, Few* few, void* buf) {
    float l[V], c[V];
    load_row<V>(g.logits, g.dtype, row * g.ld, g.n, lane, l);
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < V; ++i) m = max_nan(m, l[i]);
    const bool nan = __any_sync(ALL, !(m == m) || bad_bias);
    const bool scored = g.bias || g.groups > 1;          // else the logits have the scores' order
    if (!g.sigmoid) m = warp_max(m);
    if (nan || (!g.sigmoid && m == INFINITY)) {          // a softmax of infinities has no value
        if (lane < g.k) {
            g.weights[row * g.k + lane] = NAN;
            g.experts[row * g.k + lane] = lane;
        }
        return;
    }
    if (!(m > -INFINITY)) m = 0.0f;
    float inv = 1.0f;                                    // of the softmax's sum
    if (!g.sigmoid && (scored || !g.renorm)) {
        float z = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            c[i] = exp2_fast((l[i] - m) * LOG2E);
            z += c[i];
        }
        inv = inverse_fast(fmaxf(lm::warp_sum(z), 1e-30f));
    }
    // Errors of the f32 scores, relative: the exponent's rounding counts as up
    // to |l| or |l - m| <= 88 half ulps (further down the score is 0), the others'
    // as a few, the softmax's sum's as up to 36; 128 ulps (2^-17) are allowed.
    const float tell = 0x1p-17f, most = g.sigmoid ? 1.0f : inv;
    bool longer = false;
    if (scored) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            c[i] = (g.sigmoid ? inverse_fast(1.0f + exp2_fast(-LOG2E * l[i])) : c[i] * inv) + bias[i];
            if (!(l[i] > -INFINITY)) c[i] = -INFINITY;
        }
        if (g.groups > 1) {
            longer = keep_groups<float, V>(g, c, bit, static_cast<float*>(buf), lane, tell * 4.0f * most);
            if (!g.bias) {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (c[i] > -INFINITY) c[i] = l[i];
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) c[i] = l[i];
    }
    // The k-th largest of the lanes' largest (equal lanes as one: no higher).
    float top = c[0];
#pragma unroll
    for (int i = 1; i < V; ++i) top = fmaxf(top, c[i]);
    u32 key = __float_as_uint(top), last = 0;
    key = top > -INFINITY ? key ^ ((u32)((int)key >> 31) | 0x80000000u) : 0u;
    for (int r = 0; r < g.k; ++r) {
        last = __reduce_max_sync(ALL, key);
        if (key == last) key = 0u;
    }
    float bound = last ? __uint_as_float(last ^ (last & 0x80000000u ? 0x80000000u : ALL)) : -INFINITY;
    if (g.bias) bound -= 4.0f * tell * (most + fabsf(bound));          // and all that may be as large in 64 bits
    if (!(bound > -INFINITY)) bound = -3.4028235e38f;    // shut ones stay out
    int n = 0;
    const u32 before = (1u << lane) - 1u;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const bool in = c[i] >= bound;
        const u32 who = __ballot_sync(ALL, in);
        const int at = n + __popc(who & before);
        if (in && at < 32) few[at] = {c[i], i * 32 + lane};
        n += __popc(who);
    }
    __syncwarp();
    longer |= n > 32;
    int e = -1, rank = 32;
    float mine = 0.0f;
    if (!longer) {
        Few own = {-INFINITY, -1};
        if (lane < n) {
            own = few[lane];
            mine = load_one(g.logits, g.dtype, row * g.ld + own.e);
            e = own.e;
            rank = 0;
        }
        const float off = 2.0f * tell * most + 0x1p-21f * fabsf(own.c);
        bool near = false;
        for (int q = 0; q < n; ++q) {
            const Few f = few[q];
            rank += f.c > own.c || (f.c == own.c && f.e < own.e);
            near |= q != lane && fabsf(f.c - own.c) <= off;
        }
        if (g.bias && __any_sync(ALL, near && lane < n)) {
            if (g.sigmoid) {
                const double d = e >= 0 ? 1.0 / (1.0 + exp(-(double)mine)) + (double)g.bias[e] : -INFINITY;
                rank = lane < n ? 0 : 32;
                for (int q = 0; q < n; ++q) {
                    const double f = __shfl_sync(ALL, d, q);
                    const int fe = __shfl_sync(ALL, e, q);
                    rank += f > d || (f == d && fe < e);
                }
            } else {
                longer = true;
            }
        }
        n = min(n, g.k);
    }
    if (__any_sync(ALL, longer)) {
        e = choose_long<V>(g, row, lane, static_cast<double*>(buf));
        rank = lane;
        if (e >= 0) mine = load_one(g.logits, g.dtype, row * g.ld + e);
        n = __popc(__ballot_sync(ALL, e >= 0));
        if (e < 0) rank = 32;
    }
    __syncwarp();                                        // few is read: the next row may write it
    const bool chosen = rank < g.k;
    // Weights.  Renormalised ones are made relative to the largest chosen, so
    // that they hold where all scores are tiny.
    float w;
    if (g.renorm) {
        const float high = warp_max(chosen ? mine : -INFINITY);
        const float num = !chosen ? 0.0f
                          : g.sigmoid ? expf(fminf(mine, 0.0f) - fminf(high, 0.0f)) / (1.0f + expf(-fabsf(mine)))
                                      : expf(mine - high);
        w = num / lm::warp_sum(num);
    } else {
        w = g.sigmoid ? 1.0f / (1.0f + expf(-mine)) : expf(mine - m) * inv;
    }
    if (chosen) {
        g.weights[row * g.k + rank] = w * g.scale;
        g.experts[row * g.k + rank] = e;
    }
    if (lane >= n && lane < g.k) {                       // no open expert left
        g.weights[row * g.k + lane] = 0.0f;
        g.experts[row * g.k + lane] = -1;
    }
}

// Exclusive sums of tot[0 .. n) into first[0 .. n]; one warp.
__device__ __forceinline__ void scan_counts(const int* tot, int* first, int n, int lane) {
    int carry = 0;
    for (int b = 0; b < n; b += 32) {
        const int e = b + lane, t = e < n ? tot[e] : 0;
        int v = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(ALL, v, o);
            if (lane >= o) v += u;
        }
        if (e < n) first[e] = carry + v - t;
        carry += __shfl_sync(ALL, v, 31);
    }
    if (lane == 0) first[n] = carry;
}

// Numbers entries [a, b) of the choices, each expert's from `base` of it on (0
// without); cnt is [warps][n] zeros, each warp takes a run of consecutive
// entries.  total[e], where given: the entries of expert e.
__device__ __forceinline__ void number_choices(const RouteArgs& g, int64_t a, int64_t b, int* cnt, int* total) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const int per = (((int)(b - a) + warps - 1) / warps + 31) & ~31;
    int* mine = cnt + warp * g.n;
    const u32 before = (1u << lane) - 1u;
    const int64_t first = a + (int64_t)warp * per, end = first + per < b ? first + per : b;
    for (int64_t i = first; i < end; i += 32) {
        const int e = i + lane < end ? g.experts[i + lane] : -1;
        const u32 same = __match_any_sync(ALL, e);
        if (e >= 0 && !(same & before)) mine[e] += __popc(same);
        __syncwarp();
    }
    __syncthreads();
    for (int e = threadIdx.x; e < g.n; e += blockDim.x) {
        int run = 0;
#pragma unroll 8
        for (int w = 0; w < warps; ++w) {
            const int t = cnt[w * g.n + e];
            cnt[w * g.n + e] = run;
            run += t;
        }
        total[e] = run;
    }
    __syncthreads();
    for (int64_t i = first; i < end; i += 32) {
        const int e = i + lane < end ? g.experts[i + lane] : -1;
        const u32 same = __match_any_sync(ALL, e);
        const int p = e >= 0 ? mine[e] + __popc(same & before) : -1;
        if (i + lane < end) g.place[i + lane] = p;
        __syncwarp();
        if (e >= 0 && !(same & before)) mine[e] += __popc(same);
        __syncwarp();
    }
}

template <int V> constexpr int THREADS = V <= 8 ? 1024 : 512;          // 64 registers a thread hold 8 slots, not 16

// Shared memory of route_kernel, in bytes: counts and their sums, the few, the groups' scores.
struct Layout {
    int total, first, cnt, few, buf, bytes;
    __host__ __device__ Layout(int n, int warps, bool groups) {
        total = 0;
        first = total + 4 * n;
        cnt = first + 4 * (n + 1);
        few = (cnt + 4 * n * warps + 7) & ~7;
        buf = few + 256 * warps;
        bytes = buf + (groups ? 8 * n * warps : 0);
    }
};

// Each block routes chunk_rows rows and numbers their choices; alone (FEW:
// one block, all rows) it makes the places of them.
template <int V, bool FEW> __global__ void __launch_bounds__(THREADS<V>, 1) route_kernel(const RouteArgs g) {
    extern __shared__ __align__(16) unsigned char smem[];
    if (!FEW) second_may_start();
    constexpr int WARPS = THREADS<V> / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Layout at(g.n, WARPS, g.groups > 1);
    int *total = reinterpret_cast<int*>(smem + at.total), *first = reinterpret_cast<int*>(smem + at.first);
    int* cnt = reinterpret_cast<int*>(smem + at.cnt);
    for (int i = threadIdx.x; i < WARPS * g.n; i += THREADS<V>) cnt[i] = 0;
    float bias[V];
    u32 bit[V];
    bool bad = false;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        bias[i] = g.bias && i * 32 + lane < g.n ? g.bias[i * 32 + lane] : 0.0f;
        bad |= !(bias[i] == bias[i]);
    }
    group_bits<V>(g, lane, bit);
    const int64_t a = blockIdx.x * g.chunk_rows, b = a + g.chunk_rows < g.rows ? a + g.chunk_rows : g.rows;
    for (int64_t row = a + warp; row < b; row += WARPS)
        route_row<V>(g, row, lane, bias, bit, bad, reinterpret_cast<Few*>(smem + at.few) + warp * 32, smem + at.buf + 8 * g.n * warp);
    __syncthreads();
    number_choices(g, a * g.k, b * g.k, cnt, total);
    if (!FEW) {
        for (int e = threadIdx.x; e < g.n; e += THREADS<V>) g.counts[(int64_t)blockIdx.x * g.n + e] = total[e];
    } else {
        if (warp == 0) scan_counts(total, first, g.n, lane);
        __syncthreads();
        for (int e = threadIdx.x; e <= g.n; e += THREADS<V>) g.offsets[e] = first[e];
        for (int i = threadIdx.x; i < (int)g.rows * g.k; i += THREADS<V>) {
            const int e = g.experts[i];
            if (e >= 0) g.place[i] += first[e];
        }
    }
}

// Adds the counts of the experts before, and of the blocks before.
constexpr int PLACE_THREADS = 1024;
__global__ void __launch_bounds__(PLACE_THREADS, 1) place_kernel(const RouteArgs g) {
    __shared__ int total[MAX_EXPERTS], first[MAX_EXPERTS + 1], before[MAX_EXPERTS];
    for (int e = threadIdx.x; e < g.n; e += PLACE_THREADS) total[e] = before[e] = 0;
    __syncthreads();
    first_is_done();
    const int parts = PLACE_THREADS / g.n;               // at least 1: n <= 1024
    const int part = threadIdx.x / g.n, mine = threadIdx.x % g.n;
    const int64_t a = blockIdx.x * g.chunk_rows * g.k, all = g.rows * g.k;
    const int64_t b = a + g.chunk_rows * g.k < all ? a + g.chunk_rows * g.k : all;
    if (part < parts) {
        int sum = 0, early = 0;
#pragma unroll 16
        for (int c = part; c < g.chunks; c += parts) {
            const int v = __ldcg(&g.counts[(int64_t)c * g.n + mine]);
            sum += v;
            early += c < (int)blockIdx.x ? v : 0;
        }
        atomicAdd(&total[mine], sum);
        atomicAdd(&before[mine], early);
    }
    __syncthreads();
    if (threadIdx.x < 32) scan_counts(total, first, g.n, threadIdx.x);
    __syncthreads();
    if (blockIdx.x == 0)
        for (int e = threadIdx.x; e <= g.n; e += PLACE_THREADS) g.offsets[e] = first[e];
    for (int64_t i = a + threadIdx.x; i < b; i += PLACE_THREADS) {
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

template <int V> int launch_route(RouteArgs& g, int dev, cudaStream_t st) {
    const int bytes = Layout(g.n, THREADS<V> / 32, g.groups > 1).bytes;
    if (g.rows <= SMALL_ROWS) {
        if (int rc = more_smem<route_kernel<V, true>>(bytes, dev)) return rc;
        g.chunk_rows = g.rows;
        route_kernel<V, true><<<1, THREADS<V>, bytes, st>>>(g);
        return launched("route");
    }
    if (int rc = more_smem<route_kernel<V, false>>(bytes, dev)) return rc;
    route_kernel<V, false><<<g.chunks, THREADS<V>, bytes, st>>>(g);
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
    return chunks_of(rows, sms) * experts * 4;
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
    g.dtype = dtype;
    g.sigmoid = score == BAFE_CUDA_SCORE_SIGMOID;
    g.renorm = renormalize != 0;
    g.scale = fscale;
    if (rows > SMALL_ROWS) {
        const int64_t chunks = chunks_of(rows, sms);
        if (!workspace || workspace_bytes < chunks * n * 4 || !element_aligned(4, {workspace}))
            return fail(8, "route: workspace too small or unaligned (see bafe_cuda_route_workspace)");
        g.counts = static_cast<int*>(workspace);
        g.chunk_rows = (rows + chunks - 1) / chunks;
        g.chunks = (int)((rows + g.chunk_rows - 1) / g.chunk_rows);
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return with_slots(g.n, [&](auto v) { return launch_route<decltype(v)::value>(g, dev, st); });
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
