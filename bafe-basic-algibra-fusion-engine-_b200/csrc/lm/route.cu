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
// A warp takes a row, expert i * 32 + lane in slot i of a lane's registers, and
// picks one expert a round: the lanes' largest in one warp reduction.  The
// order is the one of the scores in 64 bits: two f32 scores nearer to one
// another than their errors could be the other way round, so a row with such
// a pair among its k + 1 first (or its groups at the border) is chosen again
// in 64 bits.  (Without bias and groups the logits themselves have the
// scores' order, and nothing is computed for the choice.)
//
// The order by expert is a counting sort in two kernels: each block counts the
// choices of its rows per expert; the second kernel sums the counts of the
// blocks before it and gives every choice its place, warps and lanes in order.
// No atomics whose order matters: the same places every run.  Few rows take
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

// Shuts the experts of the groups that are not kept; buf: n values.  Returns
// whether the worst kept and the best other group differ by no more than
// `slack` (the errors of four scores).
template <class F, int V>
__device__ __forceinline__ bool keep_groups(const RouteArgs& g, F (&c)[V], F* buf, int lane, F slack) {
    const F shut = -INFINITY;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (i * 32 + lane < g.n) buf[i * 32 + lane] = c[i];
    __syncwarp();
    // lanes per group: a power of two
    const int shift = g.groups > 1 ? __clz(g.groups - 1) - 27 : 5;     // 32 >> ceil(log2(groups)) = 1 << shift
    const int per = 1 << shift, mine = lane >> shift;
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
    u32 stay = 0;
    {
        const u32 lanes = __ballot_sync(ALL, kept);
        // one bit a group
        for (int h = 0; h < g.groups; ++h) stay |= (lanes >> (h << shift) & 1u) << h;
    }
    const F in = -warp_max(kept ? -worth : shut), out = warp_max(mine < g.groups && !kept ? worth : shut);
    const u32 inverse = (u32)((0x100000000ull + g.group_size - 1) / (u32)g.group_size);   // exact for indices below 2^16
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int e = i * 32 + lane;
        const int h = g.group_size == 1 ? e : (int)__umulhi((u32)e, inverse);
        if (!(stay >> (h & 31) & 1u)) c[i] = shut;
    }
    return out > shut && in - out <= slack + F(0x1p-21) * (fabs(in) + fabs(out));
}

// Routes a row; lane j < k returns choice j.
template <int V>
__device__ __forceinline__ int route_row(const RouteArgs& g, int64_t row, int lane, const float (&bias)[V], void* buf) {
    float l[V], c[V];
    load_row<V>(g.logits, g.dtype, row * g.ld, g.n, lane, l);
    bool bad = false;
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        bad |= !(l[i] == l[i]);
        m = fmaxf(m, l[i]);
    }
    m = warp_max(m);
    bad |= !g.sigmoid && m == INFINITY;                  // a softmax of infinities has no value
    if (!(m > -INFINITY)) m = 0.0f;
    const bool scored = g.bias || g.groups > 1;          // else the logits have the scores' order
    float inv = 1.0f;                                    // of the softmax's sum
    if (!g.sigmoid && (scored || !g.renorm)) {
        float z = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            c[i] = expf(l[i] - m);
            z += c[i];
        }
        inv = 1.0f / fmaxf(lm::warp_sum(z), 1e-30f);
    }
    int e = -1;
    bool again = false;
    if (scored) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            c[i] = (g.sigmoid ? 1.0f / (1.0f + expf(-l[i])) : c[i] * inv) + bias[i];
            bad |= l[i] > -INFINITY && !(c[i] == c[i]);
            if (!(l[i] > -INFINITY)) c[i] = -INFINITY;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) c[i] = l[i];
    }
    if (__any_sync(ALL, bad)) {
        e = lane < g.k ? lane : -1;
        if (e >= 0) {
            g.weights[row * g.k + lane] = NAN;
            g.experts[row * g.k + lane] = e;
        }
        return e;
    }
    // Errors of the f32 scores.  Sigmoid: expf, the addition and the division
    // are off by an ulp or less each, 8 ulps (2^-21) are allowed.  Softmax: the
    // exponent's rounding counts up to |l - m| <= 88 half ulps (below that the
    // score is 0 or denormal), the sum's up to 36, 128 ulps (2^-17) are allowed.
    const float tell = g.sigmoid ? 0x1p-21f : 0x1p-17f;
    if (g.groups > 1) {
        again = keep_groups<float, V>(g, c, static_cast<float*>(buf), lane, tell * 4.0f * (g.sigmoid ? 1.0f : inv));
        if (!g.bias) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (c[i] > -INFINITY) c[i] = l[i];
        }
    }
    float best;
    choose<float, V>(c, g.bias ? g.k + 1 : g.k, lane, e, best);
    float mine = e >= 0 ? load_one(g.logits, g.dtype, row * g.ld + e) : 0.0f;
    if (g.bias) {
        const float b = e >= 0 ? g.bias[e] : 0.0f;
        const float s = g.sigmoid ? 1.0f / (1.0f + expf(-mine)) : expf(mine - m) * inv;
        const float off = tell * s + 0x1p-22f * fabsf(best) + 1e-37f;
        const float next = __shfl_down_sync(ALL, best, 1), off2 = __shfl_down_sync(ALL, off, 1);
        const float next_l = __shfl_down_sync(ALL, mine, 1), next_b = __shfl_down_sync(ALL, b, 1);
        const int next_e = __shfl_down_sync(ALL, e, 1);
        // equal logits and equal biases are equal in 64 bits too
        again |= lane < g.k && next_e >= 0 && best - next <= off + off2 && !(mine == next_l && b == next_b);
    }
    if (__any_sync(ALL, again)) {
        double d[V];
        if (g.sigmoid) {
#pragma unroll
            for (int i = 0; i < V; ++i) d[i] = 1.0 / (1.0 + exp(-(double)l[i]));
        } else {
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
        for (int i = 0; i < V; ++i) d[i] = l[i] > -INFINITY ? d[i] + (double)bias[i] : -INFINITY;
        if (g.groups > 1) keep_groups<double, V>(g, d, static_cast<double*>(buf), lane, 0.0);
        if (!g.bias) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (d[i] > -INFINITY) d[i] = l[i];
        }
        double unused;
        choose<double, V>(d, g.k, lane, e, unused);
        mine = e >= 0 ? load_one(g.logits, g.dtype, row * g.ld + e) : 0.0f;
    }
    if (lane >= g.k) e = -1;
    // Weights.  Renormalised ones are made relative to the largest chosen, so
    // that they hold where all scores are tiny.
    float w;
    if (g.renorm) {
        const float top = warp_max(e >= 0 ? mine : -INFINITY);
        const float num = e < 0 ? 0.0f
                          : g.sigmoid ? expf(fminf(mine, 0.0f) - fminf(top, 0.0f)) / (1.0f + expf(-fabsf(mine)))
                                      : expf(mine - top);
        w = num / lm::warp_sum(num);
    } else {
        w = g.sigmoid ? 1.0f / (1.0f + expf(-mine)) : expf(mine - m) * inv;
    }
    if (lane < g.k) {
        g.weights[row * g.k + lane] = e < 0 ? 0.0f : w * g.scale;
        g.experts[row * g.k + lane] = e;
    }
    return e;
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

// Places of entries [a, b) of experts: cnt is [warps][n], each warp a run of
// consecutive entries.
__device__ __forceinline__ void count_runs(const RouteArgs& g, int a, int b, int* cnt, int per_warp) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int i = threadIdx.x; i < (int)(blockDim.x >> 5) * g.n; i += blockDim.x) cnt[i] = 0;
    __syncthreads();
    int* mine = cnt + warp * g.n;
    for (int i = 0; i < per_warp; i += 32) {
        const int at = a + warp * per_warp + i + lane;
        const int e = at < b ? g.experts[at] : -1;
        const u32 same = __match_any_sync(ALL, e);
        if (e >= 0 && lane == __ffs(same) - 1) mine[e] += __popc(same);
        __syncwarp();
    }
    __syncthreads();
}
__device__ __forceinline__ void place_runs(const RouteArgs& g, int a, int b, int* cnt, const int* base, int per_warp) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    for (int e = threadIdx.x; e < g.n; e += blockDim.x) {
        int run = base[e];
        for (int w = 0; w < warps; ++w) {
            const int t = cnt[w * g.n + e];
            cnt[w * g.n + e] = run;
            run += t;
        }
    }
    __syncthreads();
    int* mine = cnt + warp * g.n;
    for (int i = 0; i < per_warp; i += 32) {
        const int at = a + warp * per_warp + i + lane;
        const int e = at < b ? g.experts[at] : -1;
        const u32 same = __match_any_sync(ALL, e);
        const int p = e >= 0 ? mine[e] + __popc(same & ((1u << lane) - 1u)) : -1;
        if (at < b) g.place[at] = p;
        __syncwarp();
        if (e >= 0 && lane == __ffs(same) - 1) mine[e] += __popc(same);
        __syncwarp();
    }
}
__device__ __forceinline__ int run_length(int entries) {
    const int warps = blockDim.x >> 5;
    return ((entries + warps - 1) / warps + 31) & ~31;
}

template <int V> constexpr int THREADS = V <= 8 ? 1024 : 512;          // 64 registers a thread hold 8 slots, not 16

// FEW: one block routes and sorts all rows.  Else each block routes
// chunk_rows rows and leaves its counts.
template <int V, bool FEW> __global__ void __launch_bounds__(THREADS<V>, 1) route_kernel(const RouteArgs g) {
    extern __shared__ __align__(16) unsigned char smem[];
    if (!FEW) second_may_start();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = THREADS<V> / 32;
    int* hist = reinterpret_cast<int*>(smem);            // [n + 1] and a pad
    void* buf = smem + (size_t)((g.n + 2) & ~1) * 4 + (size_t)warp * g.n * 8;
    if (!FEW) {
        for (int e = threadIdx.x; e < g.n; e += blockDim.x) hist[e] = 0;
        __syncthreads();
    }
    float bias[V];
#pragma unroll
    for (int i = 0; i < V; ++i) bias[i] = g.bias && i * 32 + lane < g.n ? g.bias[i * 32 + lane] : 0.0f;
    const int64_t a = blockIdx.x * g.chunk_rows, b = a + g.chunk_rows < g.rows ? a + g.chunk_rows : g.rows;
    for (int64_t row = a + warp; row < b; row += warps) {
        const int e = route_row<V>(g, row, lane, bias, buf);
        if (!FEW && e >= 0) atomicAdd(&hist[e], 1);
    }
    __syncthreads();
    if (!FEW) {
        for (int e = threadIdx.x; e < g.n; e += blockDim.x) g.counts[(int64_t)blockIdx.x * g.n + e] = hist[e];
    } else {
        int *first = hist, *tot = first + ((g.n + 2) & ~1), *cnt = tot + g.n;
        const int entries = (int)g.rows * g.k, per = run_length(entries);
        count_runs(g, 0, entries, cnt, per);
        for (int e = threadIdx.x; e < g.n; e += blockDim.x) {
            int t = 0;
            for (int w = 0; w < warps; ++w) t += cnt[w * g.n + e];
            tot[e] = t;
        }
        __syncthreads();
        if (warp == 0) scan_counts(tot, first, g.n, lane);
        __syncthreads();
        for (int e = threadIdx.x; e <= g.n; e += blockDim.x) g.offsets[e] = first[e];
        place_runs(g, 0, entries, cnt, first, per);
    }
}

constexpr int PLACE_THREADS = 1024;
__global__ void __launch_bounds__(PLACE_THREADS, 1) place_kernel(const RouteArgs g) {
    extern __shared__ __align__(16) unsigned char smem[];
    int* first = reinterpret_cast<int*>(smem);           // [n + 1] and a pad
    int *tot = first + ((g.n + 2) & ~1), *before = tot + g.n, *cnt = before + g.n;
    const int lane = threadIdx.x & 31;
    for (int e = threadIdx.x; e < 2 * g.n; e += blockDim.x) tot[e] = 0;
    __syncthreads();
    first_is_done();
    // counts of the blocks before this one, and of all
    const int parts = PLACE_THREADS / g.n;               // at least 1: n <= 1024
    const int part = threadIdx.x / g.n, e = threadIdx.x % g.n;
    if (part < parts) {
        int all = 0, mine = 0;
#pragma unroll 8
        for (int c = part; c < g.chunks; c += parts) {
            const int v = __ldcg(&g.counts[(int64_t)c * g.n + e]);
            all += v;
            mine += c < (int)blockIdx.x ? v : 0;
        }
        atomicAdd(&tot[e], all);
        atomicAdd(&before[e], mine);
    }
    const int64_t a = blockIdx.x * g.chunk_rows * g.k, end = g.rows * g.k;
    const int64_t b = a + g.chunk_rows * g.k < end ? a + g.chunk_rows * g.k : end;
    const int per = run_length((int)(b - a));
    count_runs(g, (int)a, (int)b, cnt, per);             // its barriers are behind the sums too
    if (threadIdx.x < 32) scan_counts(tot, first, g.n, lane);
    __syncthreads();
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i <= g.n; i += blockDim.x) g.offsets[i] = first[i];
    for (int i = threadIdx.x; i < g.n; i += blockDim.x) before[i] += first[i];
    __syncthreads();
    place_runs(g, (int)a, (int)b, cnt, before, per);
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
    const int warps = THREADS<V> / 32, head = ((g.n + 2) & ~1) * 4;
    const int bufs = g.groups > 1 ? warps * g.n * 8 : 0;
    if (g.rows <= SMALL_ROWS) {
        const int runs = g.n * 4 + warps * g.n * 4, bytes = head + (bufs > runs ? bufs : runs);
        if (int rc = more_smem<route_kernel<V, true>>(bytes, dev)) return rc;
        g.chunk_rows = g.rows;
        route_kernel<V, true><<<1, THREADS<V>, bytes, st>>>(g);
        return launched("route");
    }
    if (int rc = more_smem<route_kernel<V, false>>(head + bufs, dev)) return rc;
    route_kernel<V, false><<<g.chunks, THREADS<V>, head + bufs, st>>>(g);
    return launched("route");
}

// Launch of the places' kernel: as launch_second, with shared memory.
int launch_place(const RouteArgs& g, int dev, cudaStream_t st) {
    const int bytes = ((g.n + 2) & ~1) * 4 + 2 * g.n * 4 + PLACE_THREADS / 32 * g.n * 4;
    if (int rc = more_smem<place_kernel>(bytes, dev)) return rc;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = (unsigned)g.chunks;
    cfg.blockDim = PLACE_THREADS;
    cfg.dynamicSmemBytes = (size_t)bytes;
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, place_kernel, g);           // its error is read by launched
    return launched("route: places");
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
    const bool few = rows <= SMALL_ROWS;
    if (!few) {
        const int64_t chunks = chunks_of(rows, sms);
        if (!workspace || workspace_bytes < chunks * n * 4 || !element_aligned(4, {workspace}))
            return fail(8, "route: workspace too small or unaligned (see bafe_cuda_route_workspace)");
        g.counts = static_cast<int*>(workspace);
        g.chunk_rows = (rows + chunks - 1) / chunks;
        g.chunks = (int)((rows + g.chunk_rows - 1) / g.chunk_rows);
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (int rc = with_slots(g.n, [&](auto v) { return launch_route<decltype(v)::value>(g, dev, st); })) return rc;
    return few ? 0 : launch_place(g, dev, st);
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
