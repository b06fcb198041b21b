// rms_norm.cu -- root-mean-square norm with the residual's addition, its
// e4m3 form with one scale per row, and its gradient.
//
//   h = round(x + residual)             (rounded to the stored type: what a
//                                        later layer reads is what is normed)
//   r = 1 / sqrt(mean(h^2) + eps)
//   y = h * r * weight
// e4m3 form: scale = max|y| / 448, q = round_e4m3(y / scale).
// Gradient, with g = dy * weight:
//   dx = r * g - h * r^3 * mean(g * h)  (+ dh, the gradient that reaches h
//                                        past the norm)
//   dweight = sum over rows of dy * h * r
//
// Everything between the loads and the stores is in 32 bits; each output is
// rounded once.
//
// Bound by memory: a forward element costs 2-8 bytes and about 6
// operations.  Each row is read once and kept in registers between the sum
// of squares and the scaling (rows of up to 32 x 1024 elements; longer ones
// are read a second time, from L2 where they fit).  The e4m3 form needs the
// row's largest |y| as well: max|h * weight| is taken in the same pass and
// scaled by r afterwards, so both statistics cost one block reduction.
#include "common.cuh"

namespace bafe_cuda {
namespace lm {
namespace {

constexpr float E4M3_MAX = 448.0f;
// Smallest scale of a row that is not zero: its reciprocal stays finite.
constexpr float MIN_SCALE = 7.888609052210118e-31f;   // 2^-100

struct NormArgs {
    const void* x;
    const void* res;       // null: no residual
    const void* w;
    void* y;
    float* scale;          // e4m3 form
    void* h;               // residual sum, with res
    int64_t x_ld, res_ld, y_ld, h_ld;
    int64_t rows, width;
    float eps, inv_width;
};

// Sums `a` and takes the NaN-keeping maximum of `b` over the `warps` warps
// of a row; every thread gets both.  `buf` alternates between rows, so one
// barrier per row is enough.
template <bool WITH_MAX>
__device__ __forceinline__ void row_reduce(float& a, float& b, int warps, float2* buf) {
    a = warp_sum(a);
    if (WITH_MAX) b = warp_max_nan(b);
    if (warps == 1) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) buf[warp] = make_float2(a, b);
    __syncthreads();
    const float2 v = lane < warps ? buf[lane] : make_float2(0.0f, 0.0f);
    a = warp_sum(v.x);
    if (WITH_MAX) b = warp_max_nan(v.y);
}

// Sums of two values over a row's warps.
__device__ __forceinline__ void row_sums(float& a, float& b, int warps, float2* buf) {
    a = warp_sum(a);
    b = warp_sum(b);
    if (warps == 1) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) buf[warp] = make_float2(a, b);
    __syncthreads();
    const float2 v = lane < warps ? buf[lane] : make_float2(0.0f, 0.0f);
    a = warp_sum(v.x);
    b = warp_sum(v.y);
}

// The scale of a row whose largest |y| is `top`: 1 for a zero row and for
// one that holds a NaN (its elements carry the NaN).
__device__ __forceinline__ float row_scale(float top) {
    if (!(top > 0.0f)) return 1.0f;
    return fmaxf(top * (1.0f / E4M3_MAX), MIN_SCALE);
}

__device__ __forceinline__ unsigned char to_e4m3(float v) {
    return (unsigned char)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
}

// h of one vector: x, or the stored sum of x and the residual.
template <class T, int VE>
__device__ __forceinline__ Vec<T, VE> add_residual(const Vec<T, VE>& x, const Vec<T, VE>& r) {
    Vec<T, VE> h;
#pragma unroll
    for (int e = 0; e < VE; ++e) h.v[e] = from_f32<T>(to_f32(x.v[e]) + to_f32(r.v[e]));
    return h;
}

// Rows of up to blockDim.x (per row) * NV * VE elements, in registers.
// blockDim = (threads per row, rows per block): several rows share a block
// only when a row is one warp.
template <class T, class W, bool OUT8, int VE, int NV>
__global__ void __launch_bounds__(1024) rms_norm_kernel(const NormArgs g) {
    __shared__ float2 red[2][32];
    const int tpr = blockDim.x, warps = tpr >> 5;
    const T* xs = static_cast<const T*>(g.x);         // y or residual_out may be x
    const W* __restrict__ ws = static_cast<const W*>(g.w);
    int flip = 0;
    for (int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; row < g.rows;
         row += (int64_t)gridDim.x * blockDim.y, flip ^= 1) {
        const T* xr = xs + row * g.x_ld;
        Vec<T, VE> h[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t c = ((int64_t)j * tpr + threadIdx.x) * VE;
            if (c < g.width) h[j] = load_vec<T, VE>(xr + c);
        }
        if (g.res) {
            const T* rr = static_cast<const T*>(g.res) + row * g.res_ld;
            T* hr = static_cast<T*>(g.h) + row * g.h_ld;
            Vec<T, VE> r[NV];
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int64_t c = ((int64_t)j * tpr + threadIdx.x) * VE;
                if (c < g.width) r[j] = load_vec<T, VE>(rr + c);
            }
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int64_t c = ((int64_t)j * tpr + threadIdx.x) * VE;
                if (c < g.width) {
                    h[j] = add_residual<T, VE>(h[j], r[j]);
                    store_vec<T, VE>(hr + c, h[j]);
                }
            }
        }
        float sum = 0.0f, top = 0.0f;
        Vec<W, VE> w[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t c = ((int64_t)j * tpr + threadIdx.x) * VE;
            if (c < g.width) w[j] = load_vec<W, VE>(ws + c);
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t c = ((int64_t)j * tpr + threadIdx.x) * VE;
            if (c < g.width) {
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    const float v = to_f32(h[j].v[e]);
                    sum += v * v;
                    if (OUT8) top = max_nan(top, fabsf(v * to_f32(w[j].v[e])));
                }
            }
        }
        row_reduce<OUT8>(sum, top, warps, red[flip]);
        const float r = rsqrtf(sum * g.inv_width + g.eps);
        if constexpr (OUT8) {
            const float s = row_scale(top * r);
            const float f = r * (1.0f / s);
            unsigned char* yr = static_cast<unsigned char*>(g.y) + row * g.y_ld;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int64_t c = ((int64_t)j * tpr + threadIdx.x) * VE;
                if (c < g.width) {
                    Vec<unsigned char, VE> q;
#pragma unroll
                    for (int e = 0; e < VE; ++e) q.v[e] = to_e4m3(to_f32(h[j].v[e]) * to_f32(w[j].v[e]) * f);
                    store_vec<unsigned char, VE>(yr + c, q);
                }
            }
            if (threadIdx.x == 0) g.scale[row] = s;
        } else {
            T* yr = static_cast<T*>(g.y) + row * g.y_ld;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int64_t c = ((int64_t)j * tpr + threadIdx.x) * VE;
                if (c < g.width) {
                    Vec<T, VE> y;
#pragma unroll
                    for (int e = 0; e < VE; ++e) y.v[e] = from_f32<T>(to_f32(h[j].v[e]) * r * to_f32(w[j].v[e]));
                    store_vec<T, VE>(yr + c, y);
                }
            }
        }
    }
}

// Rows too long for registers: the same in two passes over the row.  The
// second reads h (or x) again; each thread reads only elements that it wrote
// itself, so no barrier beyond the reduction's is needed.
template <class T, class W, bool OUT8, int VE>
__global__ void __launch_bounds__(1024) rms_norm_long_kernel(const NormArgs g) {
    __shared__ float2 red[2][32];
    const W* __restrict__ ws = static_cast<const W*>(g.w);
    int flip = 0;
    for (int64_t row = blockIdx.x; row < g.rows; row += gridDim.x, flip ^= 1) {
        const T* xr = static_cast<const T*>(g.x) + row * g.x_ld;
        const T* rr = static_cast<const T*>(g.res) + (g.res ? row * g.res_ld : 0);
        T* hr = static_cast<T*>(g.h) + (g.res ? row * g.h_ld : 0);
        float sum = 0.0f, top = 0.0f;
        for (int64_t c = (int64_t)threadIdx.x * VE; c < g.width; c += (int64_t)blockDim.x * VE) {
            Vec<T, VE> h = load_vec<T, VE>(xr + c);
            if (g.res) {
                h = add_residual<T, VE>(h, load_vec<T, VE>(rr + c));
                store_vec<T, VE>(hr + c, h);
            }
            const Vec<W, VE> w = load_vec<W, VE>(ws + c);
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const float v = to_f32(h.v[e]);
                sum += v * v;
                if (OUT8) top = max_nan(top, fabsf(v * to_f32(w.v[e])));
            }
        }
        row_reduce<OUT8>(sum, top, blockDim.x >> 5, red[flip]);
        const float r = rsqrtf(sum * g.inv_width + g.eps);
        const float s = OUT8 ? row_scale(top * r) : 1.0f;
        const float f = OUT8 ? r * (1.0f / s) : r;
        const T* src = g.res ? hr : xr;
        for (int64_t c = (int64_t)threadIdx.x * VE; c < g.width; c += (int64_t)blockDim.x * VE) {
            const Vec<T, VE> h = load_vec<T, VE>(src + c);
            const Vec<W, VE> w = load_vec<W, VE>(ws + c);
            if constexpr (OUT8) {
                Vec<unsigned char, VE> q;
#pragma unroll
                for (int e = 0; e < VE; ++e) q.v[e] = to_e4m3(to_f32(h.v[e]) * to_f32(w.v[e]) * f);
                store_vec<unsigned char, VE>(static_cast<unsigned char*>(g.y) + row * g.y_ld + c, q);
            } else {
                Vec<T, VE> y;
#pragma unroll
                for (int e = 0; e < VE; ++e) y.v[e] = from_f32<T>(to_f32(h.v[e]) * f * to_f32(w.v[e]));
                store_vec<T, VE>(static_cast<T*>(g.y) + row * g.y_ld + c, y);
            }
        }
        if (OUT8 && threadIdx.x == 0) g.scale[row] = s;
    }
}

// --------------------------------------------------------------- gradient --

struct NormGradArgs {
    const void* dy;
    const void* h;
    const void* w;
    const void* dh;        // null: none
    void* dx;
    float* part;           // [slots][width]: one partial sum of dweight per slot
    int64_t dy_ld, h_ld, dh_ld, dx_ld;
    int64_t rows, width;
    float eps, inv_width;
};

// Slot (block, row of the block) walks rows slot, slot + slots, ...; its
// share of dweight stays in registers over all of them and is written once.
// Partials are summed in slot order by norm_grad_weight_kernel: no atomics,
// the same bits every run.
template <class T, class W, int VE, int NV>
__global__ void __launch_bounds__(1024) rms_norm_grad_kernel(const NormGradArgs g) {
    __shared__ float2 red[2][32];
    const int tpr = blockDim.x, warps = tpr >> 5;
    const W* __restrict__ ws = static_cast<const W*>(g.w);
    const int64_t slot = (int64_t)blockIdx.x * blockDim.y + threadIdx.y, slots = (int64_t)gridDim.x * blockDim.y;
    float acc[NV * VE];
    Vec<W, VE> w[NV];
#pragma unroll
    for (int i = 0; i < NV * VE; ++i) acc[i] = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int64_t c = ((int64_t)j * tpr + threadIdx.x) * VE;
        if (c < g.width) w[j] = load_vec<W, VE>(ws + c);
    }
    int flip = 0;
    for (int64_t row = slot; row < g.rows; row += slots, flip ^= 1) {
        const T* dyr = static_cast<const T*>(g.dy) + row * g.dy_ld;
        const T* hr = static_cast<const T*>(g.h) + row * g.h_ld;
        Vec<T, VE> dy[NV], h[NV], dh[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t c = ((int64_t)j * tpr + threadIdx.x) * VE;
            if (c < g.width) {
                dy[j] = load_vec<T, VE>(dyr + c);
                h[j] = load_vec<T, VE>(hr + c);
            }
        }
        if (g.dh) {
            const T* dhr = static_cast<const T*>(g.dh) + row * g.dh_ld;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int64_t c = ((int64_t)j * tpr + threadIdx.x) * VE;
                if (c < g.width) dh[j] = load_vec<T, VE>(dhr + c);
            }
        }
        float sq = 0.0f, gh = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t c = ((int64_t)j * tpr + threadIdx.x) * VE;
            if (c < g.width) {
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    const float v = to_f32(h[j].v[e]);
                    sq += v * v;
                    gh += to_f32(dy[j].v[e]) * to_f32(w[j].v[e]) * v;
                }
            }
        }
        row_sums(sq, gh, warps, red[flip]);
        const float r = rsqrtf(sq * g.inv_width + g.eps);
        const float k = r * r * (gh * g.inv_width);
        T* dxr = static_cast<T*>(g.dx) + row * g.dx_ld;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t c = ((int64_t)j * tpr + threadIdx.x) * VE;
            if (c < g.width) {
                Vec<T, VE> o;
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    const float v = to_f32(h[j].v[e]), d = to_f32(dy[j].v[e]);
                    float dx = r * (d * to_f32(w[j].v[e]) - v * k);
                    if (g.dh) dx += to_f32(dh[j].v[e]);
                    o.v[e] = from_f32<T>(dx);
                    acc[j * VE + e] += d * (v * r);
                }
                store_vec<T, VE>(dxr + c, o);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int64_t c = ((int64_t)j * tpr + threadIdx.x) * VE;
        if (c < g.width) {
#pragma unroll
            for (int e = 0; e < VE; ++e) g.part[slot * g.width + c + e] = acc[j * VE + e];
        }
    }
}

// Rows too long for registers: two passes, the partial sums of dweight in
// the slot's own workspace row (each thread adds to its own elements only).
template <class T, class W, int VE>
__global__ void __launch_bounds__(1024) rms_norm_grad_long_kernel(const NormGradArgs g) {
    __shared__ float2 red[2][32];
    const W* __restrict__ ws = static_cast<const W*>(g.w);
    float* part = g.part + (int64_t)blockIdx.x * g.width;
    bool first = true;
    int flip = 0;
    for (int64_t row = blockIdx.x; row < g.rows; row += gridDim.x, flip ^= 1) {
        const T* dyr = static_cast<const T*>(g.dy) + row * g.dy_ld;
        const T* hr = static_cast<const T*>(g.h) + row * g.h_ld;
        const T* dhr = static_cast<const T*>(g.dh) + (g.dh ? row * g.dh_ld : 0);
        T* dxr = static_cast<T*>(g.dx) + row * g.dx_ld;
        float sq = 0.0f, gh = 0.0f;
        for (int64_t c = (int64_t)threadIdx.x * VE; c < g.width; c += (int64_t)blockDim.x * VE) {
            const Vec<T, VE> dy = load_vec<T, VE>(dyr + c), h = load_vec<T, VE>(hr + c);
            const Vec<W, VE> w = load_vec<W, VE>(ws + c);
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const float v = to_f32(h.v[e]);
                sq += v * v;
                gh += to_f32(dy.v[e]) * to_f32(w.v[e]) * v;
            }
        }
        row_sums(sq, gh, blockDim.x >> 5, red[flip]);
        const float r = rsqrtf(sq * g.inv_width + g.eps);
        const float k = r * r * (gh * g.inv_width);
        for (int64_t c = (int64_t)threadIdx.x * VE; c < g.width; c += (int64_t)blockDim.x * VE) {
            const Vec<T, VE> dy = load_vec<T, VE>(dyr + c), h = load_vec<T, VE>(hr + c);
            const Vec<W, VE> w = load_vec<W, VE>(ws + c);
            Vec<T, VE> dh;
            if (g.dh) dh = load_vec<T, VE>(dhr + c);
            Vec<T, VE> o;
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const float v = to_f32(h.v[e]), d = to_f32(dy.v[e]);
                float dx = r * (d * to_f32(w.v[e]) - v * k);
                if (g.dh) dx += to_f32(dh.v[e]);
                o.v[e] = from_f32<T>(dx);
                part[c + e] = (first ? 0.0f : part[c + e]) + d * (v * r);
            }
            store_vec<T, VE>(dxr + c, o);
        }
        first = false;
    }
}

// dweight = the slots' partial sums, added in a fixed order: 8 groups of
// slots per column, then the groups.
template <class W>
__global__ void __launch_bounds__(256) norm_grad_weight_kernel(const float* __restrict__ part, W* __restrict__ dw,
                                                               int slots, int64_t width) {
    __shared__ float s[8][33];
    const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
    float a = 0.0f;
    if (c < width)
        for (int i = threadIdx.y; i < slots; i += 8) a += part[(int64_t)i * width + c];
    s[threadIdx.y][threadIdx.x] = a;
    __syncthreads();
    if (threadIdx.y == 0 && c < width) {
        float t = s[0][threadIdx.x];
#pragma unroll
        for (int i = 1; i < 8; ++i) t += s[i][threadIdx.x];
        dw[c] = from_f32<W>(t);
    }
}

// -------------------------------------------------------------- dispatch --

// Threads and vectors per thread of a row of `n` vectors: a warp for the
// shortest rows, then wider blocks, so that each thread keeps `want` vectors
// until the block is full.
struct RowShape { int tpr, nv, rows_per_block; };
RowShape row_shape(int64_t n, int want, int most) {
    int nv = want;
    while (nv > 1 && n <= (int64_t)32 * (nv / 2)) nv /= 2;
    int64_t t = (n + nv - 1) / nv;
    while (t > 1024 && nv < most) {
        nv *= 2;
        t = (n + nv - 1) / nv;
    }
    if (t > 1024) return {0, 0, 0};                   // too long for registers
    const int tpr = (int)((t + 31) / 32 * 32);
    return {tpr, nv, tpr == 32 ? 4 : 1};
}

template <class K>
int blocks_per_sm(K kernel, int threads) {
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, 0) != cudaSuccess || n < 1) {
        cudaGetLastError();
        n = 1;
    }
    return n;
}

template <class T, class W, bool OUT8, int VE, int NV>
int launch_norm(const NormArgs& a, const RowShape& s, int sms, cudaStream_t st) {
    auto k = rms_norm_kernel<T, W, OUT8, VE, NV>;
    const int64_t want = (a.rows + s.rows_per_block - 1) / s.rows_per_block;
    const int64_t room = (int64_t)sms * blocks_per_sm(k, s.tpr * s.rows_per_block);
    k<<<(unsigned)(want < room ? want : room), dim3(s.tpr, s.rows_per_block), 0, st>>>(a);
    return launched("rms_norm");
}

template <class T, class W, bool OUT8>
int norm_typed(const NormArgs& a, bool vec, int sms, cudaStream_t st) {
    constexpr int VE = 16 / sizeof(T);
    if (vec) {
        const RowShape s = row_shape((a.width + VE - 1) / VE, 2, 4);
        switch (s.nv) {
            case 1: return launch_norm<T, W, OUT8, VE, 1>(a, s, sms, st);
            case 2: return launch_norm<T, W, OUT8, VE, 2>(a, s, sms, st);
            case 4: return launch_norm<T, W, OUT8, VE, 4>(a, s, sms, st);
        }
        rms_norm_long_kernel<T, W, OUT8, VE><<<(unsigned)(a.rows < 2 * sms ? a.rows : 2 * sms), 1024, 0, st>>>(a);
        return launched("rms_norm");
    }
    const RowShape s = row_shape(a.width, 8, 16);
    switch (s.nv) {
        case 1: return launch_norm<T, W, OUT8, 1, 1>(a, s, sms, st);
        case 2: return launch_norm<T, W, OUT8, 1, 2>(a, s, sms, st);
        case 4: return launch_norm<T, W, OUT8, 1, 4>(a, s, sms, st);
        case 8: return launch_norm<T, W, OUT8, 1, 8>(a, s, sms, st);
        case 16: return launch_norm<T, W, OUT8, 1, 16>(a, s, sms, st);
    }
    rms_norm_long_kernel<T, W, OUT8, 1><<<(unsigned)(a.rows < 2 * sms ? a.rows : 2 * sms), 1024, 0, st>>>(a);
    return launched("rms_norm");
}

template <class T, class W>
int norm_out(const NormArgs& a, bool out8, bool vec, int sms, cudaStream_t st) {
    return out8 ? norm_typed<T, W, true>(a, vec, sms, st) : norm_typed<T, W, false>(a, vec, sms, st);
}

// The gradient's shape: its slots are the workspace's rows, so the size
// query and the launch both come here.
struct GradShape { RowShape s; int grid; bool vec; };
constexpr int GRAD_BLOCKS_PER_SM = 2;
GradShape grad_shape(int64_t rows, int64_t width, int esize, bool vec, int sms) {
    const int ve = vec ? 16 / esize : 1;
    GradShape g;
    g.vec = vec;
    g.s = vec ? row_shape((width + ve - 1) / ve, 2, 4) : row_shape(width, 8, 16);
    const int rpb = g.s.nv ? g.s.rows_per_block : 1;
    const int tpb = g.s.nv ? g.s.tpr * rpb : 1024;
    // enough blocks to keep 2048 threads on each SM, two at least
    int per_sm = 2048 / tpb;
    if (per_sm < GRAD_BLOCKS_PER_SM) per_sm = GRAD_BLOCKS_PER_SM;
    if (per_sm > 8) per_sm = 8;
    const int64_t want = (rows + rpb - 1) / rpb, room = (int64_t)sms * per_sm;
    g.grid = (int)(want < room ? want : room);
    return g;
}

template <class T, class W>
int grad_typed(const NormGradArgs& a, const GradShape& g, void* dw, cudaStream_t st) {
    constexpr int VE = 16 / sizeof(T);
    const dim3 block(g.s.nv ? g.s.tpr : 1024, g.s.nv ? g.s.rows_per_block : 1);
    const unsigned grid = (unsigned)g.grid;
    if (g.vec) {
        switch (g.s.nv) {
            case 1: rms_norm_grad_kernel<T, W, VE, 1><<<grid, block, 0, st>>>(a); break;
            case 2: rms_norm_grad_kernel<T, W, VE, 2><<<grid, block, 0, st>>>(a); break;
            case 4: rms_norm_grad_kernel<T, W, VE, 4><<<grid, block, 0, st>>>(a); break;
            default: rms_norm_grad_long_kernel<T, W, VE><<<grid, block, 0, st>>>(a);
        }
    } else {
        switch (g.s.nv) {
            case 1: rms_norm_grad_kernel<T, W, 1, 1><<<grid, block, 0, st>>>(a); break;
            case 2: rms_norm_grad_kernel<T, W, 1, 2><<<grid, block, 0, st>>>(a); break;
            case 4: rms_norm_grad_kernel<T, W, 1, 4><<<grid, block, 0, st>>>(a); break;
            case 8: rms_norm_grad_kernel<T, W, 1, 8><<<grid, block, 0, st>>>(a); break;
            case 16: rms_norm_grad_kernel<T, W, 1, 16><<<grid, block, 0, st>>>(a); break;
            default: rms_norm_grad_long_kernel<T, W, 1><<<grid, block, 0, st>>>(a);
        }
    }
    if (int rc = launched("rms_norm_grad")) return rc;
    norm_grad_weight_kernel<W><<<(unsigned)((a.width + 31) / 32), dim3(32, 8), 0, st>>>(
        a.part, static_cast<W*>(dw), (int)(grid * block.y), a.width);
    return launched("rms_norm_grad weight sum");
}

int esize_of(int dtype) { return dtype == BAFE_DTYPE_F32 ? 4 : 2; }

int check_sizes(int64_t rows, int64_t width, int dtype, int wdtype, double eps) {
    if (rows < 0 || width < 1 || width > (int64_t(1) << 30)) return fail(8, "rms_norm: rows must be >= 0 and width in [1, 2^30]");
    if (!is_float_type(dtype)) return fail(8, "rms_norm: the rows must be f32, f16 or bf16");
    if (wdtype != dtype && wdtype != BAFE_DTYPE_F32) return fail(8, "rms_norm: the weight must have the rows' type or f32");
    if (!(eps >= 0.0)) return fail(8, "rms_norm: eps must be >= 0");
    return 0;
}

// Sixteen-byte loads and stores of every row of a tensor.
bool rows_vec(const void* p, int64_t ld, int esize) { return !p || (aligned16(p) && (ld * esize) % 16 == 0); }

}  // namespace

int current_device(int& dev, int& sms) {
    static int cached[64] = {0};
    if (cudaGetDevice(&dev) != cudaSuccess) {
        cudaGetLastError();
        return fail(4, "no CUDA device available");
    }
    if (dev < 0 || dev >= 64) return fail(4, "device ordinal out of range");
    if (!cached[dev]) {
        int n = 0;
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) {
            cudaGetLastError();
            return fail(4, "cannot read the device's SM count");
        }
        cached[dev] = n;
    }
    sms = cached[dev];
    return 0;
}

}  // namespace lm
}  // namespace bafe_cuda

#define BAFE_API extern "C" __attribute__((visibility("default")))

using namespace bafe_cuda;
using namespace bafe_cuda::lm;

BAFE_API int bafe_cuda_rms_norm(const void* x, int64_t x_ld, const void* residual, int64_t residual_ld,
                                const void* weight, void* y, int64_t y_ld, float* y_scale, void* residual_out,
                                int64_t residual_out_ld, int64_t rows, int64_t width, int dtype, int weight_dtype,
                                int y_dtype, double eps, void* stream) {
    if (int rc = check_sizes(rows, width, dtype, weight_dtype, eps)) return rc;
    const bool out8 = y_dtype == DTYPE_E4M3;
    if (!out8 && y_dtype != dtype) return fail(8, "rms_norm: y must have the rows' type or e4m3");
    if (rows == 0) return 0;
    if (!x || !weight || !y) return fail(8, "rms_norm: null operand");
    if (out8 && !y_scale) return fail(8, "rms_norm: e4m3 output needs its scales");
    if ((residual == nullptr) != (residual_out == nullptr))
        return fail(8, "rms_norm: residual and residual_out go together");
    if (x_ld < width || y_ld < width || (residual && (residual_ld < width || residual_out_ld < width)))
        return fail(8, "rms_norm: row strides must be at least the width");
    int dev = 0, sms = 0;
    if (int rc = current_device(dev, sms)) return rc;
    NormArgs a;
    a.x = x; a.res = residual; a.w = weight; a.y = y; a.scale = y_scale; a.h = residual_out;
    a.x_ld = x_ld; a.res_ld = residual_ld; a.y_ld = y_ld; a.h_ld = residual_out_ld;
    a.rows = rows; a.width = width;
    a.eps = (float)eps;
    a.inv_width = (float)(1.0 / (double)width);
    const int es = esize_of(dtype), ve = 16 / es;
    // q's vector is ve bytes wide
    const bool y_vec = out8 ? (reinterpret_cast<uintptr_t>(y) % ve == 0 && y_ld % ve == 0) : rows_vec(y, y_ld, es);
    const bool vec = width % ve == 0 && rows_vec(x, x_ld, es) && rows_vec(residual, residual_ld, es) &&
                     rows_vec(residual_out, residual_out_ld, es) && y_vec && aligned16(weight);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool wf = weight_dtype == BAFE_DTYPE_F32;
    if (dtype == BAFE_DTYPE_F32) return norm_out<float, float>(a, out8, vec, sms, st);
    if (dtype == BAFE_DTYPE_F16)
        return wf ? norm_out<__half, float>(a, out8, vec, sms, st) : norm_out<__half, __half>(a, out8, vec, sms, st);
    return wf ? norm_out<__nv_bfloat16, float>(a, out8, vec, sms, st)
              : norm_out<__nv_bfloat16, __nv_bfloat16>(a, out8, vec, sms, st);
}

BAFE_API int64_t bafe_cuda_rms_norm_grad_workspace(int64_t rows, int64_t width, int dtype) {
    if (check_sizes(rows, width, dtype, dtype, 0.0)) return -1;
    int dev = 0, sms = 0;
    if (current_device(dev, sms)) return -1;
    // whichever of the two forms a call takes
    int64_t most = 1;
    for (int vec = 0; vec < 2; ++vec) {
        const GradShape g = grad_shape(rows, width, esize_of(dtype), vec != 0, sms);
        const int64_t slots = (int64_t)g.grid * (g.s.nv ? g.s.rows_per_block : 1);
        if (slots > most) most = slots;
    }
    return most * width * 4;
}

BAFE_API int bafe_cuda_rms_norm_grad(const void* dy, int64_t dy_ld, const void* h, int64_t h_ld, const void* weight,
                                     const void* dh, int64_t dh_ld, void* dx, int64_t dx_ld, void* dweight,
                                     int64_t rows, int64_t width, int dtype, int weight_dtype, double eps,
                                     void* workspace, int64_t workspace_bytes, void* stream) {
    if (int rc = check_sizes(rows, width, dtype, weight_dtype, eps)) return rc;
    if (!weight || !dweight) return fail(8, "rms_norm_grad: null operand");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (rows == 0) {
        cudaError_t e = cudaMemsetAsync(dweight, 0, (size_t)width * esize_of(weight_dtype), st);
        return e == cudaSuccess ? 0 : (cudaGetLastError(), fail(7, "rms_norm_grad: cudaMemsetAsync"));
    }
    if (!dy || !h || !dx) return fail(8, "rms_norm_grad: null operand");
    if (dy_ld < width || h_ld < width || dx_ld < width || (dh && dh_ld < width))
        return fail(8, "rms_norm_grad: row strides must be at least the width");
    int dev = 0, sms = 0;
    if (int rc = current_device(dev, sms)) return rc;
    const int es = esize_of(dtype), ve = 16 / es;
    const bool vec = width % ve == 0 && rows_vec(dy, dy_ld, es) && rows_vec(h, h_ld, es) && rows_vec(dh, dh_ld, es) &&
                     rows_vec(dx, dx_ld, es) && aligned16(weight);
    const GradShape g = grad_shape(rows, width, es, vec, sms);
    const int64_t need = (int64_t)g.grid * (g.s.nv ? g.s.rows_per_block : 1) * width * 4;
    if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 3u))
        return fail(8, "rms_norm_grad: workspace too small (see bafe_cuda_rms_norm_grad_workspace)");
    NormGradArgs a;
    a.dy = dy; a.h = h; a.w = weight; a.dh = dh; a.dx = dx; a.part = static_cast<float*>(workspace);
    a.dy_ld = dy_ld; a.h_ld = h_ld; a.dh_ld = dh_ld; a.dx_ld = dx_ld;
    a.rows = rows; a.width = width;
    a.eps = (float)eps;
    a.inv_width = (float)(1.0 / (double)width);
    const bool wf = weight_dtype == BAFE_DTYPE_F32;
    if (dtype == BAFE_DTYPE_F32) return grad_typed<float, float>(a, g, dweight, st);
    if (dtype == BAFE_DTYPE_F16)
        return wf ? grad_typed<__half, float>(a, g, dweight, st) : grad_typed<__half, __half>(a, g, dweight, st);
    return wf ? grad_typed<__nv_bfloat16, float>(a, g, dweight, st)
              : grad_typed<__nv_bfloat16, __nv_bfloat16>(a, g, dweight, st);
}
