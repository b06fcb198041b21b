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
// of squares and the scaling.  The e4m3 form needs the row's largest |y| as
// well: max|h * weight| is taken in the same pass and scaled by r
// afterwards, so both statistics cost one block reduction.
//
// A block walks rows with a fixed step.  Its next rows travel into shared
// memory with 16-byte asynchronous copies (each thread copies what it will
// read itself, so no barrier guards them) while the current row waits at
// its reduction: the bytes in flight do not depend on registers or on how
// many blocks happen to be loading.
//
// Rows of any width use 16-byte accesses as long as all operands' rows start
// at the same offset from a 16-byte boundary (contiguous tensors of an odd
// width do): the step is a multiple of the elements of 16 bytes, so a
// block's rows all start at one offset, its vectors lie on the boundaries,
// and only the first and the last vector of a row are taken apart.
// Operands that are not aligned alike, and a weight off a 16-byte boundary,
// go element by element (8192 x 4096 bf16: 104 against 25 us), and rows of
// more than 16384 elements in two passes.
#include "common.cuh"

#include <type_traits>

namespace bafe_cuda {
namespace lm {
namespace {

constexpr float E4M3_MAX = 448.0f;
constexpr int MAX_TPR = 512;           // threads of a row that is kept in registers
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
    int depth;             // rows per block row in shared memory
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

// Keeps the compiler from holding a converted copy of v across this point.
template <class T, int N>
__device__ __forceinline__ void opaque(Pack<T, N>& v) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) * N / 4); ++i) asm volatile("" : "+r"(v.w[i]));
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Until all but the newest depth - 1 groups have arrived.
__device__ __forceinline__ void copies_wait(int depth) {
    if (depth == 3) asm volatile("cp.async.wait_group 2;" ::: "memory");
    else if (depth == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// This thread's vectors of a row: vector j holds columns col(j) .. col(j) + VE,
// as far as they belong to the row.  (A variant without the tests, for rows
// of whole vectors only, ran slower: the compiler then works on all vectors
// at once and spills; 64 against 50 us for the gradient at 8192 x 4096
// bf16.)
template <int VE, int NV>
struct Lane {
    int first;             // column of vector 0 (negative: the row starts inside it)
    int step;              // columns from one vector to the next
    int width;
    uint32_t mask;         // bit j: any of vector j belongs to the row; bit 16 + j: all of it
    __device__ __forceinline__ Lane(int first_, int step_, int width_) : first(first_), step(step_), width(width_), mask(0) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (col(j) < width) mask |= 1u << j;
            if (col(j) >= 0 && col(j) + VE <= width) mask |= 1u << (16 + j);
        }
    }
    __device__ __forceinline__ int col(int j) const { return first + j * step; }
    __device__ __forceinline__ bool any(int j) const { return mask >> j & 1u; }
    __device__ __forceinline__ bool full(int j) const { return mask >> (16 + j) & 1u; }
    __device__ __forceinline__ bool has(int j, int e) const { return (unsigned)(col(j) + e) < (unsigned)width; }
};
template <class T, int VE, class L>
__device__ __noinline__ Pack<T, VE> load_part(const T* row, const L l, int j) {
    float f[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) f[e] = l.has(j, e) ? to_f32(row[l.col(j) + e]) : 0.0f;
    Pack<T, VE> p;
    pack(f, p);            // exact: they were of type T
    return p;
}
// The elements of a vector that belong to the row, out of line: a copy of
// this in each store costs instructions even where it is skipped.
template <class T, int VE, class L>
__device__ __noinline__ void store_part(T* row, const L l, int j, const Pack<T, VE> p) {
    constexpr int PER = 4 / sizeof(T);
#pragma unroll
    for (int e = 0; e < VE; ++e) {
        if (!l.has(j, e)) continue;
        const uint32_t bits = p.w[e / PER] >> (8 * sizeof(T) * (e % PER));
        T* at = row + l.col(j) + e;
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint32_t*>(at) = bits;
        else if constexpr (sizeof(T) == 2) *reinterpret_cast<unsigned short*>(at) = (unsigned short)bits;
        else *reinterpret_cast<unsigned char*>(at) = (unsigned char)bits;
    }
}
// at: where the row's vector 0 starts.
template <class T, int VE, class L>
__device__ __forceinline__ void store_any(T* at, const L& l, int j, const Pack<T, VE>& p) {
    if (l.full(j)) *reinterpret_cast<Pack<T, VE>*>(at + j * l.step) = p;
    else store_part<T, VE>(at - l.first, l, j, p);
}
// Starts the copy of one row's vectors into this thread's slots, `stride`
// apart.  at: where the row's vector 0 starts.
template <class T, int VE, int NV, class L>
__device__ __forceinline__ void fetch(Pack<T, VE>* slot, const T* at, const L& l, int stride) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        if (l.full(j)) copy16((uint32_t)__cvta_generic_to_shared(slot + j * stride), at + j * l.step);
        else if (l.any(j)) slot[j * stride] = load_part<T, VE>(at - l.first, l, j);
    }
}
template <class W, int VE, class L>
__device__ __forceinline__ Pack<W, VE> load_weight(const W* ws, const L& l, int j) {
    if (l.full(j) && (l.first & (VE - 1)) == 0) return *reinterpret_cast<const Pack<W, VE>*>(ws + l.col(j));
    return load_part<W, VE>(ws, l, j);
}

constexpr int MAX_DEPTH = 3;           // rows in flight or in use per block row; fewer where shared memory ends

// Rows of up to blockDim.x * NV * VE elements (VE: 16 bytes).  blockDim =
// (threads per row, rows per block): several rows share a block only when a
// row is one warp.  Shared memory: [depth][operands][NV][threads] vectors.
template <class T, class W, bool OUT8, int NV>
__global__ void __launch_bounds__(MAX_TPR, NV * (16 / sizeof(T)) <= 16 ? 2 : 1) rms_norm_kernel(const NormArgs g) {
    constexpr int VE = 16 / sizeof(T);
    extern __shared__ __align__(16) unsigned char smem_raw[];
    __shared__ float2 red[2][32];
    const int tpr = blockDim.x, warps = tpr >> 5, threads = tpr * blockDim.y;
    const bool res = g.res != nullptr;
    const int64_t step = (int64_t)gridDim.x * blockDim.y;
    int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    // the same for all of this block row's rows: step * x_ld is a multiple of VE, or there is no second row
    const Lane<VE, NV> l((int)threadIdx.x * VE - (int)(row * g.x_ld & (VE - 1)), tpr * VE, (int)g.width);
    // Places that move on by a step: of the row to be fetched next, of the
    // current one (y or residual_out may be x).  Overhead per row is what
    // this kernel has to spare: 16 elements a thread take as many
    // instructions as the addresses and the reduction.
    const T* x_next = static_cast<const T*>(g.x) + row * g.x_ld + l.first;
    const T* r_next = static_cast<const T*>(g.res) + (res ? row * g.res_ld + l.first : 0);
    T* h_at = static_cast<T*>(g.h) + (res ? row * g.h_ld + l.first : 0);
    typedef typename std::conditional<OUT8, E4m3, T>::type Y;
    Y* y_at = static_cast<Y*>(g.y) + row * g.y_ld + l.first;
    const int64_t x_move = step * g.x_ld, r_move = step * g.res_ld, h_move = step * g.h_ld, y_move = step * g.y_ld;
    int64_t ahead = row;                               // row of x_next
    Pack<T, VE>* const slot0 = reinterpret_cast<Pack<T, VE>*>(smem_raw) + threadIdx.y * tpr + threadIdx.x;
    const int deep = (res ? 2 : 1) * NV * threads;     // vectors from one depth to the next
    Pack<T, VE>* slot = slot0;
    auto start = [&](Pack<T, VE>* s) {
        if (ahead < g.rows) {
            fetch<T, VE, NV>(s, x_next, l, threads);
            x_next += x_move;
            if (res) {
                fetch<T, VE, NV>(s + NV * threads, r_next, l, threads);
                r_next += r_move;
            }
            ahead += step;
        }
        copies_commit();
    };
    for (int d = 0; d < g.depth; ++d) start(slot0 + d * deep);
    Pack<W, VE> w[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j)
        if (l.any(j)) w[j] = load_weight<W, VE>(static_cast<const W*>(g.w), l, j);
    int d = 0;
    for (int flip = 0; row < g.rows; row += step, flip ^= 1) {
        copies_wait(g.depth);
        Pack<T, VE> h[NV];
        Pair sum2 = pair(0.0f, 0.0f);
        float top = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (l.any(j)) {
                h[j] = slot[j * threads];
                if (res) {
                    add(h[j], slot[(NV + j) * threads]);     // the stored sum is what is normed
                    store_any<T, VE>(h_at, l, j, h[j]);
                }
                Pair v[VE / 2], wf[VE / 2];
                unpack(h[j], v);
                if (OUT8) {
                    opaque(w[j]);
                    unpack(w[j], wf);
                }
#pragma unroll
                for (int e = 0; e < VE / 2; ++e) {     // elements outside the row are 0
                    sum2 = fma2(v[e], v[e], sum2);
                    if (OUT8) {
                        float a, b;
                        split(mul2(v[e], wf[e]), a, b);
                        top = max_abs_nan(max_abs_nan(top, a), b);
                    }
                }
            }
        }
        float sum, odd;
        split(sum2, sum, odd);
        sum += odd;
        top = fabsf(top);
        row_reduce<OUT8>(sum, top, warps, red[flip]);
        start(slot);                                   // into the slots just read
        slot += deep;
        if (++d == g.depth) { d = 0; slot = slot0; }
        const float s = rsqrtf(sum * g.inv_width + g.eps);
        const float scale = OUT8 ? row_scale(top * s) : 1.0f;
        const float f = OUT8 ? __fdividef(s, scale) : s;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (l.any(j)) {
                opaque(w[j]);
                opaque(h[j]);
                Pair v[VE / 2], wf[VE / 2];
                unpack(h[j], v);
                unpack(w[j], wf);
#pragma unroll
                for (int e = 0; e < VE / 2; ++e) v[e] = mul2(mul2(v[e], pair(f, f)), wf[e]);
                Pack<Y, VE> y;
                pack_pairs<Y, VE>(v, y);
                store_any<Y, VE>(y_at, l, j, y);
            }
        }
        if (OUT8 && threadIdx.x == 0) g.scale[row] = scale;
        h_at += h_move;
        y_at += y_move;
    }
}

// Rows too long for registers, and operands that are not aligned alike (VE =
// 1): the same in two passes over the row.  The second reads h (or x) again; each thread reads only elements that it wrote
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
    int depth;             // rows per block row in shared memory
};

// Slot (block, row of the block) walks rows slot, slot + slots, ...; its
// share of dweight stays in registers over all of them and is written once.
// Partials are summed in slot order by norm_grad_weight_kernel: no atomics,
// the same bits every run.  Rows travel as in the forward kernel.
template <class T, class W, int NV>
__global__ void __launch_bounds__(MAX_TPR, 1) rms_norm_grad_kernel(const NormGradArgs g) {
    constexpr int VE = 16 / sizeof(T);
    extern __shared__ __align__(16) unsigned char smem_raw[];
    __shared__ float2 red[2][32];
    const int tpr = blockDim.x, warps = tpr >> 5, threads = tpr * blockDim.y;
    const bool more = g.dh != nullptr;
    second_may_start();
    const int64_t first_row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y, step = (int64_t)gridDim.x * blockDim.y;
    const Lane<VE, NV> l((int)threadIdx.x * VE - (int)(first_row * g.h_ld & (VE - 1)), tpr * VE, (int)g.width);
    const T* dy_next = static_cast<const T*>(g.dy) + first_row * g.dy_ld + l.first;
    const T* h_next = static_cast<const T*>(g.h) + first_row * g.h_ld + l.first;
    const T* dh_next = static_cast<const T*>(g.dh) + (more ? first_row * g.dh_ld + l.first : 0);
    T* dx_at = static_cast<T*>(g.dx) + first_row * g.dx_ld + l.first;
    const int64_t dy_move = step * g.dy_ld, h_move = step * g.h_ld, dh_move = step * g.dh_ld, dx_move = step * g.dx_ld;
    int64_t ahead = first_row;
    Pack<T, VE>* const slot0 = reinterpret_cast<Pack<T, VE>*>(smem_raw) + threadIdx.y * tpr + threadIdx.x;
    const int deep = (more ? 3 : 2) * NV * threads;
    Pack<T, VE>* slot = slot0;
    auto start = [&](Pack<T, VE>* s) {
        if (ahead < g.rows) {
            fetch<T, VE, NV>(s, dy_next, l, threads);
            fetch<T, VE, NV>(s + NV * threads, h_next, l, threads);
            dy_next += dy_move;
            h_next += h_move;
            if (more) {
                fetch<T, VE, NV>(s + 2 * NV * threads, dh_next, l, threads);
                dh_next += dh_move;
            }
            ahead += step;
        }
        copies_commit();
    };
    for (int d = 0; d < g.depth; ++d) start(slot0 + d * deep);
    Pair acc[NV][VE / 2];
    Pack<W, VE> w[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        if (l.any(j)) w[j] = load_weight<W, VE>(static_cast<const W*>(g.w), l, j);
#pragma unroll
        for (int e = 0; e < VE / 2; ++e) acc[j][e] = pair(0.0f, 0.0f);
    }
    int d = 0, flip = 0;
    for (int64_t row = first_row; row < g.rows; row += step, flip ^= 1) {
        copies_wait(g.depth);
        Pack<T, VE> dy[NV], h[NV], dh[NV];
        Pair sq2 = pair(0.0f, 0.0f), gh2 = sq2;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (l.any(j)) {
                dy[j] = slot[j * threads];
                h[j] = slot[(NV + j) * threads];
                if (more) dh[j] = slot[(2 * NV + j) * threads];
                opaque(w[j]);
                Pair v[VE / 2], dv[VE / 2], wf[VE / 2];
                unpack(h[j], v);
                unpack(dy[j], dv);
                unpack(w[j], wf);
#pragma unroll
                for (int e = 0; e < VE / 2; ++e) {     // elements outside the row are 0
                    sq2 = fma2(v[e], v[e], sq2);
                    gh2 = fma2(mul2(dv[e], wf[e]), v[e], gh2);
                }
            }
        }
        float sq, gh, odd_sq, odd_gh;
        split(sq2, sq, odd_sq);
        split(gh2, gh, odd_gh);
        sq += odd_sq;
        gh += odd_gh;
        row_sums(sq, gh, warps, red[flip]);
#pragma unroll
        for (int j = 0; j < NV; ++j) {                 // in registers before the slots are filled again
            if (l.any(j)) {
                opaque(dy[j]);
                opaque(h[j]);
                opaque(w[j]);
                if (more) opaque(dh[j]);
            }
        }
        start(slot);
        slot += deep;
        if (++d == g.depth) { d = 0; slot = slot0; }
        const float r = rsqrtf(sq * g.inv_width + g.eps);
        const float k = gh * g.inv_width * r * r * r;  // r^3 by itself leaves the range before h^2 does
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (l.any(j)) {
                Pair v[VE / 2], dv[VE / 2], o[VE / 2];
                unpack(h[j], v);
                unpack(dy[j], dv);
#pragma unroll
                for (int e = 0; e < VE / 2; ++e) {
                    dv[e] = mul2(dv[e], pair(r, r));   // dy r: half of dweight's term and of dx's
                    acc[j][e] = fma2(dv[e], v[e], acc[j][e]);
                }
                if (more) {
                    unpack(dh[j], o);
                } else {
#pragma unroll
                    for (int e = 0; e < VE / 2; ++e) o[e] = pair(0.0f, 0.0f);
                }
                Pair wf[VE / 2];
                unpack(w[j], wf);
#pragma unroll
                for (int e = 0; e < VE / 2; ++e) o[e] = fma2(v[e], pair(-k, -k), fma2(dv[e], wf[e], o[e]));
                Pack<T, VE> dx;
                pack_pairs<T, VE>(o, dx);
                store_any<T, VE>(dx_at, l, j, dx);
            }
        }
        dx_at += dx_move;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            float a, b;
            split(acc[j][e / 2], a, b);
            if (l.has(j, e)) g.part[first_row * g.width + l.col(j) + e] = e & 1 ? b : a;
        }
    }
}

// Rows too long for registers, and operands that are not aligned alike (VE =
// 1): two passes, the partial sums of dweight in
// the slot's own workspace row (each thread adds to its own elements only).
template <class T, class W, int VE>
__global__ void __launch_bounds__(1024) rms_norm_grad_long_kernel(const NormGradArgs g) {
    __shared__ float2 red[2][32];
    const W* __restrict__ ws = static_cast<const W*>(g.w);
    float* part = g.part + (int64_t)blockIdx.x * g.width;
    bool first = true;
    second_may_start();
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

// dweight = the slots' partial sums, added in a fixed order: 32 groups of
// slots per column, each a chain over every 32nd slot, then the groups.
template <class W>
__global__ void __launch_bounds__(1024) norm_grad_weight_kernel(const float* part, W* dw,
                                                                int slots, int64_t width) {
    __shared__ float s[32][33];
    const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
    float a = 0.0f;
    first_is_done();
    if (c < width) {
#pragma unroll 8
        for (int i = threadIdx.y; i < slots; i += 32) a += __ldcg(part + (int64_t)i * width + c);
    }
    s[threadIdx.y][threadIdx.x] = a;
    __syncthreads();
    const float t = warp_sum(s[threadIdx.x][threadIdx.y]);
    const int64_t col = (int64_t)blockIdx.x * 32 + threadIdx.y;
    if (threadIdx.x == 0 && col < width) dw[col] = from_f32<W>(t);
}

// -------------------------------------------------------------- dispatch --

// How rows are spread over threads: `nv` 16-byte vectors a thread, a warp at
// least, and a block of four rows where a row is one warp.  nv = 0: the row
// is too long for registers.  Two vectors a thread measured best where the
// row is long enough; one leaves threads idle in long rows' reductions,
// four halves the blocks that fit an SM.
constexpr int SMEM_PER_SM = 220 * 1024;
struct RowShape {
    int tpr, nv, rows_per_block, grid;
    int bytes(int operands) const { return operands * nv * tpr * rows_per_block * 16; }    // of one depth
    int depth(int operands) const {
        const int n = (SMEM_PER_SM - 1024) / bytes(operands);
        return n < MAX_DEPTH ? n : MAX_DEPTH;
    }
    int smem(int operands) const { return depth(operands) * bytes(operands); }
};
constexpr int LONG_BLOCKS_PER_SM = 2;
RowShape row_shape(int64_t rows, int64_t width, int esize, bool shifted, int sms, int per_sm) {
    const int ve = 16 / esize;
    const int64_t n = shifted ? (width + 2 * ve - 2) / ve : (width + ve - 1) / ve;   // vectors that a row may touch
    RowShape s;
    s.nv = n <= 64 ? 1 : 2;
    while (s.nv < 32 / ve && n > (int64_t)MAX_TPR * s.nv) s.nv *= 2;
    if (n > (int64_t)MAX_TPR * s.nv) {
        const int64_t room = (int64_t)sms * LONG_BLOCKS_PER_SM;
        return {1024, 0, 1, (int)(rows < room ? rows : room)};
    }
    const int64_t t = (n + s.nv - 1) / s.nv;
    s.tpr = (int)((t + 31) / 32 * 32);
    s.rows_per_block = s.tpr == 32 ? 4 : 1;
    const int64_t want = (rows + s.rows_per_block - 1) / s.rows_per_block;
    // several rows per block: a step of whole 16 bytes (see the top)
    const int64_t room = ((int64_t)sms * per_sm) / 8 * 8;
    s.grid = (int)(want < room ? want : room);
    return s;
}

// Blocks that an SM holds, by registers (64 a thread forward with up to 16
// elements a thread, else 128: at 80 the gradient spills, 71 against 50 us
// at 8192 x 4096 bf16) and by shared memory.  The grid is no larger, so that all blocks walk side by side.
constexpr int NORM_THREADS = 1024, WIDE_THREADS = 512, GRAD_THREADS = WIDE_THREADS;
RowShape shape_for(int64_t rows, int64_t width, int esize, bool shifted, int operands, int threads_per_sm, int sms) {
    const RowShape one = row_shape(rows, width, esize, shifted, sms, 1);
    if (!one.nv) return one;
    if (one.nv * (16 / esize) > 16) threads_per_sm = WIDE_THREADS;
    int n = threads_per_sm / (one.tpr * one.rows_per_block);
    const int fit = SMEM_PER_SM / (one.smem(operands) + 1024);
    if (n > fit) n = fit;
    return row_shape(rows, width, esize, shifted, sms, n < 1 ? 1 : n > 16 ? 16 : n);
}

template <class K>
int allow_smem(K kernel, bool (&done)[64], int dev) {
    if (done[dev]) return 0;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 224 * 1024) != cudaSuccess) {
        cudaGetLastError();
        return fail(14, "rms_norm: cudaFuncSetAttribute");
    }
    done[dev] = true;
    return 0;
}

template <class T, class W, bool OUT8, int NV>
int launch_norm(NormArgs a, const RowShape& s, int dev, cudaStream_t st) {
    static bool done[64] = {false};
    auto k = rms_norm_kernel<T, W, OUT8, NV>;
    if (int rc = allow_smem(k, done, dev)) return rc;
    a.depth = s.depth(a.res ? 2 : 1);
    k<<<s.grid, dim3(s.tpr, s.rows_per_block), s.smem(a.res ? 2 : 1), st>>>(a);
    return launched("rms_norm");
}

// vec: all operands aligned alike
template <class T, class W, bool OUT8>
int norm_typed(const NormArgs& a, bool vec, int dev, int sms, cudaStream_t st) {
    constexpr int VE = 16 / sizeof(T);
    const RowShape s = shape_for(a.rows, a.width, sizeof(T), a.x_ld % VE || a.width % VE, a.res ? 2 : 1, NORM_THREADS, sms);
    const unsigned grid = (unsigned)(a.rows < LONG_BLOCKS_PER_SM * sms ? a.rows : LONG_BLOCKS_PER_SM * sms);
    if (!vec) {
        rms_norm_long_kernel<T, W, OUT8, 1><<<grid, a.width > 512 ? 1024 : 128, 0, st>>>(a);
        return launched("rms_norm");
    }
    switch (s.nv) {
        case 1: return launch_norm<T, W, OUT8, 1>(a, s, dev, st);
        case 2: return launch_norm<T, W, OUT8, 2>(a, s, dev, st);
        case 4: return launch_norm<T, W, OUT8, 4>(a, s, dev, st);
        case 8: if constexpr (VE == 4) return launch_norm<T, W, OUT8, 8>(a, s, dev, st);
    }
    if (a.width % VE || a.x_ld % VE) rms_norm_long_kernel<T, W, OUT8, 1><<<grid, 1024, 0, st>>>(a);
    else rms_norm_long_kernel<T, W, OUT8, VE><<<grid, 1024, 0, st>>>(a);
    return launched("rms_norm");
}

template <class T, class W>
int norm_out(const NormArgs& a, bool out8, bool vec, int dev, int sms, cudaStream_t st) {
    return out8 ? norm_typed<T, W, true>(a, vec, dev, sms, st) : norm_typed<T, W, false>(a, vec, dev, sms, st);
}

// The gradient's shape: its slots are the workspace's rows, so the size
// query and the launch both come here.
RowShape grad_shape(int64_t rows, int64_t width, int esize, bool vec, bool shifted, int operands, int sms) {
    if (!vec) {
        const int64_t room = (int64_t)sms * LONG_BLOCKS_PER_SM;
        return {1024, 0, 1, (int)(rows < room ? rows : room)};
    }
    return shape_for(rows, width, esize, shifted, operands, GRAD_THREADS, sms);
}

template <class T, class W, int NV>
int launch_grad(NormGradArgs a, const RowShape& s, int dev, cudaStream_t st) {
    static bool done[64] = {false};
    auto k = rms_norm_grad_kernel<T, W, NV>;
    if (int rc = allow_smem(k, done, dev)) return rc;
    a.depth = s.depth(a.dh ? 3 : 2);
    k<<<s.grid, dim3(s.tpr, s.rows_per_block), s.smem(a.dh ? 3 : 2), st>>>(a);
    return launched("rms_norm_grad");
}

template <class T, class W>
int grad_typed(const NormGradArgs& a, const RowShape& s, bool aligned, int dev, void* dw, cudaStream_t st) {
    constexpr int VE = 16 / sizeof(T);
    int rc = 0;
    switch (s.nv) {
        case 1: rc = launch_grad<T, W, 1>(a, s, dev, st); break;
        case 2: rc = launch_grad<T, W, 2>(a, s, dev, st); break;
        case 4: rc = launch_grad<T, W, 4>(a, s, dev, st); break;
        case 8: if constexpr (VE == 4) rc = launch_grad<T, W, 8>(a, s, dev, st); break;
        default:
            if (aligned) rms_norm_grad_long_kernel<T, W, VE><<<s.grid, s.tpr, 0, st>>>(a);
            else rms_norm_grad_long_kernel<T, W, 1><<<s.grid, a.width > 512 ? s.tpr : 128, 0, st>>>(a);
            rc = launched("rms_norm_grad");
    }
    if (rc) return rc;
    return launch_second("rms_norm_grad weight sum", norm_grad_weight_kernel<W>, dim3((unsigned)((a.width + 31) / 32)), dim3(32, 32),
                         st, a.part, static_cast<W*>(dw), s.grid * s.rows_per_block, a.width);
}

int esize_of(int dtype) { return dtype == BAFE_DTYPE_F32 ? 4 : 2; }

int check_sizes(int64_t rows, int64_t width, int dtype, int wdtype, double eps) {
    if (rows < 0 || width < 1 || width > (int64_t(1) << 30)) return fail(8, "rms_norm: rows must be >= 0 and width in [1, 2^30]");
    if (!is_float_type(dtype)) return fail(8, "rms_norm: the rows must be f32, f16 or bf16");
    if (wdtype != dtype && wdtype != BAFE_DTYPE_F32) return fail(8, "rms_norm: the weight must have the rows' type or f32");
    if (!(eps >= 0.0)) return fail(8, "rms_norm: eps must be >= 0");
    return 0;
}

// Whether a tensor's rows start where x's do, relative to 16 bytes of x's
// type (`ve` elements): its base on such a boundary and its row stride alike.
bool alike(const void* p, int64_t ld, int esize, int64_t x_ld, int ve) {
    return !p || (reinterpret_cast<uintptr_t>(p) % (ve * esize) == 0 && (ld - x_ld) % ve == 0);
}

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
    const int es = esize_of(dtype), ve = 16 / es;
    if (!element_aligned(es, {x, residual, residual_out, out8 ? nullptr : y}) || !element_aligned(4, {out8 ? y_scale : nullptr}) ||
        !element_aligned(esize_of(weight_dtype), {weight}))
        return fail(8, "rms_norm: operands must start on a multiple of their element's size");
    int dev = 0, sms = 0;
    if (int rc = current_device(dev, sms)) return rc;
    NormArgs a;
    a.x = x; a.res = residual; a.w = weight; a.y = y; a.scale = y_scale; a.h = residual_out;
    a.x_ld = x_ld; a.res_ld = residual_ld; a.y_ld = y_ld; a.h_ld = residual_out_ld;
    a.rows = rows; a.width = width;
    a.eps = (float)eps;
    a.inv_width = (float)(1.0 / (double)width);
    const bool vec = alike(x, x_ld, es, x_ld, ve) && alike(residual, residual_ld, es, x_ld, ve) &&
                     alike(residual_out, residual_out_ld, es, x_ld, ve) &&
                     alike(y, y_ld, out8 ? 1 : es, x_ld, ve) && aligned16(weight);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool wf = weight_dtype == BAFE_DTYPE_F32;
    if (dtype == BAFE_DTYPE_F32) return norm_out<float, float>(a, out8, vec, dev, sms, st);
    if (dtype == BAFE_DTYPE_F16)
        return wf ? norm_out<__half, float>(a, out8, vec, dev, sms, st) : norm_out<__half, __half>(a, out8, vec, dev, sms, st);
    return wf ? norm_out<__nv_bfloat16, float>(a, out8, vec, dev, sms, st)
              : norm_out<__nv_bfloat16, __nv_bfloat16>(a, out8, vec, dev, sms, st);
}

BAFE_API int64_t bafe_cuda_rms_norm_grad_workspace(int64_t rows, int64_t width, int dtype) {
    if (check_sizes(rows, width, dtype, dtype, 0.0)) return -1;
    int dev = 0, sms = 0;
    if (current_device(dev, sms)) return -1;
    // whichever form a call takes
    int64_t most = 1;
    for (int form = 0; form < 6; ++form) {
        const RowShape s = grad_shape(rows, width, esize_of(dtype), form < 4, form & 1, form & 2 ? 3 : 2, sms);
        const int64_t slots = (int64_t)s.grid * s.rows_per_block;
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
    const int es = esize_of(dtype), ve = 16 / es;
    if (!element_aligned(es, {dy, h, dh, dx}) || !element_aligned(esize_of(weight_dtype), {weight, dweight}))
        return fail(8, "rms_norm_grad: operands must start on a multiple of their element's size");
    int dev = 0, sms = 0;
    if (int rc = current_device(dev, sms)) return rc;
    const bool vec = alike(dy, dy_ld, es, h_ld, ve) && alike(h, h_ld, es, h_ld, ve) && alike(dh, dh_ld, es, h_ld, ve) &&
                     alike(dx, dx_ld, es, h_ld, ve) && aligned16(weight);
    const bool shifted = h_ld % ve || width % ve;
    const RowShape g = grad_shape(rows, width, es, vec, shifted, dh ? 3 : 2, sms);
    const int64_t need = (int64_t)g.grid * g.rows_per_block * width * 4;
    if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 3u))
        return fail(8, "rms_norm_grad: workspace too small (see bafe_cuda_rms_norm_grad_workspace)");
    NormGradArgs a;
    a.dy = dy; a.h = h; a.w = weight; a.dh = dh; a.dx = dx; a.part = static_cast<float*>(workspace);
    a.dy_ld = dy_ld; a.h_ld = h_ld; a.dh_ld = dh_ld; a.dx_ld = dx_ld;
    a.rows = rows; a.width = width;
    a.eps = (float)eps;
    a.inv_width = (float)(1.0 / (double)width);
    const bool wf = weight_dtype == BAFE_DTYPE_F32, aligned = vec && !shifted;
    if (dtype == BAFE_DTYPE_F32) return grad_typed<float, float>(a, g, aligned, dev, dweight, st);
    if (dtype == BAFE_DTYPE_F16)
        return wf ? grad_typed<__half, float>(a, g, aligned, dev, dweight, st)
                  : grad_typed<__half, __half>(a, g, aligned, dev, dweight, st);
    return wf ? grad_typed<__nv_bfloat16, float>(a, g, aligned, dev, dweight, st)
              : grad_typed<__nv_bfloat16, __nv_bfloat16>(a, g, aligned, dev, dweight, st);
}
