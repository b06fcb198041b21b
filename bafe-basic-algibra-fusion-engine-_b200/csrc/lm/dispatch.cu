// dispatch.cu -- rows on their way to the experts and back: copies into the
// order by expert, weighted sums out of it, and the sums' gradient.
//
//   dispatch      y[place[t][j]] = x[t]
//   combine       out[t] = sum_j w[t][j] y[place[t][j]]
//   combine_grad  dy[place[t][j]] = w[t][j] dout[t],  dw[t][j] = <dout[t], y[place[t][j]]>
//
// All three walk the rows t, so that the rows' own side is read (or written)
// once and the k places are whole rows somewhere in y: every byte moves once.
// Memory bounds them; there is nothing to compute that would take as long.
// 8192 x 4096 bf16 by 8, 604 MB: dispatch 97.5 us (6.2 TB/s, nearly all written),
// combine 89.4 (6.8, nearly all read); the gradient's 218 MB 39.6 (5.5).
// A place outside [0, n) is no place: nothing is read or written for it.
//
// Accesses are of 16 bytes where every operand's rows allow it, else of 4,
// else of one element.
#include "common.cuh"

namespace bafe_cuda {
namespace lm {
namespace {

constexpr int MAX_K = 31;
constexpr int THREADS = 256;

struct MoveArgs {
    const unsigned char* x;            // dispatch: rows
    unsigned char* y;                  // dispatch: places
    const float* scale;
    float* scale_out;
    const int* place;
    int64_t x_ld, y_ld, place_ld;      // x_ld, y_ld in bytes
    int64_t rows, n, units;            // units: accesses of a row
    int k;
};

// blockDim: (threads along a row, rows).
template <class U> __global__ void __launch_bounds__(THREADS) dispatch_kernel(const MoveArgs g) {
    const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    const int64_t u = (int64_t)blockIdx.y * blockDim.x + threadIdx.x;
    if (row >= g.rows) return;
    const int* place = g.place + row * g.place_ld;
    if (u < g.units) {
        const U v = reinterpret_cast<const U*>(g.x + row * g.x_ld)[u];
#pragma unroll 4
        for (int j = 0; j < g.k; ++j) {
            const int p = place[j];
            if (p >= 0 && p < g.n) reinterpret_cast<U*>(g.y + p * g.y_ld)[u] = v;
        }
    }
    if (g.scale && u == 0)
        for (int j = 0; j < g.k; ++j) {
            const int p = place[j];
            if (p >= 0 && p < g.n) g.scale_out[p] = g.scale[row];
        }
}

struct SumArgs {
    const void* y;
    const void* dout;                  // gradient
    void* out;                         // combine: the sums; gradient: dy
    float* dweights;
    const int* place;
    const float* weights;              // or null (combine)
    int64_t y_ld, out_ld, dout_ld, place_ld, weights_ld;
    int64_t rows, n, units;
    int k;
};

// N elements as they lie in memory, also one 16-bit element, and their values.
template <class T, int N> struct Raw {
    Pack<T, N> p;
    __device__ __forceinline__ void load(const T* at) { p = *reinterpret_cast<const Pack<T, N>*>(at); }
    __device__ __forceinline__ void store(T* at) const { *reinterpret_cast<Pack<T, N>*>(at) = p; }
    __device__ __forceinline__ void values(float (&f)[N]) const { unpack<N>(p, f); }
    __device__ __forceinline__ void set(const float (&f)[N]) { pack<N>(f, p); }
};
template <class T> struct Raw16 {
    T p;
    __device__ __forceinline__ void load(const T* at) { p = *at; }
    __device__ __forceinline__ void store(T* at) const { *at = p; }
    __device__ __forceinline__ void values(float (&f)[1]) const { f[0] = to_f32(p); }
    __device__ __forceinline__ void set(const float (&f)[1]) { p = from_f32<T>(f[0]); }
};
template <> struct Raw<__half, 1> : Raw16<__half> {};
template <> struct Raw<__nv_bfloat16, 1> : Raw16<__nv_bfloat16> {};

// Places of a row on their way at once: of a sum (8192 x 4096 bf16, 8 places:
// 4 89.4 us, 8 99.4, with a third of the threads; 2 91.4), and of its gradient
// (4096 x 2048, 6 places: 8 39.6 us, 6 38.9, 3 40.4).
constexpr int AT_ONCE = 4, BATCH = 8;

template <class T, int N> __global__ void __launch_bounds__(THREADS) combine_kernel(const SumArgs g) {
    const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    const int64_t u = (int64_t)blockIdx.y * blockDim.x + threadIdx.x;
    if (row >= g.rows || u >= g.units) return;
    const int* place = g.place + row * g.place_ld;
    const T* y = static_cast<const T*>(g.y) + u * N;
    float sum[N];
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i] = 0.0f;
    for (int j0 = 0; j0 < g.k; j0 += AT_ONCE) {
        Raw<T, N> v[AT_ONCE];
        bool in[AT_ONCE];
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
            const int p = j0 + j < g.k ? place[j0 + j] : -1;
            in[j] = p >= 0 && p < g.n;
            if (in[j]) v[j].load(y + p * g.y_ld);
        }
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j)
            if (in[j]) {
                const float w = g.weights ? g.weights[row * g.weights_ld + j0 + j] : 1.0f;
                float f[N];
                v[j].values(f);
#pragma unroll
                for (int i = 0; i < N; ++i) sum[i] += w * f[i];
            }
    }
    Raw<T, N> r;
    r.set(sum);
    r.store(static_cast<T*>(g.out) + row * g.out_ld + u * N);
}

constexpr int GRAD_BLOCKS = 2;
// blockDim.x threads (whole warps) share a row; the dot products are summed
// over the lanes, then over the row's warps in their order.
template <class T, int N> __global__ void __launch_bounds__(THREADS, GRAD_BLOCKS) combine_grad_kernel(const SumArgs g) {
    __shared__ float part[THREADS / 32][BATCH];
    const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5, warp = threadIdx.x >> 5, first = threadIdx.y * warps;
    const bool mine = row < g.rows;
    for (int j0 = 0; j0 < g.k; j0 += BATCH) {
        int p[BATCH];
        float w[BATCH], dot[BATCH];
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
            p[j] = mine && j0 + j < g.k ? g.place[row * g.place_ld + j0 + j] : -1;
            if (p[j] >= g.n) p[j] = -1;
            w[j] = p[j] >= 0 ? g.weights[row * g.weights_ld + j0 + j] : 0.0f;
            dot[j] = 0.0f;
        }
        if (mine)
            for (int64_t u = threadIdx.x; u < g.units; u += blockDim.x) {
                Raw<T, N> r, v[BATCH];
                r.load(static_cast<const T*>(g.dout) + row * g.dout_ld + u * N);
#pragma unroll
                for (int j = 0; j < BATCH; ++j)
                    if (p[j] >= 0) v[j].load(static_cast<const T*>(g.y) + p[j] * g.y_ld + u * N);
                float d[N];
                r.values(d);
#pragma unroll
                for (int j = 0; j < BATCH; ++j)
                    if (p[j] >= 0) {
                        float f[N];
                        v[j].values(f);
#pragma unroll
                        for (int i = 0; i < N; ++i) {
                            dot[j] += d[i] * f[i];
                            f[i] = d[i] * w[j];
                        }
                        v[j].set(f);
                        v[j].store(static_cast<T*>(g.out) + p[j] * g.out_ld + u * N);
                    }
            }
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
            dot[j] = warp_sum(dot[j]);
            if (lane == 0) part[first + warp][j] = dot[j];
        }
        if (warps == 1) {                                // nothing to wait for
            __syncwarp();
            if (mine && lane < BATCH && j0 + lane < g.k) g.dweights[row * g.k + j0 + lane] = part[first][lane];
            __syncwarp();
            continue;
        }
        __syncthreads();
        if (mine && threadIdx.x < BATCH && j0 + (int)threadIdx.x < g.k) {
            float s = 0.0f;
            for (int i = 0; i < warps; ++i) s += part[first + i][threadIdx.x];
            g.dweights[row * g.k + j0 + threadIdx.x] = s;
        }
        __syncthreads();
    }
}

constexpr int64_t MAX_DIM = int64_t(1) << 30;

int check_sizes(const char* what, int64_t rows, int64_t k, int64_t n, int64_t width) {
    if (rows < 0 || rows > MAX_DIM || n < 0 || n > MAX_DIM || k < 1 || k > MAX_K || width < 1 || width > MAX_DIM)
        return fail(8, std::string(what) + ": sizes out of range (0 <= rows, n <= 2^30, 1 <= k <= 31, 1 <= width <= 2^30)");
    return 0;
}

// Bytes of an access: all of `bits` (addresses, strides and lengths, in bytes) are multiples of it.
int access(uint64_t bits, int es) { return bits % 16 == 0 ? 16 : bits % 4 == 0 && es < 4 ? 4 : es; }

// Threads along a row (at least `least`) and rows of a block.
dim3 block_of(int64_t units, int least) {
    int x = least;
    while (x < THREADS && x < units) x *= 2;
    return dim3((unsigned)x, (unsigned)(THREADS / x));
}

template <class T, class F> int with_access(int bytes, F f) {
    if (bytes == 16) return f(std::integral_constant<int, 16 / (int)sizeof(T)>());
    if (bytes == 4 && sizeof(T) < 4) return f(std::integral_constant<int, 4 / (int)sizeof(T)>());
    return f(std::integral_constant<int, 1>());
}
template <class F> int with_type(int dtype, F f) {
    if (dtype == BAFE_DTYPE_F32) return f(float());
    if (dtype == BAFE_DTYPE_BF16) return f(__nv_bfloat16());
    return f(__half());
}

}  // namespace
}  // namespace lm
}  // namespace bafe_cuda

#define BAFE_API extern "C" __attribute__((visibility("default")))

using namespace bafe_cuda;
using namespace bafe_cuda::lm;

BAFE_API int bafe_cuda_dispatch(const void* x, int64_t x_ld, const float* scale, const int* place, int64_t place_ld, void* y,
                                int64_t y_ld, float* scale_out, int64_t rows, int64_t k, int64_t n, int64_t width,
                                int element_bytes, void* stream) {
    if (int rc = check_sizes("dispatch", rows, k, n, width)) return rc;
    const int es = element_bytes;
    if (es != 1 && es != 2 && es != 4) return fail(8, "dispatch: elements must have 1, 2 or 4 bytes");
    if ((scale != nullptr) != (scale_out != nullptr)) return fail(8, "dispatch: scale and scale_out go together");
    if (rows == 0 || n == 0) return 0;
    if (!x || !place || !y) return fail(8, "dispatch: null operand");
    if ((rows > 1 && (x_ld < width || place_ld < k)) || (n > 1 && y_ld < width))
        return fail(8, "dispatch: strides must be at least the rows' lengths");
    if (!element_aligned(es, {x, y}) || !element_aligned(4, {scale, scale_out, place}))
        return fail(8, "dispatch: operands must start on a multiple of their element's size");
    MoveArgs g = {};
    g.x = static_cast<const unsigned char*>(x);
    g.y = static_cast<unsigned char*>(y);
    g.scale = scale;
    g.scale_out = scale_out;
    g.place = place;
    g.x_ld = rows > 1 ? x_ld * es : 0;
    g.y_ld = n > 1 ? y_ld * es : 0;
    g.place_ld = place_ld;
    g.rows = rows;
    g.n = n;
    g.k = (int)k;
    const int bytes = access((uintptr_t)x | (uintptr_t)y | (uint64_t)(g.x_ld | g.y_ld | width * es), es);
    g.units = width * es / bytes;
    const dim3 block = block_of(g.units, 1);
    const int64_t columns = (g.units + block.x - 1) / block.x;
    const dim3 grid((unsigned)((rows + block.y - 1) / block.y), (unsigned)columns);
    if (columns > 65535) return fail(8, "dispatch: rows too wide for their alignment");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (bytes == 16) dispatch_kernel<uint4><<<grid, block, 0, st>>>(g);
    else if (bytes == 4) dispatch_kernel<uint32_t><<<grid, block, 0, st>>>(g);
    else if (bytes == 2) dispatch_kernel<uint16_t><<<grid, block, 0, st>>>(g);
    else dispatch_kernel<unsigned char><<<grid, block, 0, st>>>(g);
    return launched("dispatch");
}

BAFE_API int bafe_cuda_combine(const void* y, int64_t y_ld, const int* place, int64_t place_ld, const float* weights,
                               int64_t weights_ld, void* out, int64_t out_ld, int64_t rows, int64_t k, int64_t n,
                               int64_t width, int dtype, void* stream) {
    if (int rc = check_sizes("combine", rows, k, n, width)) return rc;
    if (!is_float_type(dtype)) return fail(8, "combine: rows must be f32, f16 or bf16");
    if (rows == 0) return 0;
    if ((!y && n) || !place || !out) return fail(8, "combine: null operand");
    if ((n > 1 && y_ld < width) || (rows > 1 && (place_ld < k || out_ld < width || (weights && weights_ld < 0))))
        return fail(8, "combine: strides must be at least the rows' lengths");
    const int es = dtype == BAFE_DTYPE_F32 ? 4 : 2;
    if (!element_aligned(es, {y, out}) || !element_aligned(4, {place, weights}))
        return fail(8, "combine: operands must start on a multiple of their element's size");
    SumArgs g = {};
    g.y = y;
    g.out = out;
    g.place = place;
    g.weights = weights;
    g.y_ld = n > 1 ? y_ld : 0;
    g.out_ld = rows > 1 ? out_ld : 0;
    g.place_ld = place_ld;
    g.weights_ld = weights_ld;
    g.rows = rows;
    g.n = n;
    g.k = (int)k;
    const int bytes = access((uintptr_t)y | (uintptr_t)out | (uint64_t)((g.y_ld | g.out_ld | width) * es), es);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return with_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        return with_access<T>(bytes, [&](auto c) {
            constexpr int N = decltype(c)::value;
            g.units = width / N;
            const dim3 block = block_of(g.units, 1);
            const int64_t columns = (g.units + block.x - 1) / block.x;
            if (columns > 65535) return fail(8, "combine: rows too wide for their alignment");
            combine_kernel<T, N><<<dim3((unsigned)((rows + block.y - 1) / block.y), (unsigned)columns), block, 0, st>>>(g);
            return launched("combine");
        });
    });
}

BAFE_API int bafe_cuda_combine_grad(const void* dout, int64_t dout_ld, const void* y, int64_t y_ld, const int* place,
                                    int64_t place_ld, const float* weights, int64_t weights_ld, void* dy, int64_t dy_ld,
                                    float* dweights, int64_t rows, int64_t k, int64_t n, int64_t width, int dtype,
                                    void* stream) {
    if (int rc = check_sizes("combine_grad", rows, k, n, width)) return rc;
    if (!is_float_type(dtype)) return fail(8, "combine_grad: rows must be f32, f16 or bf16");
    if (rows == 0) return 0;
    if (!dout || (n && (!y || !dy)) || !place || !weights || !dweights) return fail(8, "combine_grad: null operand");
    if ((n > 1 && (y_ld < width || dy_ld < width)) || (rows > 1 && (place_ld < k || dout_ld < 0 || weights_ld < 0)))
        return fail(8, "combine_grad: strides must be at least the rows' lengths");
    const int es = dtype == BAFE_DTYPE_F32 ? 4 : 2;
    if (!element_aligned(es, {dout, y, dy}) || !element_aligned(4, {place, weights, dweights}))
        return fail(8, "combine_grad: operands must start on a multiple of their element's size");
    SumArgs g = {};
    g.y = y;
    g.dout = dout;
    g.out = dy;
    g.dweights = dweights;
    g.place = place;
    g.weights = weights;
    g.y_ld = n > 1 ? y_ld : 0;
    g.out_ld = n > 1 ? dy_ld : 0;
    g.dout_ld = rows > 1 ? dout_ld : 0;
    g.place_ld = place_ld;
    g.weights_ld = weights_ld;
    g.rows = rows;
    g.n = n;
    g.k = (int)k;
    int dev = 0, sms = 0;
    if (int rc = current_device(dev, sms)) return rc;
    const int bytes = access((uintptr_t)y | (uintptr_t)dout | (uintptr_t)dy |
                             (uint64_t)((g.y_ld | g.out_ld | g.dout_ld | width) * es), es);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return with_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        return with_access<T>(bytes, [&](auto c) {
            constexpr int N = decltype(c)::value;
            g.units = width / N;
            // a warp a row where there are rows for all: no waiting for one another
            const dim3 block = rows >= 16 * sms ? dim3(32, THREADS / 32) : block_of(g.units, 32);
            combine_grad_kernel<T, N><<<(unsigned)((rows + block.y - 1) / block.y), block, 0, st>>>(g);
            return launched("combine_grad");
        });
    });
}
