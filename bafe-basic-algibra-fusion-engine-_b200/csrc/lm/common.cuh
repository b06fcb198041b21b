// common.cuh -- shared pieces of the language-model operators (csrc/lm):
// element conversion, vector loads and stores, warp and block sums, and the
// host side's error and launch bookkeeping.
#pragma once
#include "bafe_cuda.h"
#include "internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <initializer_list>
#include <string>

namespace bafe_cuda {

// Device word that bounded waits report into (runtime.cpp).
unsigned* device_error_word(int dev);

namespace lm {

template <class T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// Rounded to nearest, ties to even: the only rounding between the 32-bit
// sums and what is stored.
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N consecutive elements moved by one load or store (two where they are
// more than 16 bytes: nothing here is aligned to more).
template <class T, int N> struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Vec { T v[N]; };

template <class T, int N>
__device__ __forceinline__ Vec<T, N> load_vec(const T* p) { return *reinterpret_cast<const Vec<T, N>*>(p); }
template <class T, int N>
__device__ __forceinline__ void store_vec(T* p, const Vec<T, N>& v) { *reinterpret_cast<Vec<T, N>*>(p) = v; }

// N consecutive elements as 32-bit words, and the values in them: two 16-bit
// values come out of a word with one instruction each, and go in with one
// (element-wise code spends several on taking the halves apart).
template <class T, int N> struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Pack { uint32_t w[sizeof(T) * N / 4]; };

template <int N> __device__ __forceinline__ void unpack(const Pack<float, N>& p, float (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = __uint_as_float(p.w[i]);
}
template <int N> __device__ __forceinline__ void unpack(const Pack<__nv_bfloat16, N>& p, float (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        f[2 * i] = __uint_as_float(p.w[i] << 16);
        f[2 * i + 1] = __uint_as_float(p.w[i] & 0xFFFF0000u);
    }
}
template <int N> __device__ __forceinline__ void unpack(const Pack<__half, N>& p, float (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i)
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}"
            : "=f"(f[2 * i]), "=f"(f[2 * i + 1]) : "r"(p.w[i]));
}
// Rounded to nearest, ties to even.
template <int N> __device__ __forceinline__ void pack(const float (&f)[N], Pack<float, N>& p) {
#pragma unroll
    for (int i = 0; i < N; ++i) p.w[i] = __float_as_uint(f[i]);
}
template <int N> __device__ __forceinline__ void pack(const float (&f)[N], Pack<__nv_bfloat16, N>& p) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) asm("cvt.rn.bf16x2.f32 %0, %2, %1;" : "=r"(p.w[i]) : "f"(f[2 * i]), "f"(f[2 * i + 1]));
}
template <int N> __device__ __forceinline__ void pack(const float (&f)[N], Pack<__half, N>& p) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) asm("cvt.rn.f16x2.f32 %0, %2, %1;" : "=r"(p.w[i]) : "f"(f[2 * i]), "f"(f[2 * i + 1]));
}
// e4m3, saturating to +-448, NaN kept.
struct E4m3 { unsigned char v; };
template <int N> __device__ __forceinline__ void pack(const float (&f)[N], Pack<E4m3, N>& p) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i)
        asm("{\n\t.reg .b16 l, h;\n\tcvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\t"
            "mov.b32 %0, {l, h};\n\t}" : "=r"(p.w[i])
            : "f"(f[4 * i]), "f"(f[4 * i + 1]), "f"(f[4 * i + 2]), "f"(f[4 * i + 3]));
}

// Two 32-bit floats that one instruction works on (each as by itself).
typedef unsigned long long Pair;
__device__ __forceinline__ Pair pair(float lo, float hi) {
    Pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void split(Pair p, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(p)); }
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
template <class T, int N> __device__ __forceinline__ void unpack(const Pack<T, N>& p, Pair (&f)[N / 2]) {
    float v[N];
    unpack(p, v);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) f[i] = pair(v[2 * i], v[2 * i + 1]);
}
template <class T, int N> __device__ __forceinline__ void pack_pairs(const Pair* f, Pack<T, N>& p) {
    float v[N];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) split(f[i], v[2 * i], v[2 * i + 1]);
    pack(v, p);
}

// Sums of the elements of two packs, each rounded to nearest once.
template <int N> __device__ __forceinline__ void add(Pack<float, N>& a, const Pack<float, N>& b) {
#pragma unroll
    for (int i = 0; i < N; ++i) a.w[i] = __float_as_uint(__uint_as_float(a.w[i]) + __uint_as_float(b.w[i]));
}
template <int N> __device__ __forceinline__ void add(Pack<__nv_bfloat16, N>& a, const Pack<__nv_bfloat16, N>& b) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) asm("add.rn.bf16x2 %0, %0, %1;" : "+r"(a.w[i]) : "r"(b.w[i]));
}
template <int N> __device__ __forceinline__ void add(Pack<__half, N>& a, const Pack<__half, N>& b) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) asm("add.rn.f16x2 %0, %0, %1;" : "+r"(a.w[i]) : "r"(b.w[i]));
}

// The larger magnitude with some sign, NaN if either is NaN.
__device__ __forceinline__ float max_abs_nan(float a, float b) {
    float r;
    asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// The larger value, NaN if either is NaN (fmaxf drops NaN).
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}
__device__ __forceinline__ float warp_max_nan(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    return v;
}

// ------------------------------------------------------------- host side --

constexpr int DTYPE_E4M3 = BAFE_CUDA_DTYPE_E4M3;

inline int fail(int code, const std::string& msg) {
    set_error(code, msg);
    return code;
}

// The current device and its SM count; an error code without a device.
int current_device(int& dev, int& sms);

// A second kernel that sums what the first one left in the workspace: the
// first says early that the second may be made ready (second_may_start), the
// second waits before it reads for the first one's end, its writes included
// (first_is_done), and reads from L2: it lives while they are written, so they
// are no constants to it.  0.8 us less than one after the other (gradient of the norm,
// 8192 x 4096 bf16: 49.5 -> 48.7 us).
__device__ __forceinline__ void second_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void first_is_done() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Reports a launch that was refused, else counts it.
inline int launched(const char* what) {
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return fail(7, std::string(what) + ": " + cudaGetErrorString(e));
    ++g_launch_count;
    return 0;
}

template <class... P, class... A>
int launch_second(const char* what, void (*kernel)(P...), dim3 grid, dim3 block, cudaStream_t st, const A&... args) {
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kernel, P(args)...);        // its error is read by launched
    return launched(what);
}

inline bool is_float_type(int dtype) {
    return dtype == BAFE_DTYPE_F32 || dtype == BAFE_DTYPE_F16 || dtype == BAFE_DTYPE_BF16;
}
// Whether operands start on a multiple of their element's size (any null one does).
inline bool element_aligned(int esize, std::initializer_list<const void*> ps) {
    uintptr_t all = 0;
    for (const void* p : ps) all |= reinterpret_cast<uintptr_t>(p);
    return (all & (uintptr_t)(esize - 1)) == 0;
}
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace lm
}  // namespace bafe_cuda
