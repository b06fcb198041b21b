// w4.cuh -- what the 4-bit weight kernels share: arguments, the tokens as
// 24-bit fixed-point numbers in three signed bytes, the stored result.
#pragma once
#include "common.cuh"

namespace bafe_cuda {
namespace lm {
namespace {

constexpr int LIMBS = 3;               // bytes of a token's value

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

// Integers as floats without a conversion instruction (a quarter or less of
// the rate of an addition): 0x4B400000 + v, for |v| < 2^22, is the float
// 1.5 * 2^23 + v.  The sums start from that integer.
constexpr int BIAS_BITS = 0x4B400000;
constexpr float BIAS = 12582912.0f;
__device__ __forceinline__ float small_float(int biased) { return __int_as_float(biased) - BIAS; }
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

__device__ __forceinline__ void load_x8(const W4Args& g, int tok, int64_t k, int64_t left, float (&f)[8]) {
    if (g.x_type == BAFE_DTYPE_BF16) load_tokens<__nv_bfloat16>(g.x, tok * g.x_ld + k, left, f);
    else if (g.x_type == BAFE_DTYPE_F16) load_tokens<__half>(g.x, tok * g.x_ld + k, left, f);
    else
#pragma unroll
        for (int j = 0; j < 8; ++j)
            f[j] = j < left ? float(static_cast<const __nv_fp8_e4m3*>(g.x)[tok * g.x_ld + k + j]) : 0.0f;
}

// Eight k of a token as bytes, k = 0 2 4 6 and 1 3 5 7 of each, and the
// power of two that one unit of them stands for (NaN: the block is not
// finite, the bytes are 0).
struct Limbs { uint32_t even[LIMBS], odd[LIMBS]; float unit; };
// Of 128 k, 8 on each lane of a half warp.
__device__ __forceinline__ Limbs token_limbs(const float (&f)[8]) {
    Limbs l;
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
    l.unit = finite ? __uint_as_float((uint32_t)(eb - 21) << 23) : __uint_as_float(0x7FC00000u);
    uint32_t y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        // adding 1.5 * 2^23 leaves the rounded integer in the low bits
        const int v = __float_as_int(fmaf(finite ? f[j] : 0.0f, up, BIAS)) - BIAS_BITS;
        y[j] = (uint32_t)(v + 0x808080) ^ 0x808080u;      // three signed bytes
    }
    const uint32_t p0 = __byte_perm(y[0], y[2], 0x5140), p1 = __byte_perm(y[4], y[6], 0x5140);
    const uint32_t p2 = __byte_perm(y[1], y[3], 0x5140), p3 = __byte_perm(y[5], y[7], 0x5140);
    l.even[0] = __byte_perm(p0, p1, 0x5410);
    l.even[1] = __byte_perm(p0, p1, 0x7632);
    l.odd[0] = __byte_perm(p2, p3, 0x5410);
    l.odd[1] = __byte_perm(p2, p3, 0x7632);
    l.even[2] = __byte_perm(__byte_perm(y[0], y[2], 0x0062), __byte_perm(y[4], y[6], 0x0062), 0x5410);
    l.odd[2] = __byte_perm(__byte_perm(y[1], y[3], 0x0062), __byte_perm(y[5], y[7], 0x0062), 0x5410);
    return l;
}
// The bytes' sums over `LANES` neighbouring lanes.
template <int LANES>
__device__ __forceinline__ void limb_sums(const Limbs& l, float (&sum)[LIMBS]) {
    auto of = [&](int m) { return __dp4a((int)l.even[m], 0x01010101, __dp4a((int)l.odd[m], 0x01010101, 0)); };
    int s01 = of(0) + of(1) * 65536, s2 = of(2);          // two below 2^15 in one word
#pragma unroll
    for (int d = 1; d < LANES; d <<= 1) {
        s01 += __shfl_xor_sync(0xFFFFFFFFu, s01, d);
        s2 += __shfl_xor_sync(0xFFFFFFFFu, s2, d);
    }
    const int s0 = (short)s01;
    sum[0] = (float)s0;
    sum[1] = (float)((s01 - s0) >> 16);
    sum[2] = (float)s2;
}

}  // namespace
}  // namespace lm
}  // namespace bafe_cuda
