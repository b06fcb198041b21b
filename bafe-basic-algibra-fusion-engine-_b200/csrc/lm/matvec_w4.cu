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
// clock, 2.8 lane-instructions each, so the unpacking has to stay below
// that: two weights are made by one shift, one three-input logic operation
// (the four bits under the exponent of 1024 in f16, 128 in bf16) and one
// packed subtraction of that exponent plus the zero point -- exact, so the
// only roundings are the 32-bit sums' and the result's.  The products go
// through mma.sync m16n8k16 (weights as the 16 rows, tokens as the 8
// columns): a fused multiply-add per weight and token on the CUDA cores
// would alone take the whole budget.  tcgen05 has nothing to add here: its
// operands would have to be unpacked into shared memory first.
//
// The order of k inside an instruction is free as long as both operands
// agree, so the weights are used as they lie in memory: a lane takes whole
// 32-bit words (8 weights), whose shifts by 0, 4, 8 and 12 give the pairs
// (0,4), (1,5), (2,6), (3,7), and the tokens are laid out in shared memory in
// that order once per block.  All 16 k of one instruction must belong to
// one group, whose scale multiplies the instruction's sums: groups of a
// multiple of 128 let each lane load 16 bytes (4 lanes: 128 k), groups of 64
// 8 bytes, other multiples of 32 4 bytes.
//
// A block walks 16-row tiles; its warps share a tile's k-blocks of 128 and
// add their sums through shared memory.  The loads of the next k-blocks (or
// the next tile's) are in flight while the current ones are multiplied.
// Where the tiles are too few for the SMs, or the tokens too large for
// shared memory, k is also cut into slices over blocks, whose sums a second
// kernel adds in slice order.
#include "common.cuh"

namespace bafe_cuda {
namespace lm {
namespace {

constexpr int MAX_TOKENS = 32;         // per launch
constexpr int CHUNK = 4;               // k-blocks of 128 a warp has in flight per buffer
constexpr int RED_LD = 20;             // floats per token in the reduction: 16 rows, padded against bank conflicts

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
    int64_t qbytes;                    // bytes of a weight row
    int tokens;
    int group32;                       // group size / 32
    int scale_type;                    // BAFE dtype
    int x8;                            // x is e4m3
    int out_bf16;
    int kblocks;                       // of 128
    int slice_kb;                      // k-blocks per slice
    int tiles;
};

// 16-bit arithmetic of the instruction's operands.
struct H16 {
    typedef __half T;
    static constexpr uint32_t MAGIC = 0x64006400u;      // 1024, 1024
    static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("sub.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
};
struct B16 {
    typedef __nv_bfloat16 T;
    static constexpr uint32_t MAGIC = 0x43004300u;      // 128, 128
    static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("sub.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
};

__device__ __forceinline__ float scale_f32(uint32_t raw, int type) {
    if (type == BAFE_DTYPE_F32) return __uint_as_float(raw);
    if (type == BAFE_DTYPE_BF16) return __uint_as_float(raw << 16);
    return __half2float(__ushort_as_half((unsigned short)raw));
}
__device__ __forceinline__ uint32_t load_scale(const void* p, int64_t i, int type) {
    if (type == BAFE_DTYPE_F32) return __ldg(static_cast<const uint32_t*>(p) + i);
    return __ldg(static_cast<const unsigned short*>(p) + i);
}

// LW words (of 8 weights) from byte `at` of a row.  WIDE: one load of
// LW * 4 bytes (row starts and lengths are multiples of it).  Otherwise
// 4-byte loads where the word lies inside the row, else byte by byte; bytes
// behind the row's end read as 0.
enum class Load { Wide, Words, Bytes };
template <int LW, Load LD>
__device__ __forceinline__ void load_words(const uint8_t* row, int64_t at, int64_t qbytes, uint32_t (&w)[LW]) {
    if constexpr (LD == Load::Wide) {
        if (at >= qbytes) {
#pragma unroll
            for (int v = 0; v < LW; ++v) w[v] = 0;
        } else if constexpr (LW == 4) {
            const uint4 t = __ldcs(reinterpret_cast<const uint4*>(row + at));
            w[0] = t.x; w[1] = t.y; w[2] = t.z; w[3] = t.w;
        } else if constexpr (LW == 2) {
            const uint2 t = __ldg(reinterpret_cast<const uint2*>(row + at));
            w[0] = t.x; w[1] = t.y;
        } else {
            w[0] = __ldg(reinterpret_cast<const uint32_t*>(row + at));
        }
    } else {
#pragma unroll
        for (int v = 0; v < LW; ++v, at += 4) {
            if (LD == Load::Words && at + 4 <= qbytes) {
                w[v] = __ldg(reinterpret_cast<const uint32_t*>(row + at));
            } else {
                uint32_t t = 0;
#pragma unroll
                for (int b = 0; b < 4; ++b)
                    if (at + b < qbytes) t |= (uint32_t)__ldg(row + at + b) << (8 * b);
                w[v] = t;
            }
        }
    }
}

// What a warp has in flight: CHUNK k-blocks of its lane's two rows.
template <int LW>
struct Buffer {
    static constexpr int U = 4 / LW;                     // scale units of a k-block
    uint32_t w[CHUNK][2][U][LW];
    uint32_t s[CHUNK][2][LW == 4 ? 1 : U];               // raw scales
    uint32_t z[CHUNK];                                   // zero points: byte [row * 2 ...] see zero_at
    uint32_t z2[LW == 1 ? CHUNK : 1];
};

template <class E, int LW, int NT, Load LD>
__global__ void __launch_bounds__(512, 1) matvec_w4_kernel(const W4Args g) {
    typedef typename E::T T;
    constexpr int U = 4 / LW;
    extern __shared__ __align__(128) unsigned char smem[];
    const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int r = lane >> 2, c = lane & 3;
    const int kb0 = blockIdx.y * g.slice_kb;
    const int nkb = min(g.kblocks - kb0, g.slice_kb);
    const int x_row = nkb * 256 + 64;                    // bytes per token: 64 keep two tokens' reads apart
    unsigned char* xs = smem;
    float* red = reinterpret_cast<float*>(smem + (((size_t)g.tokens * x_row + 127) & ~size_t(127)));
    const int red_size = warps * NT * 8 * RED_LD;

    // chunks of the k-blocks warp, warp + warps, ... of one tile
    const int per_tile = (nkb + warps * CHUNK - 1) / (warps * CHUNK);

    auto load = [&](int tile, int ch, Buffer<LW>& b) {
        int64_t row[2] = {(int64_t)tile * 16 + r, (int64_t)tile * 16 + r + 8};
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (row[h] >= g.n) row[h] = g.n - 1;         // in bounds; its sums are not stored
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) {
            const int kbl = (ch * CHUNK + i) * warps + warp;
            if (kbl >= nkb) continue;                    // the same for the whole warp
            const int64_t kb = kb0 + kbl;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint8_t* qr = g.q + row[h] * g.q_ld;
#pragma unroll
                for (int l = 0; l < U; ++l)
                    load_words<LW, LD>(qr, kb * 64 + l * (16 * LW) + c * (4 * LW), g.qbytes, b.w[i][h][l]);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int l = 0; l < U; ++l) {
                    const int64_t k32 = kb * 4 + l * LW;             // the unit's first block of 32
                    b.s[i][h][l] = k32 * 32 < g.k ? load_scale(g.scales, row[h] * g.s_ld + k32 / g.group32, g.scale_type) : 0;
                }
            if (g.zeros) {
                uint32_t z[2] = {0, 0};
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int l = 0; l < U; ++l) {
                        const int64_t k32 = kb * 4 + l * LW;
                        if (k32 * 32 < g.k)
                            z[h] |= (uint32_t)__ldg(g.zeros + row[h] * g.z_ld + k32 / g.group32) << (8 * l);
                    }
                if constexpr (LW == 1) { b.z[i] = z[0]; b.z2[i] = z[1]; }
                else b.z[i] = z[0] | (z[1] << 16);
            }
        }
    };

    float acc[NT][4];
    auto compute = [&](int ch, const Buffer<LW>& b) {
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) {
            const int kbl = (ch * CHUNK + i) * warps + warp;
            if (kbl >= nkb) continue;
#pragma unroll
            for (int l = 0; l < U; ++l) {
                uint32_t off[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t z = 8;
                    if (g.zeros) z = LW == 1 ? ((h ? b.z2[LW == 1 ? i : 0] : b.z[i]) >> (8 * l)) & 255u
                                             : (b.z[i] >> (16 * h + 8 * l)) & 255u;
                    off[h] = E::MAGIC + z * 0x10001u;    // 1024 + z, 128 + z: z is below 128
                }
                float part[NT][4];
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) part[t][e] = 0.0f;
#pragma unroll
                for (int v = 0; v < LW; ++v) {
                    uint32_t a[2][4];
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int p = 0; p < 4; ++p)
                            a[h][p] = E::sub(((b.w[i][h][l][v] >> (4 * p)) & 0x000F000Fu) | E::MAGIC, off[h]);
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        uint4 xb = make_uint4(0, 0, 0, 0);
                        const int tok = t * 8 + r;
                        if (tok < g.tokens)
                            xb = *reinterpret_cast<const uint4*>(xs + tok * x_row + (kbl * 16 + (l * LW + v) * 4 + c) * 16);
                        E::mma(part[t], a[0][0], a[1][0], a[0][1], a[1][1], xb.x, xb.y);
                        E::mma(part[t], a[0][2], a[1][2], a[0][3], a[1][3], xb.z, xb.w);
                    }
                }
                const float s0 = scale_f32(b.s[i][0][l], g.scale_type), s1 = scale_f32(b.s[i][1][l], g.scale_type);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    acc[t][0] += s0 * part[t][0];
                    acc[t][1] += s0 * part[t][1];
                    acc[t][2] += s1 * part[t][2];
                    acc[t][3] += s1 * part[t][3];
                }
            }
        }
    };
    auto clear = [&]() {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[t][e] = 0.0f;
    };
    // The warps' sums of a tile, added in warp order; two buffers in turn,
    // so that one barrier per tile is enough.
    int flip = 0;
    auto finish = [&](int tile) {
        float* rb = red + flip * red_size;
        flip ^= 1;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                rb[(warp * NT * 8 + t * 8 + 2 * c + (e & 1)) * RED_LD + r + (e >> 1) * 8] = acc[t][e];
        __syncthreads();
        for (int o = threadIdx.x; o < g.tokens * 16; o += blockDim.x) {
            const int tok = o >> 4, row = o & 15;
            const int64_t n = (int64_t)tile * 16 + row;
            if (n < g.n) {
                float v = 0.0f;
                for (int w = 0; w < warps; ++w) v += rb[(w * NT * 8 + tok) * RED_LD + row];
                if (g.part) {
                    g.part[((int64_t)blockIdx.y * g.tokens + tok) * g.n + n] = v;
                } else {
                    if (g.x_scale) v *= g.x_scale[tok];
                    if (g.out_bf16) static_cast<__nv_bfloat16*>(g.y)[tok * g.y_ld + n] = __float2bfloat16_rn(v);
                    else static_cast<__half*>(g.y)[tok * g.y_ld + n] = __float2half_rn(v);
                }
            }
        }
        clear();
    };

    int tile = blockIdx.x, ch = 0;
    Buffer<LW> b0, b1;
    load(tile, 0, b0);                                   // in flight while the tokens are laid out

    // Tokens: 8 consecutive k as one 16-byte unit in the order 0 4 1 5 2 6 3 7;
    // the unit that lane c uses with word j of its k-block at j * 4 + c.
    {
        const int units = nkb * 16;
        const int64_t k_first = (int64_t)kb0 * 128;
        for (int o = threadIdx.x; o < g.tokens * units; o += blockDim.x) {
            const int tok = o / units, u = o % units;
            const int kbl = u >> 4, in = u & 15;
            const int l = in / (4 * LW), cc = in / LW & 3, v = in % LW;
            const int64_t k = k_first + (int64_t)u * 8;
            T e[8];
            if (g.x8) {
                const __nv_fp8_e4m3* xr = static_cast<const __nv_fp8_e4m3*>(g.x) + tok * g.x_ld;
#pragma unroll
                for (int j = 0; j < 8; ++j) e[j] = from_f32<T>(k + j < g.k ? float(xr[k + j]) : 0.0f);   // exact
            } else {
                const T* xr = static_cast<const T*>(g.x) + tok * g.x_ld;
                if (k + 8 <= g.k && (reinterpret_cast<uintptr_t>(xr + k) & 15u) == 0) {
                    const Vec<T, 8> t = load_vec<T, 8>(xr + k);
#pragma unroll
                    for (int j = 0; j < 8; ++j) e[j] = t.v[j];
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) e[j] = k + j < g.k ? xr[k + j] : from_f32<T>(0.0f);
                }
            }
            Vec<T, 8> p;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                p.v[2 * j] = e[j];
                p.v[2 * j + 1] = e[j + 4];
            }
            store_vec<T, 8>(reinterpret_cast<T*>(xs + tok * x_row + (kbl * 16 + (l * LW + v) * 4 + cc) * 16), p);
        }
    }
    __syncthreads();
    clear();
    // next (tile, chunk) of the walk; false behind the last
    auto step = [&](int& t, int& h) {
        if (++h == per_tile) { h = 0; t += gridDim.x; }
        return t < g.tiles;
    };
    while (true) {
        int t1 = tile, h1 = ch;
        const bool more1 = step(t1, h1);
        if (more1) load(t1, h1, b1);
        compute(ch, b0);
        if (ch == per_tile - 1) finish(tile);
        if (!more1) break;
        int t2 = t1, h2 = h1;
        const bool more2 = step(t2, h2);
        if (more2) load(t2, h2, b0);
        compute(h1, b1);
        if (h1 == per_tile - 1) finish(t1);
        if (!more2) break;
        tile = t2;
        ch = h2;
    }
}

// The slices' sums, added in slice order.
__global__ void __launch_bounds__(256) matvec_w4_sum_kernel(const W4Args g, int slices) {
    const int64_t o = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (o >= (int64_t)g.tokens * g.n) return;
    const int tok = (int)(o / g.n);
    const int64_t n = o % g.n;
    float v = 0.0f;
    for (int s = 0; s < slices; ++s) v += g.part[(int64_t)s * g.tokens * g.n + o];
    if (g.x_scale) v *= g.x_scale[tok];
    if (g.out_bf16) static_cast<__nv_bfloat16*>(g.y)[tok * g.y_ld + n] = __float2bfloat16_rn(v);
    else static_cast<__half*>(g.y)[tok * g.y_ld + n] = __float2half_rn(v);
}

// How a launch is cut: warps per block, slices of k.
struct W4Shape { int warps, slices, slice_kb, tiles, kblocks, smem; };

constexpr int SMEM_MAX = 227 * 1024;
int w4_smem(int tokens, int slice_kb, int warps) {
    const int nt8 = (tokens + 7) / 8 <= 1 ? 8 : (tokens + 7) / 8 <= 2 ? 16 : 32;
    return ((tokens * (slice_kb * 256 + 64) + 127) & ~127) + 2 * warps * nt8 * RED_LD * 4;
}

W4Shape w4_shape(int64_t tokens, int64_t n, int64_t k, int sms) {
    W4Shape s;
    s.tiles = (int)((n + 15) / 16);
    s.kblocks = (int)((k + 127) / 128);
    s.warps = 8;
    int slices = 1;
    // fewer tiles than SMs: cut k as long as each warp keeps a k-block
    while (s.tiles * slices * 2 <= sms && s.kblocks / (slices * 2) >= s.warps) slices *= 2;
    s.slice_kb = (s.kblocks + slices - 1) / slices;
    while (w4_smem((int)tokens, s.slice_kb, s.warps) > SMEM_MAX) s.slice_kb = (s.slice_kb + 1) / 2;
    s.slices = (s.kblocks + s.slice_kb - 1) / s.slice_kb;
    // more than one block's shared memory per SM: the warps of one block
    // have to cover the memory latency alone
    if (w4_smem((int)tokens, s.slice_kb, 8) > SMEM_MAX / 2 && s.slice_kb >= 16 &&
        w4_smem((int)tokens, s.slice_kb, 16) <= SMEM_MAX)
        s.warps = 16;
    s.smem = w4_smem((int)tokens, s.slice_kb, s.warps);
    return s;
}

template <class E, int LW, int NT, Load LD>
int w4_launch(const W4Args& a, const W4Shape& s, int dev, int sms, cudaStream_t st) {
    auto k = matvec_w4_kernel<E, LW, NT, LD>;
    static bool ready[64] = {false};
    if (!ready[dev]) {
        if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX) != cudaSuccess) {
            cudaGetLastError();
            return fail(14, "matvec_w4: cudaFuncSetAttribute");
        }
        ready[dev] = true;
    }
    int per_sm = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, k, s.warps * 32, s.smem) != cudaSuccess || per_sm < 1) {
        cudaGetLastError();
        return fail(14, "matvec_w4: the kernel does not fit an SM");
    }
    int64_t room = (int64_t)sms * per_sm / s.slices;
    if (room < 1) room = 1;
    const unsigned gx = (unsigned)(s.tiles < room ? s.tiles : room);
    k<<<dim3(gx, s.slices), s.warps * 32, s.smem, st>>>(a);
    return launched("matvec_w4");
}

template <class E, int LW, Load LD>
int w4_tokens(const W4Args& a, const W4Shape& s, int dev, int sms, cudaStream_t st) {
    if (a.tokens <= 8) return w4_launch<E, LW, 1, LD>(a, s, dev, sms, st);
    if (a.tokens <= 16) return w4_launch<E, LW, 2, LD>(a, s, dev, sms, st);
    return w4_launch<E, LW, 4, LD>(a, s, dev, sms, st);
}

template <class E>
int w4_typed(const W4Args& a, const W4Shape& s, int dev, int sms, cudaStream_t st) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(a.q) | (uintptr_t)a.q_ld;
    const int64_t group = (int64_t)a.group32 * 32;
    // one load per lane has to stay inside a group, and inside the row
    if (group % 128 == 0 && at % 16 == 0 && a.qbytes % 16 == 0) return w4_tokens<E, 4, Load::Wide>(a, s, dev, sms, st);
    if (group % 64 == 0 && at % 8 == 0 && a.qbytes % 8 == 0) return w4_tokens<E, 2, Load::Wide>(a, s, dev, sms, st);
    if (at % 4 == 0) return w4_tokens<E, 1, Load::Words>(a, s, dev, sms, st);
    return w4_tokens<E, 1, Load::Bytes>(a, s, dev, sms, st);
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
    int64_t need = 0;
    for (int64_t done = 0; done < tokens && done < 2 * MAX_TOKENS; done += MAX_TOKENS) {
        const int64_t m = tokens - done < MAX_TOKENS ? tokens - done : MAX_TOKENS;
        const W4Shape s = w4_shape(m, n, k, sms);
        if (s.slices > 1 && s.slices * m * n * 4 > need) need = s.slices * m * n * 4;
    }
    if (tokens > MAX_TOKENS && tokens % MAX_TOKENS) {
        const int64_t m = tokens % MAX_TOKENS;
        const W4Shape s = w4_shape(m, n, k, sms);
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
    int dev = 0, sms = 0;
    if (int rc = current_device(dev, sms)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    for (int64_t done = 0; done < tokens; done += MAX_TOKENS) {
        const int64_t m = tokens - done < MAX_TOKENS ? tokens - done : MAX_TOKENS;
        const W4Shape s = w4_shape(m, n, k, sms);
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
        a.qbytes = (k + 1) / 2;
        a.tokens = (int)m;
        a.group32 = (int)(group / 32);
        a.scale_type = scale_dtype;
        a.x8 = x8;
        a.out_bf16 = y_dtype == BAFE_DTYPE_BF16;
        a.kblocks = s.kblocks;
        a.slice_kb = s.slice_kb;
        a.tiles = s.tiles;
        // e4m3 values are exact in f16; f16 and bf16 rows are used as they are
        const int rc = x_dtype == BAFE_DTYPE_BF16 ? w4_typed<B16>(a, s, dev, sms, st) : w4_typed<H16>(a, s, dev, sms, st);
        if (rc) return rc;
        if (s.slices > 1) {
            matvec_w4_sum_kernel<<<(unsigned)((m * n + 255) / 256), 256, 0, st>>>(a, s.slices);
            if (int rc2 = launched("matvec_w4 slice sum")) return rc2;
        }
    }
    return 0;
}
