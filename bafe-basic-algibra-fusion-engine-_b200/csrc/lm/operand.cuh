// operand.cuh -- what the tcgen05 products share (grouped.cu,
// cross_entropy.cu): bounded waits, reads of TMEM, the operands' tensor maps, and copies of
// operands that TMA cannot read in place.
#pragma once
#include "common.cuh"
#include "tc_launch.h"

#include "bafe_dev.cuh"
#include "gemm_tc.cuh"

#include <cuda.h>

#include <cstdlib>

namespace bafe_cuda {
namespace lm {
namespace {

using bafe::TmaDesc;
typedef unsigned int u32;
typedef unsigned long long u64;

// Bounded waits of a product's roles; Args has timeout_ns and the device's
// error word err.
struct Shared {
    u32 abort;
    u32 tmem_base;
};

template <class Args> __device__ __forceinline__ bool raise(volatile Shared* sh, const Args& g, u32 code) {
    sh->abort = 1u;
    atomicCAS(g.err, 0u, code);
    return false;
}
// Bounded wait on an mbarrier phase; acquire at cluster scope where the
// peer's arrivals complete the phase.
template <bool CLUSTER, class Args>
__device__ __forceinline__ bool wait(u32 bar, u32 parity, volatile Shared* sh, const Args& g, u32 code) {
    using namespace bafe::tc;
    auto ready = [&]() { return CLUSTER ? mbar_try_cluster(bar, parity) : mbar_try(bar, parity); };
    // The clock and the flag are looked at every 32nd time only: reading the
    // global timer takes longer than most waits.
    for (int i = 0; i < 32; ++i)
        if (ready()) return true;
    const u64 t0 = now_ns();
    while (true) {
        for (int i = 0; i < 32; ++i)
            if (ready()) return true;
        if (sh->abort) return false;
        if (now_ns() - t0 > g.timeout_ns) return raise(sh, g, code);
    }
}
template <class Args> __device__ __forceinline__ u64 drain_ns(const Args& g) {
    return g.timeout_ns > 200000000ull ? g.timeout_ns : 200000000ull;
}

// 32 lanes x 16 consecutive 32-bit columns; the wait names the registers so
// that no use of them moves above it.
__device__ __forceinline__ void tmem_ld16(u32 taddr, u32 (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :: "memory");
}

// Rows of a matrix (or of a stack of them, one per blockIdx.y) copied to rows
// that start on a 16-byte boundary, which TMA needs; row_bytes, src_ld and
// src_stride in bytes.  Four bytes a thread, put together from the two aligned
// words that hold them (words without a byte of the row are not read).  With
// offsets: only the matrices of experts that have rows; one whose clamped
// offsets do not ascend has none, whatever the others are.
__global__ void __launch_bounds__(256) align_rows_kernel(const unsigned char* __restrict__ src, int64_t src_ld, int64_t src_stride,
                                                         u32* __restrict__ dst, int64_t dst_words, int64_t n, int row_bytes,
                                                         const int* __restrict__ offsets, int all_rows) {
    if (offsets && min(max(offsets[blockIdx.y + 1], 0), all_rows) <= min(max(offsets[blockIdx.y], 0), all_rows)) return;
    constexpr int UP = 8;                                // words of a thread on their way at once
    const int words = (row_bytes + 3) / 4;
    for (int64_t r = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; r < n; r += (int64_t)gridDim.x * blockDim.y) {
        const unsigned char* s = src + blockIdx.y * src_stride + r * src_ld;
        u32* d = dst + (blockIdx.y * n + r) * dst_words;
        const int off = (int)(reinterpret_cast<uintptr_t>(s) & 3u);
        const u32* from = reinterpret_cast<const u32*>(s - off);
        for (int w0 = threadIdx.x; w0 < words; w0 += UP * blockDim.x) {
            u32 lo[UP], hi[UP];
#pragma unroll
            for (int u = 0; u < UP; ++u) {
                const int w = w0 + u * blockDim.x;
                if (w < words) {
                    lo[u] = from[w];
                    hi[u] = off && 4 * (w + 1) - off < row_bytes ? from[w + 1] : 0u;
                }
            }
#pragma unroll
            for (int u = 0; u < UP; ++u) {
                const int w = w0 + u * blockDim.x;
                if (w < words) d[w] = __funnelshift_r(lo[u], hi[u], 8 * off);
            }
        }
    }
}

constexpr int64_t MAX_DIM = int64_t(1) << 30;

// A matrix operand: rows of `cols` contiguous elements.
struct Matrix {
    const void* p;
    int64_t ld, stride;                // elements; stride between the experts' matrices
    int64_t rows, cols, count;
};

inline bool tma_ready(const Matrix& m, int es) {
    return aligned16(m.p) && (m.ld * es) % 16 == 0 && (m.count == 1 || (m.stride * es) % 16 == 0);
}
inline int64_t aligned_ld(int64_t cols, int es) {
    const int64_t per = 16 / es;
    return (cols + per - 1) / per * per;
}
// Workspace bytes of an operand's aligned copy; 0 when TMA can read it in place.
inline int64_t copy_bytes(const Matrix& m, int es) {
    if (tma_ready(m, es)) return 0;
    return (m.count * m.rows * aligned_ld(m.cols, es) * es + 255) / 256 * 256;
}

// offsets: the stack's matrices are the experts'.
inline int make_ready(const char* what, Matrix& m, int es, char*& ws, int sms, cudaStream_t st, const int* offsets = nullptr, int64_t all_rows = 0) {
    const int64_t bytes = copy_bytes(m, es);
    if (!bytes) return 0;
    if (m.cols * es > MAX_DIM) return fail(8, std::string(what) + ": rows of more than 2^30 bytes must start on 16-byte boundaries");
    const int64_t ld = aligned_ld(m.cols, es), words = ld * es / 4;
    // enough blocks for the device with all experts, and with one
    const int64_t want = (m.rows + 3) / 4, share = (int64_t)sms * 16 / m.count, most = share > sms ? share : sms;
    const dim3 grid((unsigned)(want < most ? want : most), (unsigned)m.count), block(64, 4);
    align_rows_kernel<<<grid, block, 0, st>>>(static_cast<const unsigned char*>(m.p), m.ld * es, m.stride * es, reinterpret_cast<u32*>(ws),
                                              words, m.rows, (int)(m.cols * es), offsets, (int)all_rows);
    if (int rc = launched((std::string(what) + ": aligned copy").c_str())) return rc;
    m.p = ws;
    m.ld = ld;
    m.stride = m.rows * ld;
    ws += bytes;
    return 0;
}

// Tensor map of a matrix operand: boxes of 128 bytes x `box_rows` rows.
inline int encode(TmaDesc* d, const Matrix& m, int es, uint32_t box_rows, std::string& err) {
    uint64_t dims[3] = {(uint64_t)m.cols, (uint64_t)m.rows, (uint64_t)m.count};
    uint64_t strides[2] = {(uint64_t)(m.ld * es), (uint64_t)((m.count == 1 ? m.rows * m.ld : m.stride) * es)};
    uint32_t box[3] = {(uint32_t)(128 / es), box_rows, 1};
    return tc_encode_tensor_map(d, es == 1 ? 0 : 2, 3, const_cast<void*>(m.p), dims, strides, box, 1, err);
}

inline unsigned long long timeout_ns() {
    const char* to = getenv("BAFE_TC_TIMEOUT_MS");
    return (unsigned long long)(to ? atof(to) : 2000.0) * 1000000ull;
}

// The storing warps wait for a whole contraction: 4 us per 64 of it on top
// of the limit, some ten times what a pair needs at full clocks.
inline unsigned long long contraction_ns(int64_t n) { return (unsigned long long)n / 64 * 4000; }

}  // namespace
}  // namespace lm
}  // namespace bafe_cuda
