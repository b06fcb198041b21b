// tc.cuh -- what the operators on the tcgen05 tensor cores share: waits that
// end (a wall-clock limit, then the CTA's abort flag and the device's error
// word), and their host side.
#pragma once
#include "common.cuh"

#include "bafe_dev.cuh"
#include "gemm_tc.cuh"

#include <cstdlib>

namespace bafe_cuda {
namespace lm {
namespace {

typedef unsigned int u32;
typedef unsigned long long u64;

// Shared state of one CTA.
struct Shared {
    u32 abort;
    u32 tmem_base;
};

// Args: a kernel's arguments, with the device's error word `err` and the limit
// `timeout_ns` of a wait.
template <class Args>
__device__ __forceinline__ bool raise(volatile Shared* sh, const Args& g, u32 code) {
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
template <class Args>
__device__ __forceinline__ u64 drain_ns(const Args& g) {
    return g.timeout_ns > 200000000ull ? g.timeout_ns : 200000000ull;
}

// The error word is allocated on the first call on a device, which may be
// inside a stream capture.
inline unsigned* error_word(int dev) {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    cudaThreadExchangeStreamCaptureMode(&mode);
    unsigned* w = device_error_word(dev);
    cudaThreadExchangeStreamCaptureMode(&mode);
    return w;
}

inline unsigned long long timeout_ns() {
    const char* to = getenv("BAFE_TC_TIMEOUT_MS");
    return (unsigned long long)(to ? atof(to) : 2000.0) * 1000000ull;
}

}  // namespace
}  // namespace lm
}  // namespace bafe_cuda
