// once_per_device.h -- a pointer per device that the first caller makes.
#pragma once
#include <atomic>
#include <mutex>

namespace bafe_cuda {

// Threads that ask at the same time get the same pointer: one makes it, the
// others wait.  What make() returns is published as a whole; null is not
// kept, the next caller tries again.
template <class T, int N>
class OncePerDevice {
public:
    template <class Make>
    T* get(int dev, Make make) {
        if (dev < 0 || dev >= N) return nullptr;
        if (T* p = at_[dev].load(std::memory_order_acquire)) return p;
        std::lock_guard<std::mutex> lk(mu_);
        T* p = at_[dev].load(std::memory_order_relaxed);
        if (!p) {
            p = make();
            at_[dev].store(p, std::memory_order_release);
        }
        return p;
    }
    // Null where nobody asked yet.
    T* peek(int dev) const { return dev < 0 || dev >= N ? nullptr : at_[dev].load(std::memory_order_acquire); }

private:
    std::mutex mu_;
    std::atomic<T*> at_[N] = {};
};

}  // namespace bafe_cuda
