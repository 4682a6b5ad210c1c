// Work to be done once per device ahead of a launch (kernel attributes are a device's, and a process may drive several).
#pragma once
#include <cuda_runtime_api.h>

#include <atomic>
#include <mutex>

namespace lt {

// run(work): work() returns 0 or an error.  Every caller returns after work has been done on its device: one that comes while another
// thread does it waits, so that no launch goes ahead of its attributes.  Work that failed is done again by the next caller.
class PerDeviceOnce {
    std::atomic<bool> done[64] = {};
    std::mutex m;

public:
    template <typename F>
    int run(F&& work) {
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return work();
        if (done[dev].load(std::memory_order_acquire)) return 0;
        std::lock_guard<std::mutex> hold(m);
        if (done[dev].load(std::memory_order_relaxed)) return 0;
        const int rc = work();
        if (rc == 0) done[dev].store(true, std::memory_order_release);
        return rc;
    }
};

}  // namespace lt

// LT_ONCE(once, statements): the statements of a launcher (LT_CUDA and LT_REQUIRE return their errors from it)
#define LT_ONCE(once, ...)                             \
    do {                                               \
        const int rc_once = (once).run([&]() -> int {  \
            __VA_ARGS__;                               \
            return 0;                                  \
        });                                            \
        if (rc_once != 0) return rc_once;              \
    } while (0)
