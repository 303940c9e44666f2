// once_per_device.h -- a set-up that a device needs once, such as a kernel's shared memory limit:
// the attribute belongs to the kernel on one device, not to the process.
#pragma once

#include <stdint.h>

#include <atomic>

namespace oasr {

class OncePerDevice {
    std::atomic<uint64_t> done_{0};  // a bit per device

  public:
    // 0, or what `set_up` returned; one that failed is tried again.  First calls may race: the set-up
    // has to bear being made twice (devices from the 64th on make it every time).
    template <typename F>
    int operator()(int device, F set_up) {
        const uint64_t bit = device >= 0 && device < 64 ? 1ull << device : 0;
        if (done_.load(std::memory_order_acquire) & bit) return 0;
        const int st = (int)set_up();
        if (st == 0) done_.fetch_or(bit, std::memory_order_release);
        return st;
    }
};

}  // namespace oasr
