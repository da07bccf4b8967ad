// tvq_once.h -- something that has to be done once on each device of a
// process and may fail (host only).
#pragma once

#include <atomic>

namespace tvq {

class OncePerDevice {
    static constexpr int kDevices = 64;
    std::atomic<bool> done_[kDevices] = {};

   public:
    // do_it() -> 0 if it worked; called until it has worked on device `dev`.
    template <typename F>
    int operator()(int dev, F&& do_it) {
        const bool known = dev >= 0 && dev < kDevices;
        if (known && done_[dev].load(std::memory_order_acquire)) return 0;
        const int rc = do_it();
        if (known && rc == 0) done_[dev].store(true, std::memory_order_release);
        return rc;
    }
};

}  // namespace tvq
