// per_device.h -- what has to be done once on every device of a process. No HIP: also built by the host compiler.
#pragma once
#include <atomic>

namespace ixg {

class OncePerDevice {
    static constexpr int kMost = 64;
    std::atomic<bool> done_[kMost] = {};

public:
    // set() unless it has succeeded on device `dev`. Its error is the call's, and the next call tries again.
    template <class F>
    auto operator()(int dev, F set) -> decltype(set()) {
        typedef decltype(set()) Error;
        const bool known = dev >= 0 && dev < kMost;
        if (known && done_[dev].load(std::memory_order_acquire)) return Error{};
        const Error e = set();
        if (known && e == Error{}) done_[dev].store(true, std::memory_order_release);
        return e;
    }
};

}  // namespace ixg
