// p8x_once.h -- something that has to be done once on each device a process launches on. No HIP in here.
#pragma once
#include <cstddef>
#include <mutex>
#include <vector>

namespace p8x {

class OncePerDevice {
    std::mutex mu_;
    std::vector<char> done_;

public:
    // set() unless it has returned 0 for this device; its error else (callers on several threads wait for each other)
    template <typename F>
    int run(int device, F set) {
        std::lock_guard<std::mutex> lock(mu_);
        if ((size_t)device >= done_.size()) done_.resize((size_t)device + 1, 0);
        if (done_[device]) return 0;
        const int rc = set();
        if (rc == 0) done_[device] = 1;
        return rc;
    }
};

}  // namespace p8x
