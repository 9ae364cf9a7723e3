// SPDX-License-Identifier: Unlicense
// Numbers that the host asks the driver for once per device.
#pragma once

#include <atomic>
#include <mutex>

namespace sam3 {

constexpr int kMaxDevices = 64;

// Host threads may ask at the same time; they get the same answer.
struct PerDevice {
    std::atomic<int> known[kMaxDevices];  // the number + 1, 0: not known (static tables start so)

    // The number of device dev (>= 0): ask(n) puts it into n and says whether it
    // could. An answer that could not be had is not kept: the next call asks again.
    template <typename Ask>
    bool get(int dev, int &n, const Ask &ask)
    {
        if (dev < 0 || dev >= kMaxDevices)
            return ask(n);
        const int k = known[dev].load(std::memory_order_acquire);
        if (k) {
            n = k - 1;
            return true;
        }
        if (!ask(n))
            return false;
        known[dev].store(n + 1, std::memory_order_release);
        return true;
    }
};

// A limit that calls raise and none lowers, each device's own.
struct PerDeviceLimit {
    std::atomic<int> most[kMaxDevices];
    std::mutex lock;

    // set(n), true where it took place, unless the limit is n or above already.
    template <typename Set>
    bool raise(int dev, int n, const Set &set)
    {
        if (dev < 0 || dev >= kMaxDevices)
            return set(n);
        if (most[dev].load(std::memory_order_acquire) >= n)
            return true;
        // one thread at a time, so that a smaller limit never comes behind a larger one
        std::lock_guard<std::mutex> hold(lock);
        if (most[dev].load(std::memory_order_relaxed) >= n)
            return true;
        if (!set(n))
            return false;
        most[dev].store(n, std::memory_order_release);
        return true;
    }
};

}  // namespace sam3
