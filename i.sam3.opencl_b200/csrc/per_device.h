// SPDX-License-Identifier: Unlicense
// Numbers that the host asks the driver for once per device.
#pragma once

namespace sam3 {

constexpr int kMaxDevices = 64;

struct PerDevice {
    int known[kMaxDevices];  // the number + 1, 0: not known (static tables start so)

    // The number of device dev (>= 0): ask(n) puts it into n and says whether it
    // could. An answer that could not be had is not kept: the next call asks again.
    template <typename Ask>
    bool get(int dev, int &n, const Ask &ask)
    {
        if (dev < 0 || dev >= kMaxDevices)
            return ask(n);
        if (known[dev]) {
            n = known[dev] - 1;
            return true;
        }
        if (!ask(n))
            return false;
        known[dev] = n + 1;
        return true;
    }
};

}  // namespace sam3
