// Host threads that ask for the same numbers and raise the same limits at the same time.
#include "per_device.h"

#include <cstdio>
#include <thread>
#include <vector>

static sam3::PerDevice numbers;
static sam3::PerDeviceLimit limits;
static int limit_of[2];  // what the fake driver was told last

int main()
{
    std::atomic<int> wrong{0};
    std::vector<std::thread> ts;
    for (int t = 0; t < 8; t++)
        ts.emplace_back([&, t] {
            for (int i = 0; i < 2000; i++) {
                const int dev = i & 1;
                int n = 0;
                if (!numbers.get(dev, n, [&](int &v) { v = 148 + dev; return true; }) || n != 148 + dev)
                    wrong++;
                if (!limits.raise(dev, 1 + (i * 7 + t * 131) % 4000, [&](int v) {
                        if (v < limit_of[dev])
                            wrong++;
                        limit_of[dev] = v;
                        return true;
                    }))
                    wrong++;
            }
        });
    for (auto &t : ts)
        t.join();
    for (int dev = 0; dev < 2; dev++)
        if (limit_of[dev] != limits.most[dev].load())
            wrong++;
    // a limit that could not be raised is tried again
    int tried = 0;
    auto no = [&](int) { tried++; return false; };
    if (limits.raise(7, 5, no) || limits.raise(7, 5, no) || tried != 2)
        wrong++;
    std::puts(wrong.load() ? "wrong" : "ok");
    return wrong.load() != 0;
}
