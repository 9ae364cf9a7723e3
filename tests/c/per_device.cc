// A question whose first answer cannot be had is asked again; an answer is kept, one
// for each device, zero among them.
#include "per_device.h"

#include <cstdio>

static sam3::PerDevice numbers;

int main()
{
    int asked = 0, n = -1;
    bool can = false;
    auto ask = [&](int &v) {
        asked++;
        v = can ? 74 : 0;
        return can;
    };
    bool ok = !numbers.get(3, n, ask) && asked == 1;
    can = true;
    ok = ok && numbers.get(3, n, ask) && n == 74 && asked == 2;
    ok = ok && numbers.get(3, n, ask) && n == 74 && asked == 2;
    ok = ok && numbers.get(0, n, ask) && n == 74 && asked == 3;
    auto none = [&](int &v) {
        asked++;
        v = 0;
        return true;
    };
    ok = ok && numbers.get(5, n, none) && n == 0 && asked == 4;
    ok = ok && numbers.get(5, n, none) && n == 0 && asked == 4;
    // devices without a place of their own are asked each time
    ok = ok && numbers.get(sam3::kMaxDevices, n, ask) && numbers.get(-1, n, ask) && n == 74 && asked == 6;
    std::puts(ok ? "ok" : "wrong");
    return !ok;
}
