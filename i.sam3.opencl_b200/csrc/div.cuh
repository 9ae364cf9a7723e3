// SPDX-License-Identifier: Unlicense
// Division of 31-bit indexes by run-time constants.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace sam3 {

// n / d for n < 2^31 by a multiplication: m = ceil(2^(31 + l) / d) with l =
// ceil(log2 d) exceeds 2^(31 + l) / d by less than 1, which adds less than n /
// 2^(31 + l) < 1 / d to the quotient.
struct Div {
    uint32_t d, m, s;
};
inline Div make_div(uint32_t d)
{
    uint32_t l = 0;
    while ((1ull << l) < d)
        l++;
    return Div{d, (uint32_t)(((1ull << (31 + l)) + d - 1) / d), l};
}
__device__ __forceinline__ uint32_t quot(uint32_t n, const Div &v)
{
    return v.d == 1 ? n : __umulhi(n, v.m) >> (v.s - 1);
}

}  // namespace sam3
