// SPDX-License-Identifier: Unlicense
// GELU of the operators with 16-bit (or narrower) results.
#pragma once

#include "tc_ptx.cuh"

namespace sam3 {

// GELU of two values for 16-bit outputs: max(x, 0) - |x| h with h = erfc(z) / 2,
// z = |x| / sqrt 2, as e^(-z^2) t P(t) / 2, t = 1 / (1 + p z) (the shape of Abramowitz &
// Stegun 7.1.26). P is fitted for this kernel by linear programming to the smallest
// relative error of erfc over z < 9.6, 3.7e-6, where the table's coefficients
// bound the absolute one and leave 0.2 % of GELU(-5) and 1 % of GELU(-8); with the
// 32-bit arithmetic h is off by 4e-6 for |x| < 5, 1e-5 at 13.
__device__ __forceinline__ void gelu_pair_rel(float &x0, float &x1)
{
    const float kP = 0.43516430f * 0.70710678118654752f;
    const float kE = -0.72134752044448170f;  // -log2(e) / 2
    const float kC[6] = {0.24603856f, 0.23720990f, 0.27436522f, 0.01132425f, 0.38257211f, -0.15151371f};
    const uint64_t x = f2_make(x0, x1);
    const uint64_t t = f2_make(rcp_approx(fmaf(kP, fabsf(x0), 1.0f)), rcp_approx(fmaf(kP, fabsf(x1), 1.0f)));
    uint64_t q = f2_make(kC[5], kC[5]);
#pragma unroll
    for (int i = 4; i >= 0; i--)
        q = fma2(q, t, f2_make(kC[i], kC[i]));
    float g0, g1, h0, h1;
    f2_split(fma2(mul2(x, f2_make(kE, kE)), x, f2_make(-1.0f, -1.0f)), g0, g1);
    f2_split(mul2(mul2(q, t), f2_make(ex2_approx(g0), ex2_approx(g1))), h0, h1);
    x0 = fmaf(-fabsf(x0), h0, fmaxf(x0, 0.0f));
    x1 = fmaf(-fabsf(x1), h1, fmaxf(x1, 0.0f));
}

}  // namespace sam3
