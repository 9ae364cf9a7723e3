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

// GELU of two values for products whose epilogue it bounds: max(x, 0) - a h, a = min(|x|,
// 8), h = erfc(a / sqrt 2) / 2 = 2^Q(a), one MUFU operation a value where the form
// above takes two. Q is a polynomial fitted for this kernel to log2 of h over [0, 8] by
// iterated weighted least squares (smallest largest error, 7.6e-6); in 32 bits h is off by
// 6e-6 of itself up to |x| = 5, 1.2e-5 up to 8, and the result by 6e-15 beyond.
// Infinities and NaN come out as they went in (-inf: -6e-15).
__device__ __forceinline__ void gelu_pair_exp(float &x0, float &x1)
{
    const float kC[9] = {-0.9999923706054688f,   -1.1513218879699707f,  -0.45819565653800964f,
                         -0.054337356239557266f, 0.008762168698012829f, -0.0010219766991212964f,
                         7.957417983561754e-05f, -3.6553351492329966e-06f, 7.428420900623678e-08f};
    const float a0 = fminf(fabsf(x0), 8.0f), a1 = fminf(fabsf(x1), 8.0f);
    const uint64_t a = f2_make(a0, a1);
    uint64_t q = f2_make(kC[8], kC[8]);
#pragma unroll
    for (int i = 7; i >= 0; i--)
        q = fma2(q, a, f2_make(kC[i], kC[i]));
    float q0, q1;
    f2_split(q, q0, q1);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(x0) : "f"(0.0f));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(x1) : "f"(0.0f));
    x0 = fmaf(-a0, ex2_approx(q0), x0);
    x1 = fmaf(-a1, ex2_approx(q1), x1);
}

}  // namespace sam3
