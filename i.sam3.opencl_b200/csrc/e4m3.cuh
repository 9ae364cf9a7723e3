// SPDX-License-Identifier: Unlicense
// Blocks of E4M3 values with a power-of-two scale.
#pragma once

#include "kernels.h"

#include <cuda_runtime.h>
#include <stdint.h>

namespace sam3 {

constexpr int kScaleBlock = 128;

// The larger of m and |x|; a NaN counts for nothing. A block's largest magnitude
// that comes out infinite is taken again over its finite values (larger_finite).
__device__ __forceinline__ float larger(float m, float x)
{
    return fmaxf(m, fabsf(x));
}
__device__ __forceinline__ float larger_finite(float m, float x)
{
    const float a = fabsf(x);
    return a < __int_as_float(0x7f800000) ? fmaxf(m, a) : m;
}
__device__ __forceinline__ bool infinite(float m)
{
    return m == __int_as_float(0x7f800000);
}

// The scale of a block whose largest finite magnitude is m, as the E8M0 byte e + 127: the smallest e >= -126 with the magnitude at most 448 2^e =
// 1.75 * 2^(8 + e). Adding 2^21 - 1 carries into the exponent exactly when the
// fraction is above 0.75.
__device__ __forceinline__ uint32_t scale_byte(float m)
{
    const uint32_t x = (__float_as_uint(m) + 0x1fffffu) >> 23;
    return x > 9 ? x - 8 : 1u;
}
__device__ __forceinline__ float scale_value(uint32_t byte)
{
    return __uint_as_float(byte << 23);
}
// 1 / scale (bytes 1 .. 247: a normal number).
__device__ __forceinline__ float scale_inverse(uint32_t byte)
{
    return __uint_as_float((254u - byte) << 23);
}

// Four values times the inverse scale, to nearest; the product is exact or far
// below E4M3's smallest number. INF: some may be infinite, which the conversion
// would saturate; 0 x added makes them NaN.
template <bool INF>
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d, float inv)
{
    uint16_t lo, hi;
    if (INF) {
        a = fmaf(a, 0.0f, a);
        b = fmaf(b, 0.0f, b);
        c = fmaf(c, 0.0f, c);
        d = fmaf(d, 0.0f, d);
    }
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b * inv), "f"(a * inv));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d * inv), "f"(c * inv));
    return (uint32_t)lo | ((uint32_t)hi << 16);
}
__device__ __forceinline__ uint2 pack8_e4m3(const float (&v)[8], float inv, bool inf)
{
    if (inf)
        return make_uint2(pack_e4m3<true>(v[0], v[1], v[2], v[3], inv), pack_e4m3<true>(v[4], v[5], v[6], v[7], inv));
    return make_uint2(pack_e4m3<false>(v[0], v[1], v[2], v[3], inv), pack_e4m3<false>(v[4], v[5], v[6], v[7], inv));
}

// A scale as it is stored (E8M0 byte or fp32 bits) and its value.
__device__ __forceinline__ uint32_t scale_raw(const void *p, int dt, long i)
{
    return dt == K_E8M0 ? (uint32_t)__ldg(reinterpret_cast<const uint8_t *>(p) + i)
                        : __ldg(reinterpret_cast<const uint32_t *>(p) + i);
}
__device__ __forceinline__ float scale_of(uint32_t raw, int dt)
{
    if (dt != K_E8M0)
        return __uint_as_float(raw);
    // 0 is 2^-127, below the normal numbers, and 255 NaN: both have one more bit
    return __uint_as_float(raw << 23 | (((raw + 1) & 255u) <= 1u ? 0x00400000u : 0u));
}
__device__ __forceinline__ void put_scale(void *p, int dt, long i, uint32_t byte)
{
    if (dt == K_E8M0)
        reinterpret_cast<uint8_t *>(p)[i] = (uint8_t)byte;
    else
        reinterpret_cast<float *>(p)[i] = scale_value(byte);
}

}  // namespace sam3
