// SPDX-License-Identifier: Unlicense
// Eight adjacent values of an operand of any floating type, as the row kernels
// read and write them: whole vectors where the operand's rows are aligned, single
// elements behind the end of a row and elsewhere.
#pragma once

#include "kernels.h"
#include "tc_ptx.cuh"
#include "vec.cuh"

namespace sam3 {

struct Raw8 {
    uint4 a, b;  // b: 32-bit values 4 .. 7
};

// The value at element i. WRITTEN: of memory that the kernel may write too (an operand that
// is also the result), which the read-only path is not defined for.
template <bool WRITTEN = false>
__device__ __forceinline__ float elem(const void *p, int dt, long i)
{
    if (dt == K_F32) {
        const float *q = reinterpret_cast<const float *>(p) + i;
        return WRITTEN ? *q : __ldg(q);
    }
    const uint16_t *q = reinterpret_cast<const uint16_t *>(p) + i;
    const uint16_t v = WRITTEN ? *q : __ldg(q);
    return dt == K_BF16 ? __uint_as_float((uint32_t)v << 16) : __half2float(__ushort_as_half(v));
}

// n of the eight values at element i; VEC: i is vector aligned.
template <bool VEC>
__device__ __forceinline__ Raw8 load8(const void *p, int dt, long i, int n)
{
    Raw8 r;
    r.a = r.b = make_uint4(0, 0, 0, 0);
    if (VEC && n >= 8) {
        if (dt == K_F32) {
            const uint4 *q = reinterpret_cast<const uint4 *>(reinterpret_cast<const float *>(p) + i);
            r.a = q[0];
            r.b = q[1];
        }
        else
            r.a = *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(p) + i);
        return r;
    }
    if (dt == K_F32) {
        const uint32_t *q = reinterpret_cast<const uint32_t *>(p) + i;
        uint32_t v[8];
#pragma unroll
        for (int e = 0; e < 8; e++)
            v[e] = e < n ? q[e] : 0u;
        r.a = make_uint4(v[0], v[1], v[2], v[3]);
        r.b = make_uint4(v[4], v[5], v[6], v[7]);
    }
    else {
        const uint16_t *q = reinterpret_cast<const uint16_t *>(p) + i;
        uint32_t v[8];
#pragma unroll
        for (int e = 0; e < 8; e++)
            v[e] = e < n ? q[e] : 0u;
        r.a = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
    }
    return r;
}

// Eight 16-bit values.
__device__ __forceinline__ void unpack8_16(const uint4 &a, int dt, float (&v)[8])
{
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
    if (dt == K_BF16) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            v[2 * e] = __uint_as_float(w[e] << 16);
            v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
        }
    }
    else {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[e]));
            v[2 * e] = f.x;
            v[2 * e + 1] = f.y;
        }
    }
}

__device__ __forceinline__ void unpack8(const Raw8 &r, int dt, float (&v)[8])
{
    if (dt != K_F32) {
        unpack8_16(r.a, dt, v);
        return;
    }
    v[0] = __uint_as_float(r.a.x);
    v[1] = __uint_as_float(r.a.y);
    v[2] = __uint_as_float(r.a.z);
    v[3] = __uint_as_float(r.a.w);
    v[4] = __uint_as_float(r.b.x);
    v[5] = __uint_as_float(r.b.y);
    v[6] = __uint_as_float(r.b.z);
    v[7] = __uint_as_float(r.b.w);
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi)
{
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}

__device__ __forceinline__ void store1(void *p, int dt, long i, float v)
{
    if (dt == K_F32)
        reinterpret_cast<float *>(p)[i] = v;
    else if (dt == K_BF16)
        reinterpret_cast<__nv_bfloat16 *>(p)[i] = from_f<__nv_bfloat16>(v);
    else
        reinterpret_cast<__half *>(p)[i] = from_f<__half>(v);
}

template <bool VEC>
__device__ __forceinline__ void store8(void *p, int dt, long i, int n, const float (&v)[8])
{
    if (dt == K_F32) {
        float *q = reinterpret_cast<float *>(p) + i;
        if (VEC && n >= 8) {
            reinterpret_cast<float4 *>(q)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4 *>(q)[1] = make_float4(v[4], v[5], v[6], v[7]);
            return;
        }
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (e < n)
                q[e] = v[e];
        return;
    }
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; e++)
        w[e] = dt == K_BF16 ? pack_bf16x2(v[2 * e], v[2 * e + 1]) : pack_f16x2(v[2 * e], v[2 * e + 1]);
    uint16_t *q = reinterpret_cast<uint16_t *>(p) + i;
    if (VEC && n >= 8) {
        *reinterpret_cast<uint4 *>(q) = make_uint4(w[0], w[1], w[2], w[3]);
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; e++)
        if (e < n)
            q[e] = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
}

// Eight E4M3 values, packed.
template <bool VEC>
__device__ __forceinline__ void store8_e4m3(void *p, long i, int n, uint2 v)
{
    uint8_t *q = reinterpret_cast<uint8_t *>(p) + i;
    if (VEC && n >= 8) {
        *reinterpret_cast<uint2 *>(q) = v;
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; e++)
        if (e < n)
            q[e] = (uint8_t)((e < 4 ? v.x : v.y) >> (8 * (e & 3)));
}

// Whether rows of the operand start at vectors of eight values (16 bytes; 8 of E4M3).
inline bool rows_vec8(const struct k_rows &r)
{
    const uintptr_t bytes = r.dt == K_E4M3 ? 8 : 16;
    return !r.p || (reinterpret_cast<uintptr_t>(r.p) % bytes == 0 && r.ld % 8 == 0 && r.s0 % 8 == 0);
}

}  // namespace sam3
