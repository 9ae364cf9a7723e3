// SPDX-License-Identifier: Unlicense
// What the two forms of cross attention (attn_cross.cu, attn_cross_tc.cu)
// share: their arguments and the rounding of pairs.
#pragma once

#include "div.cuh"
#include "kernels.h"
#include "tc_ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace sam3 {

struct XaArgs {
    const void *q, *k, *v;
    void *o;
    long qld, qs0, qs1, kld, ks0, ks1, vld, vs0, vs1, old, os0, os1;
    const int *klen;
    const uint8_t *kmask;
    int Nq, Nk, heads, kvheads, g, hd;
    long rows;    // Nq * g rows of one key head
    int nqt, cs;  // tiles of rows, CTAs sharing a tile's keys
    int kvec, qvec, ovec;  // 16-byte accesses allowed
    Div dg;                // g, for rows < 2^31
    float scale_log2;
    int *err;  // device error word (bounded waits of the tcgen05 form)
};

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi)
{
    return pack_bf16x2(lo, hi);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float ld_dsmem(uint32_t a)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}
template <typename T>
__device__ __forceinline__ T out_of(float v);
template <>
__device__ __forceinline__ float out_of<float>(float v)
{
    return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 out_of<__nv_bfloat16>(float v)
{
    return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half out_of<__half>(float v)
{
    return __float2half_rn(v);
}

// The tcgen05 form (attn_cross_tc.cu): whether it takes a call's operands (16-bit,
// 16-byte aligned starts and strides), and the call.
bool attn_cross_tc_takes(const XaArgs &a, int nb, int dt);
int attn_cross_tc(XaArgs &a, int nb, int dt, cudaStream_t s);

}  // namespace sam3
