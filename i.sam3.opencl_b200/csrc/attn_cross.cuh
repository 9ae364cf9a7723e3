// SPDX-License-Identifier: Unlicense
// What the two forms of cross attention (attn_cross.cu, attn_cross_tc.cu)
// share: their arguments and the rounding of pairs.
#pragma once

#include "cluster.cuh"
#include "div.cuh"
#include "kernels.h"
#include "tc_ptx.cuh"
#include "vec.cuh"

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
// Weights are formed times 2^kWeightShift, in the products with V and in the
// sums alike. f16 holds the weights of a row down to 2^-14 of the largest with
// all its bits and loses those below 2^-25, while the sum of the 32-bit
// weights keeps them (one key 18 nats above 5184 others: all of these were
// lost); times 2^15, the most that stays below 65504, they are whole down to
// 2^-29 and rounded by 2^-40 below. bf16 and 32 bits have the exponents.
template <typename T>
constexpr float kWeightShift = __is_same(T, __half) ? 15.0f : 0.0f;

__device__ __forceinline__ void st_dsmem4(uint32_t a, float x, float y, float z, float w)
{
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(a), "f"(x), "f"(y), "f"(z), "f"(w)
                 : "memory");
}
__device__ __forceinline__ void st_dsmem2(uint32_t a, float x, float y)
{
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(a), "f"(x), "f"(y) : "memory");
}

// The parts of a tile's rows, merged over a cluster. Row r of the tile belongs
// to CTA r % cs; every part of it is pushed into that CTA's shared memory (remote
// stores, nothing waits for them; pulling cost a round trip per row or
// element: 64 queries x 384 keys 15 us against 7), as part[(p * rl + r / cs) * PR]
// with HDP columns of output, then its largest score (not scaled) and sum. After
// a cluster barrier each CTA merges its own rows: O = sum_p O_p w_p / sum_p l_p
// w_p, w_p = 2^((max_p - max) scale_log2). SCALED: a part's output is times a
// power of two whose inverse follows the sum; where these differ, the weights
// are divided by the sum and brought to the largest inverse first, so that
// nothing overflows and the smallest numbers are rounded once.
// A part without a visible key has maximum -inf and counts nothing, unless its sum is NaN.
template <int HDP>
struct Parts {
    static constexpr int PR = HDP + 4;
    // rl: rows a CTA holds of each part; live: rows of its own that exist
    template <int THREADS, bool SCALED, typename Store>
    static __device__ __forceinline__ void merge(float *part, int np, int rl, int live, float scale_log2,
                                                 const Store &store)
    {
        // weights of a row's parts and the last factor, a thread per row
        constexpr int kMost = kMaxClusterCtas;
        for (int i = threadIdx.x; i < live; i += THREADS) {
            float m = -INFINITY, l = 0.0f;
            float2 ml[kMost];
#pragma unroll
            for (int p = 0; p < kMost; p++) {
                ml[p] = p < np ? *reinterpret_cast<const float2 *>(part + (p * rl + i) * PR + HDP)
                               : make_float2(-INFINITY, 0.0f);
                m = fmaxf(m, ml[p].x);
            }
#pragma unroll
            for (int p = 0; p < kMost; p++)
                if (p < np) {
                    const bool none = ml[p].x == -INFINITY;
                    const float w = none ? 0.0f : exp2f((ml[p].x - m) * scale_log2);
                    l += none ? (ml[p].y == ml[p].y ? 0.0f : ml[p].y) : ml[p].y * w;
                    part[(p * rl + i) * PR + HDP] = w;
                }
            const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
            float last = inv;  // what the sum is multiplied by
            if constexpr (SCALED) {
                float lo = INFINITY, hi = 0.0f;
#pragma unroll
                for (int p = 0; p < kMost; p++)
                    if (p < np && ml[p].x != -INFINITY) {
                        const float f = part[(p * rl + i) * PR + HDP + 2];
                        lo = fminf(lo, f);
                        hi = fmaxf(hi, f);
                    }
                if (lo >= hi)  // of one scale
                    last = inv * hi;
                else {
                    hi = 0.0f;
                    for (int p = 0; p < np; p++) {
                        const float *at = part + (p * rl + i) * PR + HDP;
                        hi = at[0] != 0.0f ? fmaxf(hi, at[2]) : hi;
                    }
                    for (int p = 0; p < np; p++) {
                        float *at = part + (p * rl + i) * PR + HDP;
                        at[0] = at[0] != 0.0f ? at[0] * inv * (at[2] / hi) : 0.0f;
                    }
                    last = inv == inv ? hi : inv;
                }
            }
            part[i * PR + HDP + 2] = last;
        }
        __syncthreads();
        const int ne = live * (HDP / 4);  // elements, four columns each
        for (int e = threadIdx.x; e < ne; e += THREADS) {
            const int i = e / (HDP / 4), c = (e % (HDP / 4)) * 4;
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
            for (int p = 0; p < np; p++) {
                const float *src = part + (p * rl + i) * PR;
                const float w = src[HDP];
                const float4 v = *reinterpret_cast<const float4 *>(src + c);
                acc.x = fmaf(v.x, w, acc.x);
                acc.y = fmaf(v.y, w, acc.y);
                acc.z = fmaf(v.z, w, acc.z);
                acc.w = fmaf(v.w, w, acc.w);
            }
            const float last = part[i * PR + HDP + 2];
            store(i, c, acc.x * last, acc.y * last, acc.z * last, acc.w * last);
        }
    }
};

// The tcgen05 form (attn_cross_tc.cu): whether it takes a call's operands (16-bit,
// 16-byte aligned starts and strides), and the call.
bool attn_cross_tc_takes(const XaArgs &a, int nb, int dt);
int attn_cross_tc(XaArgs &a, int nb, int dt, cudaStream_t s);

}  // namespace sam3
