// SPDX-License-Identifier: Unlicense
// The element types of the prompt-path operators: conversions and vectors.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace sam3 {

template <typename T>
__device__ __forceinline__ float to_f(T v)
{
    return (float)v;
}
// To nearest.
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v)
{
    return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v)
{
    return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_f<__half>(float v)
{
    return __float2half_rn(v);
}

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
    T v[V];
};

}  // namespace sam3
