// SPDX-License-Identifier: Unlicense
// Rotary positions: tables of angles made on the device, and the rotation of
// rows by them. The table has the layout of cb_rope_apply: [npos, rot / 2]
// (cos, sin) pairs in fp32.
#include "kernels.h"
#include "pdl.cuh"
#include "tc_ptx.cuh"
#include "tmap.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace sam3 {
namespace {

// cos and sin of the angle of `turns` turns. The turns are reduced to a
// quadrant and a remainder in [-1/8, 1/8] in 64 bits (exact, so far
// positions lose nothing), the remainder goes through sincospif in 32.
__device__ __forceinline__ float2 cos_sin_turns(double turns)
{
    const long long q = __double2ll_rn(4.0 * turns);
    const float r = (float)fma(-0.25, (double)q, turns);
    float s, c;
    sincospif(2.0f * r, &s, &c);
    const float c1 = (q & 1) ? s : c, s1 = (q & 1) ? c : s;
    const bool neg_c = ((q + 1) & 2) != 0, neg_s = (q & 2) != 0;
    return make_float2(neg_c ? -c1 : c1, neg_s ? -s1 : s1);
}

// Frequencies in turns per position, by value (captured graphs keep them).
struct Freqs {
    double t[K_ROPE_MAX / 2];
};

// One thread per table entry, entries of a position adjacent: write bound.
__global__ void __launch_bounds__(256) rope_table_kernel(const __grid_constant__ Freqs f, int half,
                                                         long first, long n, float amp,
                                                         float2 *__restrict__ cs)
{
    griddep_wait();
    griddep_launch();
    for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < n;
         i += (long)gridDim.x * blockDim.x) {
        const long p = i / half;
        const int j = (int)(i - p * half);
        const float2 v = cos_sin_turns((double)(first + p) * f.t[j]);
        cs[i] = make_float2(v.x * amp, v.y * amp);
    }
}

struct RotArgs {
    const void *x;
    void *y;
    const float2 *cs;
    const int *pos;
    long ldx, sx0, sx1, ldy, sy0, sy1;  // elements: row, sequence and head strides
    long rows;                          // nb * N
    int N, heads, hd, half, pos0, npos;
    int nrot, nch;  // chunks of a head: rotated, all (the rest is copied)
    int nhg, hpt;   // head groups of a row; heads per thread
};

template <typename T>
__device__ __forceinline__ float rd(T v)
{
    return (float)v;
}
template <typename T>
__device__ __forceinline__ T wr(float v);
template <>
__device__ __forceinline__ float wr<float>(float v)
{
    return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 wr<__nv_bfloat16>(float v)
{
    return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half wr<__half>(float v)
{
    return __float2half_rn(v);
}

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
    T v[V];
};

// A thread takes one chunk of W adjacent columns (HALVES: the W columns at j
// and the W at half + j) of up to hpt heads of one row, so that the chunk's
// (cos, sin) pairs are read once for all of them. W columns are 16 bytes of
// input, or 1 (a pair of columns 2 j, 2 j + 1 without HALVES) for rows that
// are not 16-byte aligned. Memory bound: X read and Y written once, the
// table rows from L2.
template <typename TI, typename TO, int W, bool HALVES>
__global__ void __launch_bounds__(256) rope_rotate_kernel(const __grid_constant__ RotArgs a)
{
    constexpr int CW = HALVES || W > 1 ? W : 2;     // columns of a vector
    constexpr int NP = HALVES ? W : CW / 2;         // pairs of a chunk
    using VI = Vec<TI, W>;
    using VO = Vec<TO, W>;
    griddep_wait();
    griddep_launch();
    const long total = a.rows * a.nhg * a.nch;
    for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < total;
         i += (long)gridDim.x * blockDim.x) {
        const long rg = i / a.nch;
        const int c = (int)(i - rg * a.nch);
        const long row = rg / a.nhg;
        const int hg = (int)(rg - row * a.nhg);
        const long b = row / a.N, n = row - b * a.N;
        const long p = a.pos ? (long)__ldg(a.pos + row) : a.pos0 + n;
        const bool turn = c < a.nrot && p >= 0 && p < a.npos;
        const TI *x = reinterpret_cast<const TI *>(a.x) + b * a.sx0 + n * a.ldx;
        TO *y = reinterpret_cast<TO *>(a.y) + b * a.sy0 + n * a.ldy;
        float2 cs[NP];
        if (turn) {
            const float2 *src = a.cs + p * a.half + c * NP;
            if (NP % 2 == 0) {
#pragma unroll
                for (int e = 0; e < NP; e += 2) {
                    const float4 v = __ldg(reinterpret_cast<const float4 *>(src + e));
                    cs[e] = make_float2(v.x, v.y);
                    cs[e + 1 < NP ? e + 1 : e] = make_float2(v.z, v.w);
                }
            }
            else {
#pragma unroll
                for (int e = 0; e < NP; e++)
                    cs[e] = __ldg(src + e);
            }
        }
        // copied chunks follow the rotated ones: single vectors from column 2 half on
        const bool two = c < a.nrot && (HALVES || W == 1);
        const int col = c < a.nrot ? (HALVES ? c * W : c * CW)
                                   : 2 * a.half + (c - a.nrot) * W;
        const int col2 = HALVES ? col + a.half : col + 1;
#pragma unroll 4
        for (int h = hg; h < a.heads; h += a.nhg) {
            const TI *xh = x + h * a.sx1;
            TO *yh = y + h * a.sy1;
            const VI u = *reinterpret_cast<const VI *>(xh + col);
            VI w = u;
            if (two)
                w = *reinterpret_cast<const VI *>(xh + col2);
            VO ou, ow;
#pragma unroll
            for (int e = 0; e < W; e++) {
                ou.v[e] = wr<TO>(rd(u.v[e]));
                ow.v[e] = wr<TO>(rd(w.v[e]));
            }
            if (turn) {
                if (HALVES || W == 1) {
#pragma unroll
                    for (int e = 0; e < W; e++) {
                        const float p0 = rd(u.v[e]), p1 = rd(w.v[e]);
                        ou.v[e] = wr<TO>(p0 * cs[e].x - p1 * cs[e].y);
                        ow.v[e] = wr<TO>(p0 * cs[e].y + p1 * cs[e].x);
                    }
                }
                else {
#pragma unroll
                    for (int e = 0; e + 1 < W; e += 2) {
                        const float p0 = rd(u.v[e]), p1 = rd(u.v[e + 1]);
                        ou.v[e] = wr<TO>(p0 * cs[e / 2].x - p1 * cs[e / 2].y);
                        ou.v[e + 1] = wr<TO>(p0 * cs[e / 2].y + p1 * cs[e / 2].x);
                    }
                }
            }
            *reinterpret_cast<VO *>(yh + col) = ou;
            if (two)
                *reinterpret_cast<VO *>(yh + col2) = ow;
        }
    }
}

template <typename TI, typename TO, int W, bool HALVES>
int launch(RotArgs &a, bool in_place, cudaStream_t s)
{
    const int rot = 2 * a.half;
    a.nrot = HALVES ? a.half / W : (W > 1 ? rot / W : a.half);
    a.nch = a.nrot + (in_place ? 0 : (a.hd - rot) / W);
    // Heads per thread: 4 when that leaves a few waves of threads.
    const long one = a.rows * a.heads * a.nch;
    const long fill = (long)device_sms() * 2048 * 2;
    a.hpt = one >= 4 * fill ? 4 : (one >= 2 * fill ? 2 : 1);
    a.nhg = (a.heads + a.hpt - 1) / a.hpt;
    const long total = a.rows * a.nhg * a.nch, blocks = (total + 255) / 256;
    return launch_pdl(rope_rotate_kernel<TI, TO, W, HALVES>,
                      dim3((unsigned)(blocks < 0x7fffffffL ? blocks : 0x7fffffffL)), dim3(256), 0, s,
                      (const RotArgs)a);
}

template <typename TI, typename TO>
int launch_w(RotArgs &a, int layout, bool in_place, cudaStream_t s)
{
    constexpr int W = 16 / sizeof(TI);
    const int rot = 2 * a.half;
    auto whole = [&](long v) { return v % W == 0; };
    const bool vec = whole(a.ldx) && whole(a.sx0) && whole(a.sx1) && whole(a.ldy) && whole(a.sy0) &&
                     whole(a.sy1) && whole(layout == K_ROPE_HALVES ? a.half : rot) &&
                     (in_place || whole(a.hd)) && !(reinterpret_cast<uintptr_t>(a.x) & 15) &&
                     reinterpret_cast<uintptr_t>(a.y) % (W * sizeof(TO)) == 0 &&
                     !(reinterpret_cast<uintptr_t>(a.cs) & 15);
    if (layout == K_ROPE_HALVES)
        return vec ? launch<TI, TO, W, true>(a, in_place, s) : launch<TI, TO, 1, true>(a, in_place, s);
    return vec ? launch<TI, TO, W, false>(a, in_place, s) : launch<TI, TO, 1, false>(a, in_place, s);
}

}  // namespace
}  // namespace sam3

extern "C" int k_rope_table(long npos, int rot, long first, const double *turns, float amp, float *cs,
                            k_stream s)
{
    using namespace sam3;
    if (npos <= 0 || rot <= 0 || (rot & 1) || rot > K_ROPE_MAX)
        return K_EARG;
    Freqs f;
    for (int j = 0; j < rot / 2; j++)
        f.t[j] = turns[j];
    for (int j = rot / 2; j < K_ROPE_MAX / 2; j++)
        f.t[j] = 0.0;
    const long n = npos * (rot / 2), blocks = (n + 255) / 256, most = (long)device_sms() * 8;
    return launch_pdl(rope_table_kernel, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0,
                      reinterpret_cast<cudaStream_t>(s), f, rot / 2, first, n, amp,
                      reinterpret_cast<float2 *>(cs));
}

extern "C" int k_rope_rotate(const struct k_rows *X, const struct k_rows *Y, int nb, int N, int heads,
                             int hd, int rot, int layout, const int *pos, int pos0, int npos,
                             const float *cs, k_stream s)
{
    using namespace sam3;
    if (nb <= 0 || N <= 0 || heads <= 0 || rot <= 0 || (rot & 1) || rot > hd)
        return K_EARG;
    RotArgs a = {};
    a.x = X->p;
    a.y = Y->p;
    a.ldx = X->ld;
    a.sx0 = X->s0;
    a.sx1 = X->s1;
    a.ldy = Y->ld;
    a.sy0 = Y->s0;
    a.sy1 = Y->s1;
    a.cs = reinterpret_cast<const float2 *>(cs);
    a.pos = pos;
    a.pos0 = pos0;
    a.npos = npos;
    a.N = N;
    a.rows = (long)nb * N;
    a.heads = heads;
    a.hd = hd;
    a.half = rot / 2;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(s);
    const bool in_place = X->p == Y->p;  // the caller has checked that the layouts agree
    if (X->dt == K_F32 && Y->dt == K_F32)
        return launch_w<float, float>(a, layout, in_place, st);
    if (X->dt == K_F32 && Y->dt == K_BF16)
        return launch_w<float, __nv_bfloat16>(a, layout, in_place, st);
    if (X->dt == K_F32 && Y->dt == K_F16)
        return launch_w<float, __half>(a, layout, in_place, st);
    if (X->dt == K_BF16 && Y->dt == K_BF16)
        return launch_w<__nv_bfloat16, __nv_bfloat16>(a, layout, in_place, st);
    if (X->dt == K_F16 && Y->dt == K_F16)
        return launch_w<__half, __half>(a, layout, in_place, st);
    return K_EARG;
}
