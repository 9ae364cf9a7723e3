// SPDX-License-Identifier: Unlicense
// E4M3 with a power-of-two scale per block: 1 x 128 values of a row (a half-warp
// holds it in registers, eight values a lane, its largest magnitude by four
// shuffles) or 128 x 128 (a CTA holds it, 64 values a thread). One pass: X read
// and Q written once. Memory bound.
#include "div.cuh"
#include "e4m3.cuh"
#include "kernels.h"
#include "pdl.cuh"
#include "tmap.cuh"
#include "vec8.cuh"

namespace sam3 {
namespace {

constexpr int kThreads = 256;

struct QuantArgs {
    k_rows x, q, s;
    long total;  // blocks
    int N, K, kb;
    Div dkb, dN;  // blocks of a row, rows (or row blocks) of a sequence
};

__device__ __forceinline__ uint32_t largest8(const float (&v)[8])
{
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; e++)
        m = max(m, finite_bits(v[e]));
    return m;
}

template <bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const __grid_constant__ QuantArgs a)
{
    griddep_wait();
    griddep_launch();
    const int sub = threadIdx.x & 15;
    const long step = (long)gridDim.x * (kThreads / 16);
    for (long i = (long)blockIdx.x * (kThreads / 16) + (threadIdx.x >> 4); i < a.total; i += step) {
        const long rowi = i / a.kb;
        const int kb = (int)(i - rowi * a.kb);
        const long b = quot((uint32_t)rowi, a.dN), n = rowi - b * a.N;
        const int c = kb * kScaleBlock + sub * 8;
        float v[8];
        unpack8(load8<VEC>(a.x.p, a.x.dt, b * a.x.s0 + n * a.x.ld + c, a.K - c), a.x.dt, v);
        uint32_t m = largest8(v);
#pragma unroll
        for (int o = 8; o; o >>= 1)
            m = max(m, __shfl_xor_sync(0xffffu << (threadIdx.x & 16), m, o, 16));
        const uint32_t byte = scale_byte(m);
        const float inv = scale_inverse(byte);
        store8_e4m3<VEC>(a.q.p, b * a.q.s0 + n * a.q.ld + c, a.K - c, pack_e4m3(v[0], v[1], v[2], v[3], inv),
                         pack_e4m3(v[4], v[5], v[6], v[7], inv));
        if (sub == 0)
            put_scale(a.s.p, a.s.dt, b * a.s.s0 + n * a.s.ld + kb, byte);
    }
}

template <bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_tiles_kernel(const __grid_constant__ QuantArgs a)
{
    constexpr int R = kThreads / 16, S = kScaleBlock / R;  // rows of a step, steps
    __shared__ uint32_t largest[kThreads / 32];
    griddep_wait();
    griddep_launch();
    const int sub = threadIdx.x & 15, r0 = threadIdx.x >> 4;
    for (long i = blockIdx.x; i < a.total; i += gridDim.x) {
        const long t = i / a.kb;
        const int kb = (int)(i - t * a.kb);
        const long b = quot((uint32_t)t, a.dN);
        const int nb = (int)(t - b * a.dN.d), c = kb * kScaleBlock + sub * 8;
        float v[S][8];
        uint32_t m = 0;
#pragma unroll
        for (int k = 0; k < S; k++) {
            const int n = nb * kScaleBlock + k * R + r0;
            unpack8(load8<VEC>(a.x.p, a.x.dt, b * a.x.s0 + n * a.x.ld + c, n < a.N ? a.K - c : 0), a.x.dt, v[k]);
        }
#pragma unroll
        for (int k = 0; k < S; k++)
            m = max(m, largest8(v[k]));
        m = __reduce_max_sync(0xffffffffu, m);
        if ((threadIdx.x & 31) == 0)
            largest[threadIdx.x >> 5] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kThreads / 32; w++)
            m = max(m, largest[w]);
        const uint32_t byte = scale_byte(m);
        const float inv = scale_inverse(byte);
#pragma unroll
        for (int k = 0; k < S; k++) {
            const int n = nb * kScaleBlock + k * R + r0;
            if (n < a.N)
                store8_e4m3<VEC>(a.q.p, b * a.q.s0 + n * a.q.ld + c, a.K - c,
                                 pack_e4m3(v[k][0], v[k][1], v[k][2], v[k][3], inv),
                                 pack_e4m3(v[k][4], v[k][5], v[k][6], v[k][7], inv));
        }
        if (threadIdx.x == 0)
            put_scale(a.s.p, a.s.dt, b * a.s.s0 + (long)nb * a.s.ld + kb, byte);
        __syncthreads();  // largest[] is read before the next block's is written
    }
}

}  // namespace
}  // namespace sam3

extern "C" int k_quantize_e4m3(const struct k_rows *X, const struct k_rows *Q, const struct k_rows *S, int nb,
                               int N, int K, int brows, k_stream s)
{
    using namespace sam3;
    if (nb <= 0 || N <= 0 || K <= 0 || (brows != 1 && brows != kScaleBlock))
        return K_EARG;
    QuantArgs a = {};
    a.x = *X;
    a.q = *Q;
    a.s = *S;
    a.N = N;
    a.K = K;
    a.kb = K / kScaleBlock + (K % kScaleBlock != 0);
    const int nrow = brows == 1 ? N : N / kScaleBlock + (N % kScaleBlock != 0);
    a.dN = make_div(nrow);
    a.total = (long)nb * nrow * a.kb;
    const bool vec = rows_vec8(a.x) && rows_vec8(a.q);
    const long each = brows == 1 ? kThreads / 16 : 1, need = (a.total + each - 1) / each;
    const long most = (long)device_sms() * (brows == 1 ? 64 : 16);
    const dim3 grid((unsigned)(need < most ? need : most));
    cudaStream_t st = reinterpret_cast<cudaStream_t>(s);
    if (brows == 1)
        return vec ? launch_pdl(quantize_rows_kernel<true>, grid, dim3(kThreads), 0, st, (const QuantArgs)a)
                   : launch_pdl(quantize_rows_kernel<false>, grid, dim3(kThreads), 0, st, (const QuantArgs)a);
    return vec ? launch_pdl(quantize_tiles_kernel<true>, grid, dim3(kThreads), 0, st, (const QuantArgs)a)
               : launch_pdl(quantize_tiles_kernel<false>, grid, dim3(kThreads), 0, st, (const QuantArgs)a);
}
