// SPDX-License-Identifier: Unlicense
// E4M3 with a power-of-two scale per block: 1 x 128 values of a row (a half-warp
// holds it in registers, eight values a lane, its largest magnitude by four
// shuffles; a warp where rows are not aligned) or 128 x 128 (a CTA holds it, 64 values a thread). One pass: X read
// and Q written once. Memory bound: 41472 x 4096 bf16 values by rows 90 to 99 us,
// 5.2 to 5.7 TB/s.
#include "div.cuh"
#include "e4m3.cuh"
#include "kernels.h"
#include "pdl.cuh"
#include "tmap.cuh"
#include "vec8.cuh"

#include <type_traits>

namespace sam3 {
namespace {

constexpr int kThreads = 256;

struct QuantArgs {
    k_rows x, q, s;
    long total;   // units of work: a warp's stretch of a row, or a CTA's block
    int N, K, kb;
    int small;    // total < 2^31
    Div dkb, dN;  // stretches of a row, rows (or row blocks) of a sequence
};

template <bool FINITE, int C>
__device__ __forceinline__ float largest_of(const float (&v)[C])
{
    float m = 0.0f;
#pragma unroll
    for (int e = 0; e < C; e++)
        m = FINITE ? larger_finite(m, v[e]) : larger(m, v[e]);
    return m;
}

// Of the block's half-warp.
template <bool FINITE>
__device__ __forceinline__ float largest_row(const float (&v)[8])
{
    float m = largest_of<FINITE>(v);
#pragma unroll
    for (int o = 8; o; o >>= 1)
        m = fmaxf(m, __shfl_xor_sync(0xffffu << (threadIdx.x & 16), m, o, 16));
    return m;
}

// Of the CTA; every thread gets it.
template <bool FINITE, int S, int C>
__device__ __forceinline__ float largest_tile(const float (&v)[S][C], float *smem)
{
    float m = 0.0f;
#pragma unroll
    for (int k = 0; k < S; k++)
        m = fmaxf(m, largest_of<FINITE>(v[k]));
#pragma unroll
    for (int o = 16; o; o >>= 1)
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    __syncthreads();  // the last values have been read
    if ((threadIdx.x & 31) == 0)
        smem[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 32; w++)
        m = fmaxf(m, smem[w]);
    return m;
}

// Four values of a lane, 32 columns apart, n columns left of the row.
__device__ __forceinline__ void put4(const QuantArgs &a, long q, int n, const float (&v)[4], float inv, bool inf)
{
    const uint32_t w = inf ? pack_e4m3<true>(v[0], v[1], v[2], v[3], inv) : pack_e4m3<false>(v[0], v[1], v[2], v[3], inv);
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (32 * e < n)
            reinterpret_cast<uint8_t *>(a.q.p)[q + 32 * e] = (uint8_t)(w >> (8 * e));
}

// A warp takes U pairs of neighbouring blocks of a row at a time, their loads in
// flight together; DT: X's type. Rows that are not aligned (VEC false): every lane
// takes every 32nd column, so that an access covers adjacent elements, and the warp
// one block after the other.
template <int DT, bool VEC, int U>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const __grid_constant__ QuantArgs a)
{
    griddep_wait();
    griddep_launch();
    const int lane = threadIdx.x & 31;
    const long step = (long)gridDim.x * (kThreads / 32);
    for (long i = (long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); i < a.total; i += step) {
        const long rowi = a.small ? (long)quot((uint32_t)i, a.dkb) : i / a.dkb.d;
        const int c0 = (int)(i - rowi * a.dkb.d) * (256 * U) + lane * (VEC ? 8 : 1);
        const long b = quot((uint32_t)rowi, a.dN), r = rowi - b * a.N;
        const long x = b * a.x.s0 + r * a.x.ld + c0, q = b * a.q.s0 + r * a.q.ld + c0;
        const long s = b * a.s.s0 + r * a.s.ld + c0 / kScaleBlock;
        const int n = a.K - c0;
        if constexpr (VEC) {
            Raw8 raw[U];
#pragma unroll
            for (int k = 0; k < U; k++)
                raw[k] = load8<true>(a.x.p, DT, x + 256 * k, n - 256 * k);
#pragma unroll
            for (int k = 0; k < U; k++) {
                float v[8];
                unpack8(raw[k], DT, v);
                float m = largest_row<false>(v);
                const bool inf = infinite(m);
                if (inf)
                    m = largest_row<true>(v);
                const uint32_t byte = scale_byte(m);
                if (n - 256 * k > 0) {
                    store8_e4m3<true>(a.q.p, q + 256 * k, n - 256 * k, pack8_e4m3(v, scale_inverse(byte), inf));
                    if ((lane & 15) == 0)
                        put_scale(a.s.p, a.s.dt, s + 2 * k, byte);
                }
            }
        }
        else {
            float v[2 * U][4];
#pragma unroll
            for (int k = 0; k < 2 * U; k++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    v[k][e] = 128 * k + 32 * e < n ? elem(a.x.p, DT, x + 128 * k + 32 * e) : 0.0f;
#pragma unroll
            for (int k = 0; k < 2 * U; k++) {
                auto largest = [&](bool finite) {
                    float m = 0.0f;
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        m = finite ? larger_finite(m, v[k][e]) : larger(m, v[k][e]);
#pragma unroll
                    for (int o = 16; o; o >>= 1)
                        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                    return m;
                };
                float m = largest(false);
                const bool inf = infinite(m);
                if (inf)
                    m = largest(true);
                const uint32_t byte = scale_byte(m);
                put4(a, q + 128 * k, n - 128 * k, v[k], scale_inverse(byte), inf);
                if (lane == 0 && n - 128 * k > 0)
                    put_scale(a.s.p, a.s.dt, s + k, byte);
            }
        }
    }
}

// A CTA takes a block of 128 x 128; its values stay in registers.
template <int DT, bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_tiles_kernel(const __grid_constant__ QuantArgs a)
{
    constexpr int C = VEC ? 8 : 4, L = kScaleBlock / C;     // columns of a thread, threads of a row
    constexpr int R = kThreads / L, S = kScaleBlock / R;    // rows of a step, steps
    __shared__ float largest[kThreads / 32];
    griddep_wait();
    griddep_launch();
    const int sub = threadIdx.x & (L - 1), r0 = threadIdx.x / L;
    for (long i = blockIdx.x; i < a.total; i += gridDim.x) {
        const long t = i / a.kb;
        const int kb = (int)(i - t * a.kb);
        const long b = quot((uint32_t)t, a.dN);
        const int nb = (int)(t - b * a.dN.d), c = kb * kScaleBlock + sub * (VEC ? 8 : 1);
        float v[S][C];
#pragma unroll
        for (int k = 0; k < S; k++) {
            const int n = nb * kScaleBlock + k * R + r0;
            const long x = b * a.x.s0 + n * a.x.ld + c;
            if constexpr (VEC)
                unpack8(load8<true>(a.x.p, DT, x, n < a.N ? a.K - c : 0), DT, v[k]);
            else {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    v[k][e] = n < a.N && c + 32 * e < a.K ? elem(a.x.p, DT, x + 32 * e) : 0.0f;
            }
        }
        float m = largest_tile<false>(v, largest);
        const bool inf = infinite(m);
        if (inf)
            m = largest_tile<true>(v, largest);
        const uint32_t byte = scale_byte(m);
        const float inv = scale_inverse(byte);
#pragma unroll
        for (int k = 0; k < S; k++) {
            const int n = nb * kScaleBlock + k * R + r0;
            const long q = b * a.q.s0 + n * a.q.ld + c;
            if (n >= a.N)
                continue;
            if constexpr (VEC)
                store8_e4m3<true>(a.q.p, q, a.K - c, pack8_e4m3(v[k], inv, inf));
            else
                put4(a, q, a.K - c, v[k], inv, inf);
        }
        if (threadIdx.x == 0)
            put_scale(a.s.p, a.s.dt, b * a.s.s0 + (long)nb * a.s.ld + kb, byte);
    }
}

// go(the element type as a constant).
template <typename F>
int by_type(int dt, const F &go)
{
    if (dt == K_F32)
        return go(std::integral_constant<int, K_F32>{});
    return dt == K_BF16 ? go(std::integral_constant<int, K_BF16>{}) : go(std::integral_constant<int, K_F16>{});
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
    const bool vec = rows_vec8(a.x) && rows_vec8(a.q);
    const int sms = device_sms();
    cudaStream_t st = reinterpret_cast<cudaStream_t>(s);
    if (brows == 1) {
        // Pairs of blocks a warp has in flight: four, where that still leaves
        // every SM sixteen warps.
        const long pairs = (a.kb + 1) / 2, rows = (long)nb * N;
        const int u = pairs >= 3 && rows * ((pairs + 3) / 4) >= (long)sms * 16 ? 4 : 1;
        a.dN = make_div(N);
        a.dkb = make_div((uint32_t)((pairs + u - 1) / u));
        a.total = rows * a.dkb.d;
        a.small = a.total < (1L << 31);
        const long need = (a.total + kThreads / 32 - 1) / (kThreads / 32), most = (long)sms * 64;
        const dim3 grid((unsigned)(need < most ? need : most));
        return by_type(X->dt, [&](auto dt) {
            constexpr int DT = decltype(dt)::value;
            if (u == 4)
                return vec ? launch_pdl(quantize_rows_kernel<DT, true, 4>, grid, dim3(kThreads), 0, st, (const QuantArgs)a)
                           : launch_pdl(quantize_rows_kernel<DT, false, 4>, grid, dim3(kThreads), 0, st, (const QuantArgs)a);
            return vec ? launch_pdl(quantize_rows_kernel<DT, true, 1>, grid, dim3(kThreads), 0, st, (const QuantArgs)a)
                       : launch_pdl(quantize_rows_kernel<DT, false, 1>, grid, dim3(kThreads), 0, st, (const QuantArgs)a);
        });
    }
    a.dN = make_div(N / kScaleBlock + (N % kScaleBlock != 0));
    a.total = (long)nb * a.dN.d * a.kb;
    const long most = (long)sms * 64;
    const dim3 grid((unsigned)(a.total < most ? a.total : most));
    return by_type(X->dt, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        return vec ? launch_pdl(quantize_tiles_kernel<DT, true>, grid, dim3(kThreads), 0, st, (const QuantArgs)a)
                   : launch_pdl(quantize_tiles_kernel<DT, false>, grid, dim3(kThreads), 0, st, (const QuantArgs)a);
    });
}
