// SPDX-License-Identifier: Unlicense
// Rotary positions: tables of angles made on the device, and the rotation of
// rows by them. The table has the layout of cb_rope_apply: [npos, rot / 2]
// (cos, sin) pairs in fp32.
#include "div.cuh"
#include "kernels.h"
#include "pdl.cuh"
#include "tc_ptx.cuh"
#include "tmap.cuh"
#include "vec.cuh"

#include <cuda_runtime.h>

namespace sam3 {
namespace {

// cos and sin of the angle of `turns` turns. The turns are reduced to a
// quadrant q and a remainder in [-1/8, 1/8] in 64 bits, exactly; what far
// positions lose is the rounding of the turns, position times frequency in
// 64 bits (2^-21 of an angle at position 2^31); sine and cosine of the remainder's angle |x| <= pi / 4
// are their Taylor polynomials in 32 bits, the first terms left out being
// x^11 / 11! < 2e-9 and x^12 / 12! < 2e-10.
__device__ __forceinline__ float2 cos_sin_turns(double turns)
{
    const double kMagic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer
    const double m = fma(4.0, turns, kMagic);
    const int q = __double2loint(m);
    const float x = (float)fma(-0.25, m - kMagic, turns) * 6.2831853071795865f;
    const float z = x * x;
    float s = fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
    s = fmaf(s, z, 8.3333333e-3f);
    s = fmaf(s, z, -0.16666667f);
    s = fmaf(s * z, x, x);
    float c = fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
    c = fmaf(c, z, -1.3888889e-3f);
    c = fmaf(c, z, 4.1666667e-2f);
    c = fmaf(c, z, -0.5f);
    c = fmaf(c, z, 1.0f);
    const float c1 = (q & 1) ? s : c, s1 = (q & 1) ? c : s;
    return make_float2(__uint_as_float(__float_as_uint(c1) ^ ((uint32_t)(q + 1) << 30 & 0x80000000u)),
                       __uint_as_float(__float_as_uint(s1) ^ ((uint32_t)q << 30 & 0x80000000u)));
}

// Frequencies in turns per position, by value (captured graphs keep them).
struct Freqs {
    double t[K_ROPE_MAX / 2];
};

// A thread keeps one pair j (two adjacent ones when half is even) and steps over
// positions; a block's threads are adjacent entries of the table. Write bound:
// 131072 positions x 64 pairs in 13.2 us, 5.1 TB/s (63 us with a 64-bit division per entry
// and sincospif).
template <int PAIRS>
__global__ void __launch_bounds__(256) rope_table_kernel(const __grid_constant__ Freqs f, int half,
                                                         long first, int npos, float amp,
                                                         float2 *__restrict__ cs)
{
    const int width = half / PAIRS, rows = 256 / width;  // threads of a position, positions of a block
    const int row = threadIdx.x / width, j = (threadIdx.x - row * width) * PAIRS;
    griddep_wait();
    griddep_launch();
    if (row >= rows)
        return;
    double w[PAIRS];
#pragma unroll
    for (int i = 0; i < PAIRS; i++)
        w[i] = f.t[j + i];
    const int step = gridDim.x * rows;
    float2 *dst = cs + ((long)blockIdx.x * rows + row) * half + j;
    for (long p = (long)blockIdx.x * rows + row; p < npos; p += step, dst += (long)step * half) {
        const double pos = (double)(first + p);
        float2 v[PAIRS];
#pragma unroll
        for (int i = 0; i < PAIRS; i++) {
            v[i] = cos_sin_turns(pos * w[i]);
            v[i].x *= amp;
            v[i].y *= amp;
        }
        if constexpr (PAIRS == 2)
            *reinterpret_cast<float4 *>(dst) = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
        else
            *dst = v[0];
    }
}

struct RotArgs {
    const void *x;
    void *y;
    const float2 *cs;
    const int *pos;
    long ldx, sx0, sx1, ldy, sy0, sy1;  // elements: row, sequence and head strides
    uint32_t row0;                      // first row (of nb * N) of this launch
    uint32_t total;                     // threads with work, < 2^31
    int heads, half, pos0, npos;
    int nrot;             // rotated chunks of a head, the others are copied
    Div nch, nhg, N;      // chunks of a head, head groups of a row, rows of a sequence
};

// A value that is not turned: its bits where the types agree (a NaN keeps its
// payload), else rounded.
template <typename TO, typename TI>
__device__ __forceinline__ TO copied(TI v)
{
    if constexpr (__is_same(TI, TO))
        return v;
    else
        return from_f<TO>(to_f(v));
}

// A thread takes one chunk of W adjacent columns (HALVES: the W columns at j
// and the W at half + j) of up to hpt heads of one row, so that the chunk's
// (cos, sin) pairs are read once for all of them. W columns are 16 bytes of
// input, or 1 (a pair of columns 2 j, 2 j + 1 without HALVES) for rows that
// are not 16-byte aligned. Memory bound: X read and Y written once, the
// table rows from L2; 41472 rows of 24 heads of 64 bf16 columns 48 us, 5.3 TB/s
// (81 % of a copy). Indexes without divisions (56 us with 64-bit ones).
template <typename TI, typename TO, int W, bool HALVES>
__global__ void __launch_bounds__(256) rope_rotate_kernel(const __grid_constant__ RotArgs a)
{
    constexpr int CW = HALVES || W > 1 ? W : 2;     // columns of a vector
    constexpr int NP = HALVES ? W : CW / 2;         // pairs of a chunk
    using VI = Vec<TI, W>;
    using VO = Vec<TO, W>;
    griddep_wait();
    griddep_launch();
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i < a.total) {
        const uint32_t rg = quot(i, a.nch);
        const int c = (int)(i - rg * a.nch.d);
        const uint32_t rl = quot(rg, a.nhg);
        const int hg = (int)(rg - rl * a.nhg.d);
        const uint32_t row = a.row0 + rl;
        const long b = quot(row, a.N), n = row - (uint32_t)b * a.N.d;
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
        for (int h = hg; h < a.heads; h += a.nhg.d) {
            const TI *xh = x + h * a.sx1;
            TO *yh = y + h * a.sy1;
            const VI u = *reinterpret_cast<const VI *>(xh + col);
            VI w = u;
            if (two)
                w = *reinterpret_cast<const VI *>(xh + col2);
            VO ou, ow;
#pragma unroll
            for (int e = 0; e < W; e++) {
                ou.v[e] = copied<TO>(u.v[e]);
                ow.v[e] = copied<TO>(w.v[e]);
            }
            if (turn) {
                if (HALVES || W == 1) {
#pragma unroll
                    for (int e = 0; e < W; e++) {
                        const float p0 = to_f(u.v[e]), p1 = to_f(w.v[e]);
                        ou.v[e] = from_f<TO>(p0 * cs[e].x - p1 * cs[e].y);
                        ow.v[e] = from_f<TO>(p0 * cs[e].y + p1 * cs[e].x);
                    }
                }
                else {
#pragma unroll
                    for (int e = 0; e + 1 < W; e += 2) {
                        const float p0 = to_f(u.v[e]), p1 = to_f(u.v[e + 1]);
                        ou.v[e] = from_f<TO>(p0 * cs[e / 2].x - p1 * cs[e / 2].y);
                        ou.v[e + 1] = from_f<TO>(p0 * cs[e / 2].y + p1 * cs[e / 2].x);
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
int launch(RotArgs &a, long rows, int N, int hd, bool in_place, cudaStream_t s)
{
    const int rot = 2 * a.half;
    a.nrot = HALVES ? a.half / W : (W > 1 ? rot / W : a.half);
    const int nch = a.nrot + (in_place ? 0 : (hd - rot) / W);
    // Heads per thread: as many as leave a wave of threads (24 heads x 41472
    // rows of 64 columns: 58 us with 1, 49.5 with 2, 48.0 with 4, 51.1 with 8).
    const double one = (double)rows * a.heads * nch;
    const double fill = (double)device_sms() * 2048 * 2;
    const int hpt = one >= 2 * fill ? 4 : (one >= fill ? 2 : 1);
    const int nhg = (a.heads + hpt - 1) / hpt;
    a.nch = make_div(nch);
    a.nhg = make_div(nhg);
    a.N = make_div(N);
    // one launch up to 2^31 - 256 threads, which only larger tensors pass
    const long most = 0x7fffff00L / ((long)nch * nhg);
    if (most < 1 || rows > 0x7fffffffL)
        return K_EARG;
    for (long r = 0; r < rows; r += most) {
        const long n = rows - r < most ? rows - r : most;
        a.row0 = (uint32_t)r;
        a.total = (uint32_t)(n * nch * nhg);
        const int rc = launch_pdl(rope_rotate_kernel<TI, TO, W, HALVES>, dim3((a.total + 255) / 256), dim3(256),
                                  0, s, (const RotArgs)a);
        if (rc)
            return rc;
    }
    return 0;
}

template <typename TI, typename TO>
int launch_w(RotArgs &a, long rows, int N, int hd, int layout, bool in_place, cudaStream_t s)
{
    constexpr int W = 16 / sizeof(TI);
    const int rot = 2 * a.half;
    auto whole = [&](long v) { return v % W == 0; };
    const bool vec = whole(a.ldx) && whole(a.sx0) && whole(a.sx1) && whole(a.ldy) && whole(a.sy0) &&
                     whole(a.sy1) && whole(layout == K_ROPE_HALVES ? a.half : rot) &&
                     (in_place || whole(hd)) && !(reinterpret_cast<uintptr_t>(a.x) & 15) &&
                     reinterpret_cast<uintptr_t>(a.y) % (W * sizeof(TO)) == 0 &&
                     !(reinterpret_cast<uintptr_t>(a.cs) & 15);
    if (layout == K_ROPE_HALVES)
        return vec ? launch<TI, TO, W, true>(a, rows, N, hd, in_place, s) : launch<TI, TO, 1, true>(a, rows, N, hd, in_place, s);
    return vec ? launch<TI, TO, W, false>(a, rows, N, hd, in_place, s) : launch<TI, TO, 1, false>(a, rows, N, hd, in_place, s);
}

}  // namespace
}  // namespace sam3

extern "C" int k_rope_table(int npos, int rot, long first, const double *turns, float amp, float *cs,
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
    const int half = rot / 2, pairs = half % 2 == 0 && !(reinterpret_cast<uintptr_t>(cs) & 15) ? 2 : 1;
    const int rows = 256 / (half / pairs);
    const long blocks = ((long)npos + rows - 1) / rows, most = (long)device_sms() * 8;
    const dim3 grid((unsigned)(blocks < most ? blocks : most));
    cudaStream_t st = reinterpret_cast<cudaStream_t>(s);
    return pairs == 2 ? launch_pdl(rope_table_kernel<2>, grid, dim3(256), 0, st, f, half, first, npos, amp,
                                   reinterpret_cast<float2 *>(cs))
                      : launch_pdl(rope_table_kernel<1>, grid, dim3(256), 0, st, f, half, first, npos, amp,
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
    a.heads = heads;
    a.half = rot / 2;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(s);
    const bool in_place = X->p == Y->p;  // the caller has checked that the layouts agree
    if (X->dt == K_F32 && Y->dt == K_F32)
        return launch_w<float, float>(a, (long)nb * N, N, hd, layout, in_place, st);
    if (X->dt == K_F32 && Y->dt == K_BF16)
        return launch_w<float, __nv_bfloat16>(a, (long)nb * N, N, hd, layout, in_place, st);
    if (X->dt == K_F32 && Y->dt == K_F16)
        return launch_w<float, __half>(a, (long)nb * N, N, hd, layout, in_place, st);
    if (X->dt == K_BF16 && Y->dt == K_BF16)
        return launch_w<__nv_bfloat16, __nv_bfloat16>(a, (long)nb * N, N, hd, layout, in_place, st);
    if (X->dt == K_F16 && Y->dt == K_F16)
        return launch_w<__half, __half>(a, (long)nb * N, N, hd, layout, in_place, st);
    return K_EARG;
}
