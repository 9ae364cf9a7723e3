// SPDX-License-Identifier: Unlicense
// What stands between two blocks of a transformer, one pass over the residual
// stream: h = post(H), r = X + alpha ls gate h, R = r, Y = pre(r) (1 + scale) +
// shift, in 32 bits; Y rounded to its type or quantised to E4M3 (blocks of 128
// columns are the 16 lanes of a half-warp, eight adjacent columns a lane). Memory
// bound: X and H read, R and Y written once.
//
// T threads hold a row in registers, 8 V columns a thread, so that mean and
// variance are two sums over values at hand (no E[x^2] - E[x]^2); rows wider than
// that (V = 0) are read again for each sum, from L2.
#include "div.cuh"
#include "e4m3.cuh"
#include "kernels.h"
#include "pdl.cuh"
#include "tmap.cuh"
#include "vec8.cuh"

namespace sam3 {
namespace {

struct NormArgs {
    k_norm_args p;
    Div dN;
    long rows;
    float share;  // 1 / C
};

// Sum over the T threads of a row in a fixed order; every thread gets it. A row of
// more than one warp is a CTA.
template <int T>
__device__ __forceinline__ float row_sum(float v, float *smem)
{
#pragma unroll
    for (int o = 16; o; o >>= 1)
        v += __shfl_xor_sync(0xffffffffu, v, o);
    if constexpr (T > 32) {
        __syncthreads();
        if ((threadIdx.x & 31) == 0)
            smem[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < T / 32; w++)
            v += smem[w];
    }
    return v;
}

// Where a thread's columns of row (b, n) lie.
struct At {
    long x, h, gate, r, scale, shift, y, s;
};
__device__ __forceinline__ long at_row(const k_rows &k, long b, long n)
{
    return b * k.s0 + n * k.ld;
}

// v * g + b of a norm's parameters (NULL: 1, 0).
__device__ __forceinline__ void affine8(const k_norm &k, int c, int n, float mean, float rstd, float (&v)[8])
{
#pragma unroll
    for (int e = 0; e < 8; e++) {
        v[e] = (v[e] - mean) * rstd;
        if (e < n) {
            const float g = k.g ? __ldg(k.g + c + e) : 1.0f;
            v[e] = k.b ? fmaf(v[e], g, __ldg(k.b + c + e)) : v[e] * g;
        }
    }
}

// r of eight columns from x and the (normalised) h.
template <bool VEC>
__device__ __forceinline__ void join8(const k_norm_args &p, const At &at, int c, int n, const float (&x)[8],
                                      float (&h)[8], float (&r)[8])
{
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; e++)
        f[e] = p.alpha;
    if (p.ls) {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (e < n)
                f[e] *= __ldg(p.ls + c + e);
    }
    if (p.gate.p) {
        float g[8];
        unpack8(load8<VEC>(p.gate.p, p.gate.dt, at.gate + c, n), p.gate.dt, g);
#pragma unroll
        for (int e = 0; e < 8; e++)
            f[e] *= g[e];
    }
#pragma unroll
    for (int e = 0; e < 8; e++)
        r[e] = fmaf(f[e], h[e], x[e]);
}

// Y of eight columns of r.
template <bool VEC>
__device__ __forceinline__ void out8(const k_norm_args &p, const At &at, int c, int n, float mean, float rstd,
                                     float (&v)[8])
{
    if (p.pre.kind != K_NORM_NONE)
        affine8(p.pre, c, n, mean, rstd, v);
    if (p.scale.p) {
        float m[8];
        unpack8(load8<VEC>(p.scale.p, p.scale.dt, at.scale + c, n), p.scale.dt, m);
#pragma unroll
        for (int e = 0; e < 8; e++)
            v[e] = fmaf(v[e], m[e], v[e]);
    }
    if (p.shift.p) {
        float m[8];
        unpack8(load8<VEC>(p.shift.p, p.shift.dt, at.shift + c, n), p.shift.dt, m);
#pragma unroll
        for (int e = 0; e < 8; e++)
            v[e] += m[e];
    }
    if (p.Y.dt != K_E4M3) {
        if (n > 0)
            store8<VEC>(p.Y.p, p.Y.dt, at.y + c, n, v);
        return;
    }
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; e++)
        if (e < n)
            m = max(m, finite_bits(v[e]));
#pragma unroll
    for (int o = 8; o; o >>= 1)
        m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const uint32_t byte = scale_byte(m);
    const float inv = scale_inverse(byte);
    store8_e4m3<VEC>(p.Y.p, at.y + c, n, pack_e4m3(v[0], v[1], v[2], v[3], inv),
                     pack_e4m3(v[4], v[5], v[6], v[7], inv));
    if ((threadIdx.x & 15) == 0 && n > 0)
        put_scale(p.S.p, p.S.dt, at.s + c / kScaleBlock, byte);
}

// Mean (0 for RMS) and 1 / sqrt(variance + eps) of values v (n[j] of each eight
// valid) held by the row's threads.
template <int T, int V>
__device__ __forceinline__ void stats(const k_norm &k, const float (&v)[V][8], const int (&n)[V], float share, float *smem,
                                      float &mean, float &rstd)
{
    mean = 0.0f;
    if (k.kind == K_NORM_LAYER) {
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < V; j++)
#pragma unroll
            for (int e = 0; e < 8; e++)
                s += e < n[j] ? v[j][e] : 0.0f;
        mean = row_sum<T>(s, smem) * share;
    }
    float q = 0.0f;
#pragma unroll
    for (int j = 0; j < V; j++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float d = v[j][e] - mean;
            q = e < n[j] ? fmaf(d, d, q) : q;
        }
    rstd = rsqrtf(fmaf(row_sum<T>(q, smem), share, k.eps));
}

template <int T, int V, bool VEC>
__global__ void __launch_bounds__(T == 32 ? 256 : T) norm_rows_kernel(const __grid_constant__ NormArgs a)
{
    constexpr int kRows = T == 32 ? 8 : 1;  // rows of a CTA
    __shared__ float smem[32];
    const k_norm_args &p = a.p;
    const int lane = T == 32 ? threadIdx.x & 31 : threadIdx.x;
    griddep_wait();
    griddep_launch();
    for (long row = (long)blockIdx.x * kRows + (T == 32 ? threadIdx.x >> 5 : 0); row < a.rows;
         row += (long)gridDim.x * kRows) {
        const long b = quot((uint32_t)row, a.dN), nn = row - b * p.N;
        const At at = {at_row(p.X, b, nn), at_row(p.H, b, nn), at_row(p.gate, b, nn), at_row(p.R, b, nn),
                       at_row(p.scale, b, nn), at_row(p.shift, b, nn), at_row(p.Y, b, nn), at_row(p.S, b, nn)};
        Raw8 xr[V], hr[V];
        int n[V];
#pragma unroll
        for (int j = 0; j < V; j++) {
            n[j] = p.C - (j * T + lane) * 8;
            xr[j] = load8<VEC>(p.X.p, p.X.dt, at.x + (j * T + lane) * 8, n[j]);
        }
        if (p.H.p) {
#pragma unroll
            for (int j = 0; j < V; j++)
                hr[j] = load8<VEC>(p.H.p, p.H.dt, at.h + (j * T + lane) * 8, n[j]);
        }
        float r[V][8], mean = 0.0f, rstd = 1.0f;
        if (p.H.p) {
            float h[V][8];
#pragma unroll
            for (int j = 0; j < V; j++)
                unpack8(hr[j], p.H.dt, h[j]);
            if (p.post.kind != K_NORM_NONE) {
                stats<T, V>(p.post, h, n, a.share, smem, mean, rstd);
#pragma unroll
                for (int j = 0; j < V; j++)
                    affine8(p.post, (j * T + lane) * 8, n[j], mean, rstd, h[j]);
            }
#pragma unroll
            for (int j = 0; j < V; j++) {
                float x[8];
                unpack8(xr[j], p.X.dt, x);
                join8<VEC>(p, at, (j * T + lane) * 8, n[j], x, h[j], r[j]);
            }
        }
        else {
#pragma unroll
            for (int j = 0; j < V; j++)
                unpack8(xr[j], p.X.dt, r[j]);
        }
        if (p.R.p) {
#pragma unroll
            for (int j = 0; j < V; j++)
                store8<VEC>(p.R.p, p.R.dt, at.r + (j * T + lane) * 8, n[j], r[j]);
        }
        if (!p.Y.p)
            continue;
        if (p.pre.kind != K_NORM_NONE)
            stats<T, V>(p.pre, r, n, a.share, smem, mean, rstd);
#pragma unroll
        for (int j = 0; j < V; j++)
            out8<VEC>(p, at, (j * T + lane) * 8, n[j], mean, rstd, r[j]);
    }
}

// Rows of any width: each sum and the result read the row again.
template <int T, bool VEC>
__global__ void __launch_bounds__(T) norm_wide_kernel(const __grid_constant__ NormArgs a)
{
    __shared__ float smem[32];
    const k_norm_args &p = a.p;
    griddep_wait();
    griddep_launch();
    for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const long b = quot((uint32_t)row, a.dN), nn = row - b * p.N;
        const At at = {at_row(p.X, b, nn), at_row(p.H, b, nn), at_row(p.gate, b, nn), at_row(p.R, b, nn),
                       at_row(p.scale, b, nn), at_row(p.shift, b, nn), at_row(p.Y, b, nn), at_row(p.S, b, nn)};
        float hm = 0.0f, hs = 1.0f, mean = 0.0f, rstd = 1.0f;
        auto value = [&](int c, int n, bool joined, float (&v)[8]) {
            if (!joined || p.H.p)
                unpack8(load8<VEC>(p.H.p, p.H.dt, at.h + c, n), p.H.dt, v);
            if (!joined)
                return;
            float x[8];
            unpack8(load8<VEC>(p.X.p, p.X.dt, at.x + c, n), p.X.dt, x);
            if (!p.H.p) {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    v[e] = x[e];
                return;
            }
            float h[8];
#pragma unroll
            for (int e = 0; e < 8; e++)
                h[e] = v[e];
            if (p.post.kind != K_NORM_NONE)
                affine8(p.post, c, n, hm, hs, h);
            join8<VEC>(p, at, c, n, x, h, v);
        };
        auto sums = [&](const k_norm &k, bool joined, float &m, float &rs) {
            m = 0.0f;
            if (k.kind == K_NORM_LAYER) {
                float s = 0.0f;
                for (int c = threadIdx.x * 8; c < p.C; c += T * 8) {
                    float v[8];
                    value(c, p.C - c, joined, v);
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        s += e < p.C - c ? v[e] : 0.0f;
                }
                m = row_sum<T>(s, smem) * a.share;
            }
            float q = 0.0f;
            for (int c = threadIdx.x * 8; c < p.C; c += T * 8) {
                float v[8];
                value(c, p.C - c, joined, v);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float d = v[e] - m;
                    q = e < p.C - c ? fmaf(d, d, q) : q;
                }
            }
            rs = rsqrtf(fmaf(row_sum<T>(q, smem), a.share, k.eps));
        };
        if (p.H.p && p.post.kind != K_NORM_NONE)
            sums(p.post, false, hm, hs);
        if (p.Y.p && p.pre.kind != K_NORM_NONE)
            sums(p.pre, true, mean, rstd);
        // whole half-warps for the E4M3 blocks
        for (int c0 = 0; c0 < p.C; c0 += T * 8) {
            const int c = c0 + threadIdx.x * 8, n = p.C - c;
            float v[8];
            value(c, n, true, v);
            if (p.R.p)
                store8<VEC>(p.R.p, p.R.dt, at.r + c, n, v);
            if (p.Y.p)
                out8<VEC>(p, at, c, n, mean, rstd, v);
        }
    }
}

template <int T, int V>
int launch(const NormArgs &a, bool vec, cudaStream_t st)
{
    const long per = T == 32 ? 8 : 1, need = (a.rows + per - 1) / per, most = (long)device_sms() * 16;
    const dim3 grid((unsigned)(need < most ? need : most)), block(T == 32 ? 256 : T);
    return vec ? launch_pdl(norm_rows_kernel<T, V, true>, grid, block, 0, st, a)
               : launch_pdl(norm_rows_kernel<T, V, false>, grid, block, 0, st, a);
}

}  // namespace
}  // namespace sam3

extern "C" int k_norm_residual(const struct k_norm_args *p, k_stream s)
{
    using namespace sam3;
    if (p->nb <= 0 || p->N <= 0 || p->C <= 0)
        return K_EARG;
    NormArgs a = {};
    a.p = *p;
    a.dN = make_div(p->N);
    a.rows = (long)p->nb * p->N;
    a.share = 1.0f / (float)p->C;
    const bool vec = rows_vec8(p->X) && rows_vec8(p->H) && rows_vec8(p->gate) && rows_vec8(p->R) &&
                     rows_vec8(p->scale) && rows_vec8(p->shift) && rows_vec8(p->Y);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(s);
    const int v = (p->C + 7) / 8;  // vectors of eight of a row
    if (v <= 32)
        return launch<32, 1>(a, vec, st);
    if (v <= 64)
        return launch<32, 2>(a, vec, st);
    if (v <= 128)
        return launch<32, 4>(a, vec, st);
    if (v <= 256)
        return launch<128, 2>(a, vec, st);
    if (v <= 512)
        return launch<128, 4>(a, vec, st);
    if (v <= 1024)
        return launch<256, 4>(a, vec, st);
    const long most = (long)device_sms() * 2;
    const dim3 grid((unsigned)(a.rows < most ? a.rows : most));
    return vec ? launch_pdl(norm_wide_kernel<1024, true>, grid, dim3(1024), 0, st, (const NormArgs)a)
               : launch_pdl(norm_wide_kernel<1024, false>, grid, dim3(1024), 0, st, (const NormArgs)a);
}
