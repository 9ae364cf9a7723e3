// SPDX-License-Identifier: Unlicense
// Group norm with an activation over channels-last maps (the detector's
// pixel decoder, sam3_kernels.cl:926-953, for any batch, type and group
// width): y = act((x - mean) rstd gamma[c] + beta[c]) with mean and variance
// of each sample's group of channels over all pixels.
//
// One launch, no workspace. A unit is (sample, slab), a slab the fewest
// whole groups whose channels fill kSlabBytes of a pixel's row, so that a
// warp reads whole 32-byte sectors although it reads part of each row. A
// cluster of 1 to 16 CTAs shares a unit's pixels: each CTA reads its share
// once, keeping what fits of it in shared memory, the CTAs exchange
// (count, mean, M2) per group through distributed shared memory, and the
// second pass takes the kept part from shared memory and re-reads the rest,
// latest first (L2 still holds it when the map in flight is not far larger).
//
// Statistics in fp32 without the cancellation of E[x^2] - E[x]^2: a thread
// reduces kUnroll vectors at a time to their own mean and M2 = sum (x -
// mean)^2 and merges these into its running pair (mean += d f, M2 += M2' + d^2
// n f, d = mean' - mean, f = n' / (n + n'); Chan, Golub and LeVeque 1979);
// threads and CTAs are merged by sum n_i mean_i / n and sum M2_i + n_i
// (mean_i - mean)^2 in a fixed order, so a result does not depend on timing.
#include "kernels.h"
#include "pdl.cuh"
#include "tc_ptx.cuh"
#include "tmap.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace sam3 {
namespace {

constexpr int kThreads = 512;
constexpr int kUnroll = 4;
constexpr int kSlabBytes = 64;
constexpr int kMaxSlabGroups = 128;
constexpr int kMaxCluster = 16;
constexpr int kCacheBytes = 96 * 1024;  // per CTA; two CTAs share an SM

struct GnArgs {
    const void *x;
    void *y;
    const float *g, *b;
    long ldx, sx, ldy, sy;  // elements: pixel and sample strides
    long npix;
    int cg, gps, S, nslab;  // group width, groups and channels per slab, slabs
    int lpp;                // vectors per pixel of a slab
    int rows, nk;           // pixels per step, steps per pixel (lpp > kThreads)
    int cs;                 // cluster size
    int ncache;             // steps kept in shared memory
    float eps;
    int act;
};

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v)
{
    return v;
}
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v)
{
    return __bfloat162float(v);
}
template <>
__device__ __forceinline__ float to_f<__half>(__half v)
{
    return __half2float(v);
}
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

__device__ __forceinline__ float gn_act(float v, int act)
{
    if (act == K_ACT_GELU)
        return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f));
    if (act == K_ACT_RELU)
        return v > 0.0f ? v : (v != v ? v : 0.0f);
    return v;
}

__device__ __forceinline__ float ld_cluster(uint32_t addr)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

template <typename TI, typename TO, int V>
__global__ void __launch_bounds__(kThreads, 2) groupnorm_kernel(const GnArgs a)
{
    using VI = Vec<TI, V>;
    using VO = Vec<TO, V>;
    extern __shared__ __align__(16) uint8_t cache_raw[];
    VI *cache = reinterpret_cast<VI *>(cache_raw);
    __shared__ float sn[kThreads], sm[kThreads], sq[kThreads];
    __shared__ float pub[kMaxSlabGroups][3];       // this CTA's (n, mean, M2), read by the cluster
    __shared__ float gmean[kMaxSlabGroups], grstd[kMaxSlabGroups];
    const int t = threadIdx.x;
    const int rank = (int)(blockIdx.x % a.cs), unit = (int)(blockIdx.x / a.cs);
    const int sample = unit / a.nslab, slab = unit - sample * a.nslab;
    const int c0 = slab * a.S;
    const TI *x = reinterpret_cast<const TI *>(a.x) + sample * a.sx + c0;
    TO *y = reinterpret_cast<TO *>(a.y) + sample * a.sy + c0;
    // this CTA's pixels [p0, p0 + np)
    const long per = a.npix / a.cs, extra = a.npix - per * a.cs;
    const long p0 = rank * per + (rank < extra ? rank : extra);
    const long np = per + (rank < extra ? 1 : 0);
    // A step covers `rows` pixels (nk == 1: thread = (row, vector)), or one
    // nk-th of a pixel (nk > 1, a group wider than the block).
    const int row = a.nk == 1 ? t / a.lpp : 0;
    const int lane0 = a.nk == 1 ? t - row * a.lpp : t;
    const bool in_row = a.nk > 1 || row < a.rows;
    const long steps = a.nk == 1 ? (np + a.rows - 1) / a.rows : np * a.nk;
    auto where = [&](long it, long &pix, int &lane) {
        if (a.nk == 1) {
            pix = it * a.rows + row;
            lane = lane0;
            return in_row && pix < np;
        }
        pix = it / a.nk;
        lane = t + (int)(it - pix * a.nk) * kThreads;
        return lane < a.lpp;
    };

    griddep_wait();
    griddep_launch();

    float n = 0.0f, mean = 0.0f, m2 = 0.0f;
    for (long it = 0; it < steps; it += kUnroll) {
        VI v[kUnroll];
        bool ok[kUnroll];
        int cnt = 0;
#pragma unroll
        for (int u = 0; u < kUnroll; u++) {
            long pix;
            int lane;
            ok[u] = it + u < steps && where(it + u, pix, lane);
            if (ok[u]) {
                v[u] = *reinterpret_cast<const VI *>(x + (p0 + pix) * a.ldx + lane * V);
                cnt += V;
            }
        }
        if (!cnt)
            continue;
        float s = 0.0f;
#pragma unroll
        for (int u = 0; u < kUnroll; u++)
            if (ok[u]) {
#pragma unroll
                for (int e = 0; e < V; e++)
                    s += to_f(v[u].v[e]);
                if (it + u < a.ncache)
                    cache[(it + u) * kThreads + t] = v[u];
            }
        const float c = (float)cnt, mu = s / c;
        float q = 0.0f;
#pragma unroll
        for (int u = 0; u < kUnroll; u++)
            if (ok[u]) {
#pragma unroll
                for (int e = 0; e < V; e++) {
                    const float d = to_f(v[u].v[e]) - mu;
                    q = fmaf(d, d, q);
                }
            }
        const float n1 = n + c, f = c / n1, d = mu - mean;
        mean = fmaf(d, f, mean);
        m2 += fmaf(d * d, n * f, q);
        n = n1;
    }
    sn[t] = n;
    sm[t] = mean;
    sq[t] = m2;
    __syncthreads();
    // a warp per group: the threads of the group's vectors (all when nk > 1)
    const int warp = t >> 5, lane32 = t & 31;
    const int vpg = a.nk == 1 ? a.cg / V : kThreads;  // threads of a row in a group
    const int members = a.nk == 1 ? a.rows * vpg : kThreads;
    for (int gi = warp; gi < a.gps; gi += kThreads / 32) {
        float tn = 0.0f, ts = 0.0f, tq = 0.0f;
        for (int m = lane32; m < members; m += 32) {
            const int r = m / vpg, i = r * a.lpp + gi * vpg + (m - r * vpg);
            const int idx = a.nk == 1 ? i : m;
            tn += sn[idx];
            ts = fmaf(sn[idx], sm[idx], ts);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            tn += __shfl_xor_sync(0xffffffffu, tn, o);
            ts += __shfl_xor_sync(0xffffffffu, ts, o);
        }
        const float mu = tn > 0.0f ? ts / tn : 0.0f;
        for (int m = lane32; m < members; m += 32) {
            const int r = m / vpg, i = r * a.lpp + gi * vpg + (m - r * vpg);
            const int idx = a.nk == 1 ? i : m;
            const float d = sm[idx] - mu;
            if (sn[idx] > 0.0f)
                tq += fmaf(d * d, sn[idx], sq[idx]);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1)
            tq += __shfl_xor_sync(0xffffffffu, tq, o);
        if (lane32 == 0) {
            pub[gi][0] = tn;
            pub[gi][1] = mu;
            pub[gi][2] = tq;
        }
    }
    if (a.cs > 1)
        cluster_sync_all();
    else
        __syncthreads();
    for (int gi = t; gi < a.gps; gi += kThreads) {
        const uint32_t mine = smem_addr(&pub[gi][0]);
        float tn = 0.0f, ts = 0.0f, tq = 0.0f;
        for (int r = 0; r < a.cs; r++) {
            const uint32_t p = a.cs > 1 ? mapa_shared(mine, r) : mine;
            const float pn = ld_cluster(p);
            tn += pn;
            ts = fmaf(pn, ld_cluster(p + 4), ts);
        }
        const float mu = ts / tn;
        for (int r = 0; r < a.cs; r++) {
            const uint32_t p = a.cs > 1 ? mapa_shared(mine, r) : mine;
            const float pn = ld_cluster(p);
            if (pn > 0.0f) {
                const float d = ld_cluster(p + 4) - mu;
                tq += fmaf(d * d, pn, ld_cluster(p + 8));
            }
        }
        gmean[gi] = mu;
        grstd[gi] = 1.0f / sqrtf(tq / tn + a.eps);
    }
    __syncthreads();
    // no CTA may exit while another still reads its published statistics
    if (a.cs > 1)
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");

    const bool fixed = a.nk == 1;
    float ga[V], be[V], mu = 0.0f, rs = 0.0f;
    if (fixed && in_row) {
        const int gi = lane0 * V / a.cg;
        mu = gmean[gi];
        rs = grstd[gi];
#pragma unroll
        for (int e = 0; e < V; e++) {
            ga[e] = __ldg(a.g + c0 + lane0 * V + e) * rs;
            be[e] = __ldg(a.b + c0 + lane0 * V + e);
        }
    }
    else {
        mu = gmean[0];
        rs = grstd[0];
    }
    for (long top = steps; top > 0; top -= kUnroll) {
        VI v[kUnroll];
        bool ok[kUnroll];
        long pix[kUnroll];
        int lane[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; u++) {
            const long it = top - 1 - u;
            ok[u] = it >= 0 && where(it, pix[u], lane[u]);
            if (ok[u])
                v[u] = it < a.ncache ? cache[it * kThreads + t]
                                     : *reinterpret_cast<const VI *>(x + (p0 + pix[u]) * a.ldx +
                                                                     lane[u] * V);
        }
#pragma unroll
        for (int u = 0; u < kUnroll; u++)
            if (ok[u]) {
                if (!fixed) {
#pragma unroll
                    for (int e = 0; e < V; e++) {
                        ga[e] = __ldg(a.g + c0 + lane[u] * V + e) * rs;
                        be[e] = __ldg(a.b + c0 + lane[u] * V + e);
                    }
                }
                VO w;
#pragma unroll
                for (int e = 0; e < V; e++)
                    w.v[e] = from_f<TO>(gn_act(fmaf(to_f(v[u].v[e]) - mu, ga[e], be[e]), a.act));
                *reinterpret_cast<VO *>(y + (p0 + pix[u]) * a.ldy + lane[u] * V) = w;
            }
    }
    if (a.cs > 1)
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Shared-memory limit and clusters above 8 CTAs, once per kernel and device.
template <auto Kern>
cudaError_t prepare_once()
{
    static int done[64];
    int dev = 0;
    const bool known = cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64;
    if (known && done[dev])
        return cudaSuccess;
    cudaError_t e = cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         kCacheBytes);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(Kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess && known)
        done[dev] = 1;
    return e;
}

template <typename TI, typename TO, int V>
int launch(GnArgs &a, int nb, int C, int groups, cudaStream_t s)
{
    const cudaError_t pe = prepare_once<groupnorm_kernel<TI, TO, V>>();
    if (pe != cudaSuccess)
        return (int)pe;
    // the fewest whole groups of kSlabBytes
    a.gps = 1;
    for (int d = 1; d <= groups && d <= kMaxSlabGroups && d * (a.cg / V) <= kThreads; d++)
        if (groups % d == 0) {
            a.gps = d;
            if ((long)d * a.cg * (long)sizeof(TI) >= kSlabBytes)
                break;
        }
    a.S = a.gps * a.cg;
    a.nslab = C / a.S;
    a.lpp = a.S / V;
    a.nk = a.lpp > kThreads ? (a.lpp + kThreads - 1) / kThreads : 1;
    a.rows = a.nk == 1 ? kThreads / a.lpp : 1;
    const long units = (long)nb * a.nslab;
    // CTAs per unit: enough to fill two CTAs per SM, none with less than a step
    const long slots = 2L * device_sms();
    const long steps = a.nk == 1 ? (a.npix + a.rows - 1) / a.rows : a.npix * a.nk;
    a.cs = 1;
    while (a.cs < kMaxCluster && units * a.cs * 2 <= slots && a.cs * 2 <= steps && a.cs * 2 <= a.npix)
        a.cs *= 2;
    if (units * a.cs > 0x7fffffffL)
        return K_EARG;
    const long mine = (a.npix + a.cs - 1) / a.cs;
    const long msteps = a.nk == 1 ? (mine + a.rows - 1) / a.rows : mine * a.nk;
    const long room = kCacheBytes / (long)(kThreads * V * sizeof(TI));
    a.ncache = (int)(msteps < room ? msteps : room);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.cs;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(units * a.cs));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = (size_t)a.ncache * kThreads * V * sizeof(TI);
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return (int)cudaLaunchKernelEx(&cfg, groupnorm_kernel<TI, TO, V>, (const GnArgs)a);
}

template <typename TI, typename TO>
int launch_v(GnArgs &a, int nb, int C, int groups, cudaStream_t s)
{
    // widest vector that divides a group and every row start
    auto fits = [&](int v) {
        return a.cg % v == 0 && a.ldx % v == 0 && a.ldy % v == 0 && a.sx % v == 0 && a.sy % v == 0 &&
               reinterpret_cast<uintptr_t>(a.x) % (v * sizeof(TI)) == 0 &&
               reinterpret_cast<uintptr_t>(a.y) % (v * sizeof(TO)) == 0;
    };
    if (sizeof(TI) == 2 && fits(8))
        return launch<TI, TO, sizeof(TI) == 2 ? 8 : 4>(a, nb, C, groups, s);
    if (fits(4))
        return launch<TI, TO, 4>(a, nb, C, groups, s);
    if (fits(2))
        return launch<TI, TO, 2>(a, nb, C, groups, s);
    return launch<TI, TO, 1>(a, nb, C, groups, s);
}

}  // namespace
}  // namespace sam3

extern "C" int k_groupnorm(const void *X, int xt, long ldx, long sx, void *Y, int yt, long ldy,
                           long sy, const float *g, const float *b, int nb, long npix, int C,
                           int groups, float eps, int act, k_stream s)
{
    using namespace sam3;
    if (nb <= 0 || npix <= 0 || C <= 0 || groups <= 0 || C % groups || npix > (1L << 40))
        return K_EARG;
    GnArgs a = {};
    a.x = X;
    a.y = Y;
    a.g = g;
    a.b = b;
    a.ldx = ldx;
    a.sx = sx;
    a.ldy = ldy;
    a.sy = sy;
    a.npix = npix;
    a.cg = C / groups;
    a.eps = eps;
    a.act = act;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(s);
    if (xt == K_F32 && yt == K_F32)
        return launch_v<float, float>(a, nb, C, groups, st);
    if (xt == K_F32 && yt == K_BF16)
        return launch_v<float, __nv_bfloat16>(a, nb, C, groups, st);
    if (xt == K_F32 && yt == K_F16)
        return launch_v<float, __half>(a, nb, C, groups, st);
    if (xt == K_BF16 && yt == K_BF16)
        return launch_v<__nv_bfloat16, __nv_bfloat16>(a, nb, C, groups, st);
    if (xt == K_F16 && yt == K_F16)
        return launch_v<__half, __half>(a, nb, C, groups, st);
    return K_EARG;
}
