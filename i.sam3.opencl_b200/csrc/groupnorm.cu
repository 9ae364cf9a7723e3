// SPDX-License-Identifier: Unlicense
// Group norm with an activation over channels-last maps (the detector's
// pixel decoder, sam3_kernels.cl:926-953, for any batch, type and group
// width): y = act((x - mean) rstd gamma[c] + beta[c]) with mean and variance
// of each sample's group of channels over all pixels.
//
// One launch, no workspace. A unit is (sample, slab), a slab the fewest
// whole groups whose channels fill kSlabBytes of a pixel's row in whole
// 16-byte vectors, so that a warp reads whole sectors although it reads part
// of each row. A cluster of 1 to 16 CTAs shares a unit's pixels. Each CTA
// streams its share once through a ring of cp.async slots in shared memory
// (each thread its own slots, so no barrier), which ends holding the last
// steps; the CTAs exchange (count, mean, M2) per group through distributed
// shared memory; the second pass walks back from the last step, out of the
// ring and then re-reading earlier steps into the freed slots (from L2, when
// the maps in flight are not far larger than it).
//
// A thread owns a vector of channels and steps over pixels. Statistics in
// fp32 without the cancellation of E[x^2] - E[x]^2: per channel, kUnroll
// pixels at a time are reduced to their own mean and M2 = sum (x - mean)^2 and
// merged into the running pair (mean += d f, M2 += M2' + (n f d) d, d = mean' -
// mean, f = n' / (n + n'); Chan, Golub and LeVeque 1979; with the first n = 0 no
// square of a mean is formed, which may pass 32 bits), two channels to an
// instruction; channels, threads and CTAs are merged by sum n_i mean_i / n and sum
// M2_i + n_i (mean_i - mean)^2 in a fixed order, so a result does not depend on
// timing. 4 x 288 x 288 x 256 bf16, 8 groups: 89 us, 5.2 TB/s over the 459 MB
// that cross HBM (X 1.7 times, Y once); one sample 31 us (clusters of 10, 80
// CTAs); 72 x 72 x 256 6.8 us, of which the exchange takes 2.5.
// Per-channel pairs cost about as many instructions as one pair per
// vector and let a vector span groups of any width.
#include "act.cuh"
#include "cluster.cuh"
#include "div.cuh"
#include "kernels.h"
#include "pdl.cuh"
#include "tc_ptx.cuh"
#include "tmap.cuh"
#include "vec.cuh"

#include <cuda_runtime.h>

namespace sam3 {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;
constexpr int kSlabBytes = 64;
constexpr int kMaxSlabGroups = 128;
constexpr int kMaxCluster = kMaxClusterCtas;
constexpr int kRing = 48;  // slots of 16-byte vectors, 12 batches
constexpr int kRingBytes = kThreads * kRing * 16;  // per CTA, one per SM

struct GnArgs {
    const void *x;
    void *y;
    const float *g, *b;
    long ldx, sx, ldy, sy;  // elements: pixel and sample strides
    long per, extra;        // pixels of a CTA; the first `extra` ranks have one more
    int steps, srem;        // per / rows, per % rows
    Div dcg;                // cg
    int cg, gps, S, nslab;  // group width, groups and channels per slab, slabs
    int lpp;                // vectors per pixel of a slab
    int rows, nk;           // pixels per step, blocks of vectors per pixel (lpp > kThreads)
    int cs;                 // cluster size
    int bpk, nring;         // batches of kUnroll steps per block of vectors, of the ring
    int span;               // a vector may hold channels of several groups
    float share;            // 1 / values of a group
    float eps;
    int act;
};

// Values 2 e and 2 e + 1 of a vector (one value and 0 when V is 1).
template <typename T, int V>
__device__ __forceinline__ uint64_t pair(const Vec<T, V> &v, int e)
{
    return f2_make(to_f(v.v[2 * e]), V > 1 ? to_f(v.v[V > 1 ? 2 * e + 1 : 0]) : 0.0f);
}

// Activation of two values: GELU of a 32-bit output as 0.5 x (1 + erf(x / sqrt
// 2)), which rounds 1 + erf; else max(x, lowest), NaN kept (lowest 0 is ReLU,
// -inf none).
template <typename TO, bool GELU>
__device__ __forceinline__ void gn_act(float &x, float &y, float lowest)
{
    if constexpr (GELU && sizeof(TO) == 2)
        gelu_pair_rel(x, y);
    else if constexpr (GELU) {
        x = 0.5f * x * (1.0f + erff(x * 0.70710678118654752f));
        y = 0.5f * y * (1.0f + erff(y * 0.70710678118654752f));
    }
    else {
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(lowest));
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(y) : "f"(lowest));
    }
}

// Two results side by side, rounded to nearest.
__device__ __forceinline__ void put2(float *dst, float x, float y)
{
    dst[0] = x;
    dst[1] = y;
}
__device__ __forceinline__ void put2(__nv_bfloat16 *dst, float x, float y)
{
    *reinterpret_cast<__nv_bfloat162 *>(dst) = __floats2bfloat162_rn(x, y);
}
__device__ __forceinline__ void put2(__half *dst, float x, float y)
{
    *reinterpret_cast<__half2 *>(dst) = __floats2half2_rn(x, y);
}

// A vector from global memory into a thread's own slot: cp.async where it has
// a size for it.
template <int BYTES>
__device__ __forceinline__ void fetch(uint8_t *slot, const void *src)
{
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(slot)), "l"(src) : "memory");
    else if constexpr (BYTES >= 4)
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_addr(slot)), "l"(src), "n"(BYTES)
                     : "memory");
    else
        *reinterpret_cast<uint16_t *>(slot) = *reinterpret_cast<const uint16_t *>(src);
}
__device__ __forceinline__ void fetch_commit()
{
    asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void fetch_wait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ float4 ld_cluster4(uint32_t addr)
{
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

template <typename TI, typename TO, int V, bool GELU>
__global__ void __launch_bounds__(kThreads, 1) groupnorm_kernel(const __grid_constant__ GnArgs a)
{
    using VI = Vec<TI, V>;
    using VO = Vec<TO, V>;
    constexpr int NP = (V + 1) / 2;
    // ring of slots, then the threads' statistics: (mean, M2) per thread, or per channel of it
    extern __shared__ __align__(16) uint8_t dyn[];
    constexpr int VB = (int)sizeof(VI);
    constexpr int kAhead = 4;  // batches in flight; the ring has at least one more
    uint8_t *ring = dyn + threadIdx.x * VB;
    float2 *red = reinterpret_cast<float2 *>(dyn + (size_t)a.nring * kUnroll * kThreads * VB);
    __shared__ float4 pub[kMaxSlabGroups];    // this CTA's (n, mean, M2) per part, read by the cluster
    __shared__ float2 gstat[kMaxSlabGroups];  // mean, 1 / sqrt(var + eps)
    const int t = threadIdx.x;
    const int rank = (int)(blockIdx.x % a.cs), unit = (int)(blockIdx.x / a.cs);
    const int sample = unit / a.nslab, slab = unit - sample * a.nslab;
    const int c0 = slab * a.S;
    // this CTA's pixels [p0, p0 + np)
    const bool more = rank < a.extra;
    const long p0 = rank * a.per + (more ? rank : a.extra);
    const long np = a.per + more;
    const bool roll = a.srem + more == a.rows;  // the extra pixel fills a step
    const int q = a.steps + roll, rem = roll ? 0 : a.srem + more;
    // thread = (row, vector); with nk > 1 (a group wider than the block) the
    // block walks over all pixels once per block of vectors
    const int row = a.nk == 1 ? t / a.lpp : 0;
    const int lane0 = a.nk == 1 ? t - row * a.lpp : t;
    auto count = [&](int r) { return r < a.rows ? q + (r < rem) : 0; };
    const int mine = count(row);
    const TI *x = reinterpret_cast<const TI *>(a.x) + sample * a.sx + (p0 + row) * a.ldx + c0;
    TO *y = reinterpret_cast<TO *>(a.y) + sample * a.sy + (p0 + row) * a.ldy + c0;
    const long dx = a.rows * a.ldx, dy = a.rows * a.ldy;

    griddep_wait();

    // Batches of kUnroll steps, bpk per block of vectors, in order: this thread's
    // vectors of the next one into its slots of the ring. All ring indexes
    // step round by one, without divisions.
    const int batches = a.nk * a.bpk;
    constexpr int SLOT = kUnroll * kThreads * VB;  // bytes of a batch in the ring
    auto fetch4 = [&](uint8_t *slot, const TI *src, int left) {
        if (left >= kUnroll) {
#pragma unroll
            for (int u = 0; u < kUnroll; u++)
                fetch<VB>(slot + u * kThreads * VB, src + u * dx);
        }
        else {
            for (int u = 0; u < left; u++)
                fetch<VB>(slot + u * kThreads * VB, src + u * dx);
        }
    };
    auto live = [&](int k) { return lane0 + k * kThreads < a.lpp ? mine : 0; };
    int lk = 0, lb = 0, lslot = 0;  // next batch to load: block, batch of it, slot
    const TI *lsrc = x + lane0 * V;
    auto load_next = [&]() {
        fetch4(ring + lslot * SLOT, lsrc, live(lk) - lb * kUnroll);
        lsrc += kUnroll * dx;
        lslot = lslot + 1 == a.nring ? 0 : lslot + 1;
        if (++lb == a.bpk) {
            lb = 0;
            lk++;
            lsrc = x + (lane0 + lk * kThreads) * V;
        }
    };
    for (int i = 0; i < kAhead; i++) {
        if (i < batches)
            load_next();
        fetch_commit();
    }
    int i = 0, islot = 0;  // batch at hand
    // gamma, beta and group of this thread's channels in block k of vectors
    // (the first block to be written is read while X arrives)
    float cgam[2 * NP], cbet[2 * NP];
    int cgrp[2 * NP];
    auto channel_params = [&](int k) {
        const int lane = lane0 + k * kThreads;
#pragma unroll
        for (int e = 0; e < 2 * NP; e++) {
            const int ch = (lane < a.lpp ? lane : 0) * V + (e < V ? e : 0);
            cgrp[e] = a.gps == 1 ? 0 : (int)quot(ch, a.dcg);
            cgam[e] = __ldg(a.g + c0 + ch);
            cbet[e] = __ldg(a.b + c0 + ch);
        }
    };
    channel_params(a.nk - 1);
    float tn = 0.0f, tmean = 0.0f, tm2 = 0.0f;  // the thread's, over its vectors (not span)
    for (int k = 0; k < a.nk; k++) {
        const int lane = lane0 + k * kThreads;
        const int n = lane < a.lpp ? mine : 0;
        uint64_t mean[NP], m2[NP];
#pragma unroll
        for (int e = 0; e < NP; e++)
            mean[e] = m2[e] = 0;
        for (int bi = 0; bi < a.bpk; bi++) {
            const int it = bi * kUnroll;
            if (i + kAhead < batches)
                load_next();
            fetch_commit();
            fetch_wait<kAhead>();
            const VI *slot = reinterpret_cast<const VI *>(ring + islot * SLOT);
            i++;
            islot = islot + 1 == a.nring ? 0 : islot + 1;
            if (it + kUnroll <= n) {
                VI v[kUnroll];
#pragma unroll
                for (int u = 0; u < kUnroll; u++)
                    v[u] = slot[u * kThreads];
                const float f = rcp_approx((float)(bi + 1)), w = kUnroll * (1.0f - f);
                const uint64_t f2 = f2_make(f, f), w2 = f2_make(w, w);
#pragma unroll
                for (int e = 0; e < NP; e++) {
                    static_assert(kUnroll == 4, "mean of a batch");
                    uint64_t fv[kUnroll];
#pragma unroll
                    for (int u = 0; u < kUnroll; u++)
                        fv[u] = pair<TI, V>(v[u], e);
                    const uint64_t mu = mul2(add2(add2(fv[0], fv[1]), add2(fv[2], fv[3])),
                                             f2_make(0.25f, 0.25f));
                    const uint64_t neg = f2_make(-1.0f, -1.0f);
                    uint64_t q = 0;
#pragma unroll
                    for (int u = 0; u < kUnroll; u++) {
                        const uint64_t d = fma2(mu, neg, fv[u]);
                        q = fma2(d, d, q);
                    }
                    const uint64_t d = fma2(mean[e], neg, mu);
                    mean[e] = fma2(d, f2, mean[e]);
                    m2[e] = add2(m2[e], fma2(mul2(d, w2), d, q));
                }
            }
            else {
                for (int j = it; j < n; j++) {
                    const VI v = slot[(j - it) * kThreads];
                    const float f = 1.0f / (float)(j + 1), w = (float)j * f;
                    const uint64_t f2 = f2_make(f, f), w2 = f2_make(w, w);
#pragma unroll
                    for (int e = 0; e < NP; e++) {
                        const uint64_t d = fma2(mean[e], f2_make(-1.0f, -1.0f), pair<TI, V>(v, e));
                        mean[e] = fma2(d, f2, mean[e]);
                        m2[e] = fma2(mul2(d, w2), d, m2[e]);
                    }
                }
            }
        }
        float me[2 * NP], qe[2 * NP];
#pragma unroll
        for (int e = 0; e < NP; e++) {
            f2_split(mean[e], me[2 * e], me[2 * e + 1]);
            f2_split(m2[e], qe[2 * e], qe[2 * e + 1]);
        }
        if (a.span) {  // nk is 1: channel statistics [row][channel]
            if (row < a.rows) {
#pragma unroll
                for (int e = 0; e < V; e++)
                    red[row * a.S + lane * V + e] = make_float2(me[e], qe[e]);
            }
        }
        else if (n > 0) {  // one group: merge the channels
            float s = 0.0f, q = 0.0f;
#pragma unroll
            for (int e = 0; e < V; e++)
                s += me[e];
            const float mu = s * (1.0f / V), c = (float)n;
#pragma unroll
            for (int e = 0; e < V; e++)
                q += fmaf((me[e] - mu) * (me[e] - mu), c, qe[e]);
            const float nn = c * V, n1 = tn + nn, f = nn / n1, d = mu - tmean;
            tmean = fmaf(d, f, tmean);
            tm2 += fmaf(d * (tn * f), d, q);
            tn = n1;
        }
    }
    if (!a.span)
        red[t] = make_float2(tmean, tm2);
    __syncthreads();
    // The members of a group are the threads of its vectors, or its (row,
    // channel) pairs; nparts warps share a group and each publishes its own
    // (n, mean, M2): the mean of its members first, then sum M2_i + n_i (mean_i -
    // mean)^2; n and M2 as shares of the group's values from here on, so that the
    // sums are of the size of the mean and the variance. All parts of the
    // cluster are then merged at once in the same way.
    constexpr int NW = kThreads / 32;
    const int warp = t >> 5, lane32 = t & 31;
    const int nparts = a.gps >= NW ? 1 : NW / a.gps;
    const int width = a.span ? a.cg : (a.nk == 1 ? a.cg / V : kThreads);
    const int pitch = a.span ? a.S : a.lpp;
    const int members = a.rows * width;
    const int dr = nparts * 32 / width, di = nparts * 32 - dr * width;  // to a lane's next member
    auto size = [&](int r, int i) {  // values behind member i of row r, as a share
        if (a.nk == 1)
            return (float)count(r) * (a.span ? 1 : V) * a.share;
        return (float)np * V * (float)(i < a.lpp ? (a.lpp - 1 - i) / kThreads + 1 : 0) * a.share;
    };
    for (int w = warp; w < a.gps * nparts; w += NW) {
        const int gi = w / nparts, part = w - gi * nparts;
        const int m0 = part * 32 + lane32, r0 = m0 / width, i0 = m0 - r0 * width;
        const float2 *mine_at = red + gi * width;
        float n = 0.0f, mu = 0.0f, s = 0.0f;
#pragma unroll
        for (int pass = 0; pass < 2; pass++) {
            int r = r0, i = i0;
            s = 0.0f;
            for (int m = m0; m < members; m += nparts * 32) {
                const float c = size(r, i);
                if (c > 0.0f) {
                    const float2 st = mine_at[r * pitch + i];
                    if (pass == 0)
                        n += c;
                    s += pass == 0 ? c * st.x : fmaf((st.x - mu) * (st.x - mu), c, st.y * a.share);
                }
                i += di;
                r += dr;
                if (i >= width) {
                    i -= width;
                    r++;
                }
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                s += __shfl_xor_sync(0xffffffffu, s, o);
                if (pass == 0)
                    n += __shfl_xor_sync(0xffffffffu, n, o);
            }
            if (pass == 0)
                mu = n > 0.0f ? s / n : 0.0f;
        }
        if (lane32 == 0)
            pub[w] = make_float4(n, mu, s, 0.0f);
    }
    if (a.cs > 1)
        cluster_sync_all();
    else
        __syncthreads();
    // 16 or 32 lanes per group, a lane up to kParts of its parts
    constexpr int kParts = kMaxCluster * NW / 32;
    const int nall = a.cs * nparts, lw = nall > 16 ? 32 : 16;
    for (int g0 = 0; g0 < a.gps; g0 += kThreads / lw) {
        const int gi = g0 + t / lw, l = t & (lw - 1);
        float4 q[kParts];
        float n = 0.0f, s = 0.0f;
#pragma unroll
        for (int k = 0; k < kParts; k++) {
            const int e = l + k * lw, r = e / nparts;
            q[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (gi < a.gps && e < nall) {
                const uint32_t own = smem_addr(&pub[gi * nparts + (e - r * nparts)]);
                q[k] = ld_cluster4(a.cs > 1 ? mapa_shared(own, r) : own);
            }
        }
#pragma unroll
        for (int k = 0; k < kParts; k++) {
            n += q[k].x;
            s += q[k].x > 0.0f ? q[k].x * q[k].y : 0.0f;
        }
        for (int o = lw / 2; o; o >>= 1) {
            n += __shfl_xor_sync(0xffffffffu, n, o);
            s += __shfl_xor_sync(0xffffffffu, s, o);
        }
        const float mu = s / n;
        s = 0.0f;
#pragma unroll
        for (int k = 0; k < kParts; k++)
            s += q[k].x > 0.0f ? fmaf((q[k].y - mu) * (q[k].y - mu), q[k].x, q[k].z) : 0.0f;
        for (int o = lw / 2; o; o >>= 1)
            s += __shfl_xor_sync(0xffffffffu, s, o);
        if (l == 0 && gi < a.gps)
            gstat[gi] = make_float2(mu, 1.0f / sqrtf(s / n + a.eps));
    }
    __syncthreads();
    // no CTA may exit while another still reads its published statistics
    if (a.cs > 1)
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");

    griddep_launch();
    // Back from the last batch; those before the ring's are re-read as its slots
    // come free.
    const float lowest = a.act == K_ACT_RELU ? 0.0f : -INFINITY;
    int ri = batches - 1 - a.nring;  // next batch to re-read
    int rk = ri >= 0 ? ri / a.bpk : 0, rb = ri - rk * a.bpk;
    const TI *rsrc = x + (lane0 + rk * kThreads) * V + (long)rb * kUnroll * dx;
    for (int k = a.nk - 1; k >= 0; k--) {
        const int lane = lane0 + k * kThreads;
        const int n = lane < a.lpp ? mine : 0;
        uint64_t nm[NP], ga[NP], be[NP];  // -mean, gamma rstd, beta
        {
            float sm[2 * NP], sg[2 * NP], sb[2 * NP];
            if (k < a.nk - 1)
                channel_params(k);
#pragma unroll
            for (int e = 0; e < 2 * NP; e++) {
                const float2 st = gstat[cgrp[e]];
                sm[e] = -st.x;
                sg[e] = cgam[e] * st.y;
                sb[e] = cbet[e];
            }
#pragma unroll
            for (int e = 0; e < NP; e++) {
                nm[e] = f2_make(sm[2 * e], sm[2 * e + 1]);
                ga[e] = f2_make(sg[2 * e], sg[2 * e + 1]);
                be[e] = f2_make(sb[2 * e], sb[2 * e + 1]);
            }
        }
        auto one = [&](const VI &v, TO *dst) {
            VO w;
#pragma unroll
            for (int e = 0; e < NP; e++) {
                float z0, z1;
                f2_split(fma2(add2(pair<TI, V>(v, e), nm[e]), ga[e], be[e]), z0, z1);
                gn_act<TO, GELU>(z0, z1, lowest);
                if constexpr (V > 1)
                    put2(w.v + 2 * e, z0, z1);
                else
                    w.v[0] = from_f<TO>(z0);
            }
            *reinterpret_cast<VO *>(dst) = w;
        };
        TO *py = y + lane * V + (long)a.bpk * kUnroll * dy;
        for (int bi = a.bpk - 1; bi >= 0; bi--) {
            const int left = n - bi * kUnroll;
            py -= kUnroll * dy;
            islot = islot == 0 ? a.nring - 1 : islot - 1;
            // a re-read batch has kAhead newer groups behind it at least
            if (--i + a.nring < batches)
                fetch_wait<kAhead>();
            const VI *slot = reinterpret_cast<const VI *>(ring + islot * SLOT);
            if (left >= kUnroll) {
#pragma unroll
                for (int u = 0; u < kUnroll; u++)
                    one(slot[u * kThreads], py + u * dy);
            }
            else {
                for (int u = 0; u < left; u++)
                    one(slot[u * kThreads], py + u * dy);
            }
            if (ri >= 0) {
                fetch4(ring + islot * SLOT, rsrc, live(rk) - rb * kUnroll);
                ri--;
                rsrc -= kUnroll * dx;
                if (--rb < 0) {
                    rb = a.bpk - 1;
                    rk--;
                    rsrc = x + (lane0 + rk * kThreads) * V + (long)rb * kUnroll * dx;
                }
            }
            fetch_commit();
        }
    }
    if (a.cs > 1)
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <typename TI, typename TO, int V, bool GELU>
int launch_a(GnArgs &a, int nb, long npix, int C, cudaStream_t s)
{
    const cudaError_t pe =
        cluster_prepare_once<groupnorm_kernel<TI, TO, V, GELU>>(kRingBytes + kThreads * (int)sizeof(float2));
    if (pe != cudaSuccess)
        return (int)pe;
    a.nslab = C / a.S;
    a.lpp = a.S / V;
    a.nk = a.lpp > kThreads ? (a.lpp + kThreads - 1) / kThreads : 1;
    a.rows = a.nk == 1 ? kThreads / a.lpp : 1;
    a.span = a.cg % V != 0;
    const long units = (long)nb * a.nslab;
    // CTAs per unit: the largest cluster of which all units' run at once (a
    // second wave of clusters costs more than the idle SMs: 24 units of 6
    // CTAs, 22 clusters fit, 24.6 us; of 4 CTAs, 33 fit, 15.6 us), none with less
    // than a step
    const long steps = (npix + a.rows - 1) / a.rows;
    a.cs = 1;
    for (int c = 2; c <= kMaxCluster && c <= steps; c++)
        if (units <= clusters_at_once<groupnorm_kernel<TI, TO, V, GELU>>(c, kThreads, kRingBytes))
            a.cs = c;
    a.per = npix / a.cs;
    a.extra = npix - a.per * a.cs;
    // batches of a CTA: the ring holds them all, or as many as fit
    const long msteps = (a.per + (a.extra > 0) + a.rows - 1) / a.rows;
    if (units > 0x7fffffffL / a.cs || msteps > (0x7fffffffL - kUnroll) / a.nk)
        return K_EARG;
    a.bpk = (int)((msteps + kUnroll - 1) / kUnroll);
    const size_t red = (size_t)kThreads * (a.span ? V : 1) * sizeof(float2);
    constexpr long batch = (long)kUnroll * kThreads * V * (long)sizeof(TI);
    const long room = (kRingBytes - (a.span ? (long)red : 0)) / batch, all = (long)a.bpk * a.nk;
    a.nring = (int)(all < room ? all : room);
    a.steps = (int)(a.per / a.rows);
    a.srem = (int)(a.per - (long)a.steps * a.rows);
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
    cfg.dynamicSmemBytes = (size_t)a.nring * batch + red;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = a.cs > 1 ? 2 : 1;
    return (int)cudaLaunchKernelEx(&cfg, groupnorm_kernel<TI, TO, V, GELU>, (const GnArgs)a);
}

template <typename TI, typename TO, int V>
int launch(GnArgs &a, int nb, long npix, int C, cudaStream_t s)
{
    return a.act == K_ACT_GELU ? launch_a<TI, TO, V, true>(a, nb, npix, C, s)
                               : launch_a<TI, TO, V, false>(a, nb, npix, C, s);
}

template <typename TI, typename TO>
int launch_v(GnArgs &a, int nb, long npix, int C, int groups, cudaStream_t s)
{
    // the fewest whole groups that are whole 16-byte vectors and kSlabBytes
    // long, else the fewest that are that long, else what a block can hold
    auto whole = [&](int d) { return (long)d * a.cg * (long)sizeof(TI); };
    int plain = 0, vec = 0;
    for (int d = 1; d <= groups && d <= kMaxSlabGroups && (long)d * a.cg <= kThreads; d++)
        if (groups % d == 0 && whole(d) >= kSlabBytes) {
            if (!plain)
                plain = d;
            if (!vec && whole(d) % 16 == 0)
                vec = d;
        }
    a.gps = vec ? vec : (plain ? plain : 1);
    if (!plain && !vec)  // few channels in all, or one group wider than a block
        for (int d = 1; d <= groups && d <= kMaxSlabGroups && (long)d * a.cg <= kThreads; d++)
            if (groups % d == 0)
                a.gps = d;
    a.S = a.gps * a.cg;
    // widest vector that divides a slab and every row start
    auto fits = [&](int v) {
        return a.S % v == 0 && a.ldx % v == 0 && a.ldy % v == 0 && a.sx % v == 0 && a.sy % v == 0 &&
               reinterpret_cast<uintptr_t>(a.x) % (v * sizeof(TI)) == 0 &&
               reinterpret_cast<uintptr_t>(a.y) % (v * sizeof(TO)) == 0 &&
               (a.S / v <= kThreads || a.cg % v == 0);
    };
    if (sizeof(TI) == 2 && fits(8))
        return launch<TI, TO, sizeof(TI) == 2 ? 8 : 4>(a, nb, npix, C, s);
    if (fits(4))
        return launch<TI, TO, 4>(a, nb, npix, C, s);
    if (fits(2))
        return launch<TI, TO, 2>(a, nb, npix, C, s);
    return launch<TI, TO, 1>(a, nb, npix, C, s);
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
    a.cg = C / groups;
    a.dcg = make_div(a.cg);
    a.share = (float)(1.0 / ((double)npix * a.cg));
    a.eps = eps;
    a.act = act;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(s);
    if (xt == K_F32 && yt == K_F32)
        return launch_v<float, float>(a, nb, npix, C, groups, st);
    if (xt == K_F32 && yt == K_BF16)
        return launch_v<float, __nv_bfloat16>(a, nb, npix, C, groups, st);
    if (xt == K_F32 && yt == K_F16)
        return launch_v<float, __half>(a, nb, npix, C, groups, st);
    if (xt == K_BF16 && yt == K_BF16)
        return launch_v<__nv_bfloat16, __nv_bfloat16>(a, nb, npix, C, groups, st);
    if (xt == K_F16 && yt == K_F16)
        return launch_v<__half, __half>(a, nb, npix, C, groups, st);
    return K_EARG;
}
