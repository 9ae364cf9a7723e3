// SPDX-License-Identifier: Unlicense
// Cross attention of query rows over an encoder's states of another length
// (the detector's queries and image tokens over padded prompts and over
// the image; attend, sam3_text.c:305-343, for batches of sequences with
// their own key counts, a key mask and shared key heads): per sequence b and
// head h
//   O = softmax_j(scale q . k_j over visible j) V,
// key j visible when j < klen[b] and kmask[b][j] == 0; a row without a
// visible key gets zeros. Masked and absent keys never reach the arithmetic
// (their rows are filled with zeros instead of being read), so what they
// hold, NaN included, does not matter.
//
// This file holds the forms for few rows or few keys (bandwidth and latency
// bound) on warp-level tensor instructions, in one launch without a
// workspace. The rows of a tile are the (query, head) pairs of one key head, so
// that the heads sharing it read its keys once. Four warps of 16 rows each
// take 64-key steps through a ring of cp.async stages; with 16 rows or fewer
// (single tokens) the four warps split a step's keys instead. When the tiles
// are fewer than the CTA slots, a cluster of up to 16 CTAs shares a tile's keys
// and merges (max, sum, output) through distributed shared memory (Parts in
// attn_cross.cuh). Measured: 8 sequences x 1 query of 16 heads over 1500 keys
// of 4 heads of 64 columns 8.5 us (1 CTA a tile 19; three steps 3.3 us, the
// exchange 1.3).
//
// bf16 / f16: products on mma.m16n8k16 with fp32 accumulation, P rounded to
// the operands' type (half a unit in the last place, 2^-8 / 2^-11 of a weight,
// the operands' own precision; f16 by 2^-40 of the row's largest at least,
// kWeightShift). fp32: each operand is split into two tf32 parts
// and x y taken as hi hi + hi lo + lo hi on mma.m16n8k8, off by about 2^-21 of a
// product; the dropped lo lo is of that size. Sums that may have overflowed, and
// values so small that their second parts fall below the smallest numbers, are
// seen at the end of a CTA's keys and taken again with V times a power of two
// (Retake). 201 queries x 5184 keys x 8 heads
// of 32 columns x 2: 68.6 us, bound by the splits' dependent arithmetic (issue
// slots 40 % busy at 16 warps per SM; the products alone need 25 us).
#include "attn_cross.cuh"
#include "cluster.cuh"
#include "kernels.h"
#include "pdl.cuh"
#include "tc_ptx.cuh"
#include "tmap.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace sam3 {
namespace {

constexpr int kThreads = 128;
constexpr int kMaxCluster = kMaxClusterCtas;
constexpr int kSplitSteps = 4;  // steps of a CTA from which two share them

__device__ __forceinline__ void cp16(uint32_t dst, const void *src, bool live)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
                 "r"(live ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void cp_commit()
{
    asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_wait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4],
                                                     uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
                 "{%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                              uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
                 "{%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// D = A B + C with C the same for both row halves.
template <typename T>
__device__ __forceinline__ void mma16_from(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0,
                                           float c1)
{
    if constexpr (__is_same(T, __half))
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
                     "{%8,%9}, {%10,%11,%10,%11};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
                     "{%8,%9}, {%10,%11,%10,%11};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void mma8(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
                 "{%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo, hi with tf32's 11 significand bits, off by 2^-22 of x at most.
// Only one factor of a product has hi cut, the other has it rounded: lo * lo is
// dropped, and with both cut it would always have the product's sign. Cutting
// (K, V): the largest numbers do not round up to infinity.
__device__ __forceinline__ void split_cut(float x, uint32_t &hi, uint32_t &lo)
{
    hi = __float_as_uint(x) & 0xffffe000u;
    lo = (__float_as_uint(x - __uint_as_float(hi)) + 0x1000u) & 0xffffe000u;
}
// Rounding (weights, at most 1; queries with MOST, which keeps them finite)
template <bool MOST>
__device__ __forceinline__ void split_near(float x, uint32_t &hi, uint32_t &lo)
{
    const uint32_t u = __float_as_uint(x);
    hi = (u + 0x1000u) & 0xffffe000u;
    if (MOST && (hi & 0x7fffffffu) == 0x7f800000u)
        hi = u & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u;
}

// Shared memory of a tile in 16-byte chunks. 16-bit types: rows of HDP * 2
// bytes with the chunk index XORed by the row (no conflicts for ldmatrix);
// fp32: rows padded by 16 bytes (fragment loads of 4 rows x 8 columns hit 32
// banks).
template <typename T, int HDP>
struct Tile {
    static constexpr int CPR = HDP * (int)sizeof(T) / 16;  // chunks of a row
    static constexpr int PITCH = sizeof(T) == 4 ? HDP * 4 + 16 : HDP * 2;
    static __device__ __forceinline__ uint32_t at(int row, int chunk)
    {
        if (sizeof(T) == 4)
            return (uint32_t)(row * PITCH + chunk * 16);
        const int x = CPR >= 8 ? (row & 7) : ((row >> 1) & 3);
        return (uint32_t)(row * PITCH + ((chunk ^ x) << 4));
    }
};

template <typename T, int HDP, int WM>
struct Cfg {
    static constexpr int BK = sizeof(T) == 4 && HDP == 128 ? 32 : 64;  // keys per step
    static constexpr int STAGES = sizeof(T) == 4 ? 2 : (HDP == 128 ? 3 : 4);
    static constexpr int KV_BYTES = BK * Tile<T, HDP>::PITCH;
    static constexpr int STAGE_BYTES = 2 * KV_BYTES;
    static constexpr int BM = 16 * WM, WK = 4 / WM;
    // shared memory: query rows, stages, visible keys of the stages, and in a
    // cluster the parts of the rows that this CTA merges
    static constexpr int OFF_RING = BM * Tile<T, HDP>::PITCH;
    static constexpr int OFF_VIS = OFF_RING + STAGES * STAGE_BYTES;
    static constexpr int OFF_PART = OFF_VIS + (STAGES * BK + 15) / 16 * 16;
    static constexpr int SMEM_WHOLE = OFF_PART;
    static constexpr int SMEM_PARTS = OFF_PART + BM * Parts<HDP>::PR * 4;
    static_assert(WK * BM * Parts<HDP>::PR * 4 <= STAGES * STAGE_BYTES, "the warps' parts lie over the stages");
};

// Query row of row gr of a key head's (query, head) rows.
__device__ __forceinline__ long query_of(const XaArgs &a, long gr)
{
    return gr < 0x7fffffffL ? (long)quot((uint32_t)gr, a.dg) : gr / a.g;
}

// 32 bits: unnormalised outputs from kMostOut on, or none of kLeastOut, make a
// CTA take its keys again with the values times 2^k that puts the largest of them
// near 2^kTargetExp: every sum of up to 2^30 of them stays finite, parts
// of numbers down to the smallest are normal ones. 2^k is 2^64 at most, so that
// weights times 2^-k are normal too. (A factor of 1 / (2 Nk) in all weights,
// which needs no second pass, took those bits from values below 2^-100.)
struct Retake {
    static constexpr float kMostOut = 2.6584560e36f;    // 2^121: parts of 4 warps and 16 CTAs add up
    static constexpr float kLeastOut = 8.2718061e-25f;  // 2^-80
    static constexpr int kTargetExp = 64, kSmallExp = -70;
};

template <typename T, int HDP, int WM>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 && HDP == 32 ? 4 : 1)
    attn_cross_kernel(const __grid_constant__ XaArgs a)
{
    using TL = Tile<T, HDP>;
    using CF = Cfg<T, HDP, WM>;
    constexpr int WK = 4 / WM, BM = 16 * WM, BK = CF::BK, KW = BK / WK;
    constexpr int CPR = TL::CPR, EPC = 16 / (int)sizeof(T);  // elements per chunk
    constexpr int STAGES = CF::STAGES;
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int NT = KW / 8, DT = HDP / 8;  // score and output tiles of a warp
    extern __shared__ __align__(16) uint8_t smem[];
    uint8_t *ring = smem + CF::OFF_RING, *vis = smem + CF::OFF_VIS;
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const int wk = warp / WM;
    const int g4 = lane >> 2, t4 = lane & 3;

    const int rank = (int)(blockIdx.x % a.cs);
    const long item = blockIdx.x / a.cs;
    const int qt = (int)(item % a.nqt);
    // the warp's group of 16 rows: turned by the CTA, so that a tile's missing
    // group falls on another quarter of the SM each time
    const int wm = (int)((warp + item + rank) % WM);
    const long bh = item / a.nqt;
    const int b = (int)(bh / a.kvheads), kh = (int)(bh - (long)b * a.kvheads);
    // (every CTA of the cluster runs once the wait before the merge is over)
    if (a.cs > 1)
        asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    // groups of 16 rows dealt evenly to the tiles (201 rows: 3, 3, 3 and 4
    // groups, not 4, 4, 4 and 1)
    const long groups = (a.rows + 15) / 16;
    const long r0 = groups * qt / a.nqt * 16;
    const long r1 = min(a.rows, groups * (qt + 1) / a.nqt * 16);

    griddep_wait();

    int len = a.Nk;
    if (a.klen)
        len = min(max(__ldg(a.klen + b), 0), a.Nk);
    const uint8_t *mask = a.kmask ? a.kmask + (long)b * a.Nk : nullptr;
    const int steps_all = (len + BK - 1) / BK;
    const int s0 = (int)((long)steps_all * rank / a.cs);
    const int nsteps = (int)((long)steps_all * (rank + 1) / a.cs) - s0;
    const T *kb = reinterpret_cast<const T *>(a.k) + b * a.ks0 + kh * a.ks1;
    const T *vb = reinterpret_cast<const T *>(a.v) + b * a.vs0 + kh * a.vs1;
    const int hdc = (a.hd + EPC - 1) / EPC;  // chunks of a row that hold columns

    // ---- query rows
    {
        const T *qb = reinterpret_cast<const T *>(a.q) + b * a.qs0 + (long)kh * a.g * a.qs1;
        for (int i = t; i < BM * CPR; i += kThreads) {
            const int r = i / CPR, c = i % CPR;
            const long gr = r0 + r, qi = query_of(a, gr);
            const T *src = qb + qi * a.qld + (gr - qi * a.g) * a.qs1 + c * EPC;
            const bool live = gr < r1 && c < hdc;
            const uint32_t dst = smem_addr(smem + TL::at(r, c));
            if (a.qvec)
                cp16(dst, live ? src : a.q, live);
            else {
                T w[EPC];
#pragma unroll
                for (int e = 0; e < EPC; e++)
                    w[e] = live && c * EPC + e < a.hd ? src[e] : from_f<T>(0.0f);
                *reinterpret_cast<uint4 *>(smem + TL::at(r, c)) = *reinterpret_cast<const uint4 *>(w);
            }
        }
        cp_commit();
    }
    // ---- ring of key / value steps; each thread's chunks are fixed
    constexpr int PER = (BK * CPR + kThreads - 1) / kThreads;
    auto load = [&](int s, const bool (&see)[PER]) {
        const int st = s % STAGES;
        uint8_t *kd = ring + st * CF::STAGE_BYTES, *vd = kd + CF::KV_BYTES;
        const int j0 = (s0 + s) * BK;
#pragma unroll
        for (int p = 0; p < PER; p++) {
            const int i = t + p * kThreads;
            if (BK * CPR % kThreads && i >= BK * CPR)
                break;
            const int r = i / CPR, c = i % CPR;
            const bool live = see[p] && c < hdc;
            const T *ks = kb + (long)(j0 + r) * a.kld + c * EPC, *vs = vb + (long)(j0 + r) * a.vld + c * EPC;
            const uint32_t off = TL::at(r, c);
            if (a.kvec) {
                cp16(smem_addr(kd + off), live ? ks : kb, live);
                cp16(smem_addr(vd + off), live ? vs : vb, live);
            }
            else {
                T w[EPC], x[EPC];
#pragma unroll
                for (int e = 0; e < EPC; e++) {
                    const bool in = live && c * EPC + e < a.hd;
                    w[e] = in ? ks[e] : from_f<T>(0.0f);
                    x[e] = in ? vs[e] : from_f<T>(0.0f);
                }
                *reinterpret_cast<uint4 *>(kd + off) = *reinterpret_cast<const uint4 *>(w);
                *reinterpret_cast<uint4 *>(vd + off) = *reinterpret_cast<const uint4 *>(x);
            }
            if (mask && c == 0)
                vis[st * BK + r] = see[p];
        }
    };
    // which of this thread's rows of step s are visible (the mask bytes are
    // read one step before the rows they guard)
    auto look = [&](int s, bool (&see)[PER]) {
#pragma unroll
        for (int p = 0; p < PER; p++) {
            const int i = t + p * kThreads, j = (s0 + s) * BK + i / CPR;
            see[p] = s < nsteps && j < len;
            if (mask && see[p])
                see[p] = __ldg(mask + j) == 0;
        }
    };
    // 32 bits, rare (Retake): exponent of the largest finite value of this CTA's
    // visible keys, below -149 for none
    [[maybe_unused]] auto largest_value = [&]() {
        uint32_t big = 0;
        const long j0 = (long)s0 * BK, n = (min((long)(s0 + nsteps) * BK, (long)len) - j0) * a.hd;
        for (long i = t; i < n; i += kThreads) {
            const long j = j0 + i / a.hd;
            if (mask && __ldg(mask + j))
                continue;
            const uint32_t u = __float_as_uint((float)vb[j * a.vld + i % a.hd]) & 0x7fffffffu;
            if (u < 0x7f800000u)
                big = max(big, u);
        }
        __shared__ uint32_t warps[kThreads / 32];
        big = __reduce_max_sync(0xffffffffu, big);
        if (lane == 0)
            warps[warp] = big;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kThreads / 32; w++)
            big = max(big, warps[w]);
        return big ? ilogbf(__uint_as_float(big)) : -1000;
    };
    // a thread's own chunks of the values of stage st, before others read them
    [[maybe_unused]] auto scale_values = [&](int st, int ex) {
        const float f = __int_as_float((127 + ex) << 23);
#pragma unroll 1
        for (int i = t; i < BK * CPR; i += kThreads) {
            float4 *x = reinterpret_cast<float4 *>(ring + st * CF::STAGE_BYTES + CF::KV_BYTES + TL::at(i / CPR, i % CPR));
            const float4 v = *x;
            *x = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
        }
    };
    const bool busy = r0 + wm * 16 < r1;
    float o[DT][4], mx[2], sum[2];
    uint32_t qf[F32 ? 1 : HDP / 16][4];
    [[maybe_unused]] int vexp = 0;  // V is taken times 2^vexp (32 bits)

    for (;;) {
        bool see[PER];
#pragma unroll 1
        for (int s = 0; s < STAGES - 1; s++) {
            look(s, see);
            if (s < nsteps)
                load(s, see);
            cp_commit();
        }
        look(STAGES - 1, see);
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                o[d][e] = 0.0f;
        mx[0] = mx[1] = -INFINITY;
        sum[0] = sum[1] = 0.0f;

        for (int s = 0; s < nsteps; s++) {
            cp_wait<STAGES - 2>();
            if constexpr (F32) {
                if (vexp != 0)
                    scale_values(s % STAGES, vexp);
            }
            __syncthreads();
            if (s + STAGES - 1 < nsteps)
                load(s + STAGES - 1, see);
            cp_commit();
            look(s + STAGES, see);
            if (!busy)
                continue;  // only loads: none of the warp's rows exist
            const int st = s % STAGES;
            const uint8_t *ks = ring + st * CF::STAGE_BYTES, *vs = ks + CF::KV_BYTES;
            const uint32_t ka = smem_addr(ks), va = smem_addr(vs);
            const int jw = wk * KW;  // this warp's first key of the step

            float sc[NT][4];
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    sc[n][e] = 0.0f;
            if constexpr (!F32) {
                if (s == 0) {
#pragma unroll
                    for (int kk = 0; kk < HDP / 16; kk++)
                        ldsm4(smem_addr(smem) + TL::at(wm * 16 + (lane & 15), kk * 2 + (lane >> 4)), qf[kk]);
                }
#pragma unroll
                for (int kk = 0; kk < HDP / 16; kk++) {
#pragma unroll
                    for (int n = 0; n < NT; n += 2) {
                        // keys n*8 .. n*8+15, columns kk*16 .. kk*16+15
                        uint32_t kf[4];
                        ldsm4(ka + TL::at(jw + n * 8 + (lane & 7) + ((lane >> 4) << 3),
                                          kk * 2 + ((lane >> 3) & 1)),
                              kf);
                        mma16<T>(sc[n], qf[kk], kf[0], kf[1]);
                        mma16<T>(sc[n + 1], qf[kk], kf[2], kf[3]);
                    }
                }
            }
            else {
                const float *qs = reinterpret_cast<const float *>(smem) + (wm * 16 + g4) * (TL::PITCH / 4) + t4;
                const float *kf = reinterpret_cast<const float *>(ks) + (jw + g4) * (TL::PITCH / 4) + t4;
                // As P V below: 16 columns sum from zero and are added outside the
                // matrix unit. Output of 300 queries x 2000 keys, 128 columns: 2.8e-7
                // off, all columns in one chain 1.2e-6 (201 x 5184 x 32 columns 69 us,
                // then 67; 8 columns at a time 71).
#pragma unroll 1
                for (int kk = 0; kk < HDP / 8; kk += 2) {
                    uint32_t ah[2][4], al[2][4];
#pragma unroll
                    for (int u = 0; u < 2; u++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            split_near<true>(qs[(e & 1) * 8 * (TL::PITCH / 4) + (kk + u) * 8 + (e >> 1) * 4], ah[u][e],
                                             al[u][e]);
                    // four tiles side by side: a product waits for the one four before it
                    constexpr int NB = NT < 4 ? NT : 4;
#pragma unroll
                    for (int n0 = 0; n0 < NT; n0 += NB) {
                        float part[NB][4];
#pragma unroll
                        for (int n = 0; n < NB; n++)
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                part[n][e] = 0.0f;
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            uint32_t bh[NB][2], bl[NB][2];
#pragma unroll
                            for (int n = 0; n < NB; n++)
#pragma unroll
                                for (int e = 0; e < 2; e++)
                                    split_cut(kf[(n0 + n) * 8 * (TL::PITCH / 4) + (kk + u) * 8 + 4 * e], bh[n][e],
                                              bl[n][e]);
#pragma unroll
                            for (int n = 0; n < NB; n++)
                                mma8(part[n], al[u], bh[n][0], bh[n][1]);
#pragma unroll
                            for (int n = 0; n < NB; n++)
                                mma8(part[n], ah[u], bl[n][0], bl[n][1]);
#pragma unroll
                            for (int n = 0; n < NB; n++)
                                mma8(part[n], ah[u], bh[n][0], bh[n][1]);
                        }
#pragma unroll
                        for (int n = 0; n < NB; n++)
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                sc[n0 + n][e] += part[n][e];
                    }
                }
            }
            // ---- online softmax of rows g4 and g4 + 8
            const int j0 = (s0 + s) * BK + jw;
            if (mask) {
                const uint8_t *vw = vis + st * BK + jw;
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    const uint16_t two = *reinterpret_cast<const uint16_t *>(vw + n * 8 + t4 * 2);
                    if (!(two & 0xff))
                        sc[n][0] = sc[n][2] = -INFINITY;
                    if (!(two >> 8))
                        sc[n][1] = sc[n][3] = -INFINITY;
                }
            }
            else if (j0 + KW > len) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (j0 + n * 8 + t4 * 2 + (e & 1) >= len)
                            sc[n][e] = -INFINITY;
            }
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float m = -INFINITY;
#pragma unroll
                for (int n = 0; n < NT; n++)
                    m = max3f(m, sc[n][2 * h], sc[n][2 * h + 1]);
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                // Differences of scores are taken before they are scaled: a product
                // m scale rounded on its own would leave 2^(its rounding) in every
                // weight, past 2^30 more than 32 bits hold.
                const float mn = fmaxf(mx[h], m), base = mn == -INFINITY ? 0.0f : mn;
                const float corr = exp2f((mx[h] - base) * a.scale_log2);
                mx[h] = mn;
                const uint64_t neg2 = f2_make(-base, -base), sl2 = f2_make(a.scale_log2, a.scale_log2),
                               shift2 = f2_make(kWeightShift<T>, kWeightShift<T>);
                float add = 0.0f;
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    float x, y;
                    f2_split(fma2(add2(f2_make(sc[n][2 * h], sc[n][2 * h + 1]), neg2), sl2, shift2), x, y);
                    sc[n][2 * h] = ex2_approx(x);
                    sc[n][2 * h + 1] = ex2_approx(y);
                    add += sc[n][2 * h] + sc[n][2 * h + 1];
                }
                sum[h] = fmaf(sum[h], corr, add);
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    o[d][2 * h] *= corr;
                    o[d][2 * h + 1] *= corr;
                }
            }
            // ---- O += P V
            if constexpr (!F32) {
#pragma unroll
                for (int n = 0; n < NT; n += 2) {
                    const uint32_t pf[4] = {pack2<T>(sc[n][0], sc[n][1]), pack2<T>(sc[n][2], sc[n][3]),
                                            pack2<T>(sc[n + 1][0], sc[n + 1][1]),
                                            pack2<T>(sc[n + 1][2], sc[n + 1][3])};
#pragma unroll
                    for (int d = 0; d < DT; d += 2) {
                        uint32_t vf[4];
                        ldsm4t(va + TL::at(jw + n * 8 + (lane & 15), d + (lane >> 4)), vf);
                        mma16<T>(o[d], pf, vf[0], vf[1]);
                        mma16<T>(o[d + 1], pf, vf[2], vf[3]);
                    }
                }
            }
            else {
                // The product's k index runs over keys in any order as long as both
                // operands agree: index t4 is key 2 t4, t4 + 4 is key 2 t4 + 1, as
                // the scores already lie.
                // Each step's sum starts from zero and is added to O outside the
                // matrix unit, whose own additions truncate (5184 keys in one chain
                // were 8e-6 off).
                const float *vf = reinterpret_cast<const float *>(vs) + (jw + 2 * t4) * (TL::PITCH / 4) + g4;
                uint32_t ph[NT][4], pl[NT][4];
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    split_near<false>(sc[n][0], ph[n][0], pl[n][0]);
                    split_near<false>(sc[n][2], ph[n][1], pl[n][1]);
                    split_near<false>(sc[n][1], ph[n][2], pl[n][2]);
                    split_near<false>(sc[n][3], ph[n][3], pl[n][3]);
                }
#pragma unroll
                for (int d0 = 0; d0 < DT; d0 += 4) {
                    float hi[4][4], lo[4][4];
#pragma unroll
                    for (int d = 0; d < 4; d++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            hi[d][e] = lo[d][e] = 0.0f;
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        uint32_t bh[4][2], bl[4][2];
#pragma unroll
                        for (int d = 0; d < 4; d++)
#pragma unroll
                            for (int e = 0; e < 2; e++)
                                split_cut(vf[(n * 8 + e) * (TL::PITCH / 4) + (d0 + d) * 8], bh[d][e], bl[d][e]);
#pragma unroll
                        for (int d = 0; d < 4; d++)
                            mma8(lo[d], pl[n], bh[d][0], bh[d][1]);
#pragma unroll
                        for (int d = 0; d < 4; d++)
                            mma8(hi[d], ph[n], bh[d][0], bh[d][1]);
#pragma unroll
                        for (int d = 0; d < 4; d++)
                            mma8(lo[d], ph[n], bl[d][0], bl[d][1]);
                    }
#pragma unroll
                    for (int d = 0; d < 4; d++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            o[d0 + d][e] += hi[d][e] + lo[d][e];
                }
            }
        }
        cp_wait<0>();
        if constexpr (!F32)
            break;
        else {
            if (vexp != 0 || nsteps == 0)
                break;
            bool most = false, least = false;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    most |= !(fabsf(o[d][e]) < Retake::kMostOut);
                    least |= fabsf(o[d][e]) >= Retake::kLeastOut;
                }
            if (!__syncthreads_or(busy && (most || !least)))
                break;
            most = __syncthreads_or(most);
            least = __syncthreads_or(least);
            if (!most && least)
                break;
            const int top = largest_value();
            if (top < -149 || (!most && top >= Retake::kSmallExp))
                break;  // nothing but zeros; or small sums of larger values
            vexp = min(Retake::kTargetExp - top, 64);
            if (vexp == 0)
                break;
        }
    }
    // The next kernel's CTAs may come now: earlier they would take the free
    // slots of some SMs and leave it badly spread (201 queries over 5184 keys in
    // 32 bits: 83 us alone, 100 us in a row of such calls).
    griddep_launch();
#pragma unroll
    for (int h = 0; h < 2; h++) {
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
    }
    T *ob = reinterpret_cast<T *>(a.o) + b * a.os0 + (long)kh * a.g * a.os1;
    const float unscale = F32 ? __int_as_float((127 - vexp) << 23) : 1.0f;

    if (WK == 1 && a.cs == 1) {  // the tile is whole: straight from registers
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const long gr = r0 + wm * 16 + g4 + 8 * h, qi = query_of(a, gr);
            if (gr >= r1)
                continue;
            T *dst = ob + qi * a.old + (gr - qi * a.g) * a.os1;
            const float inv = sum[h] > 0.0f || sum[h] != sum[h] ? 1.0f / sum[h] : 0.0f;
#pragma unroll
            for (int d = 0; d < DT; d++) {
                const int c = d * 8 + t4 * 2;
                if (c >= a.hd)
                    continue;
                float x = o[d][2 * h] * inv, y = o[d][2 * h + 1] * inv;
                if constexpr (F32) {
                    x *= unscale;
                    y *= unscale;
                }
                if (a.ovec) {
                    if constexpr (F32)
                        *reinterpret_cast<float2 *>(dst + c) = make_float2(x, y);
                    else
                        *reinterpret_cast<uint32_t *>(dst + c) = pack2<T>(x, y);
                }
                else {
                    dst[c] = from_f<T>(x);
                    dst[c + 1] = from_f<T>(y);
                }
            }
        }
        return;
    }
    // ---- results of the warps' key parts and of the cluster's CTAs
    using PT = Parts<HDP>;
    const int rows = (int)(r1 - r0);
    auto store = [&](int r, int c, const float (&v)[4]) {  // columns c .. c + 3 of the tile's row r
        const long gr = r0 + r, qi = query_of(a, gr);
        T *dst = ob + qi * a.old + (gr - qi * a.g) * a.os1 + c;
#pragma unroll
        for (int e = 0; e < 4; e += 2)
            if (c + e < a.hd) {
                if (a.ovec) {
                    if constexpr (F32)
                        *reinterpret_cast<float2 *>(dst + e) = make_float2(v[e], v[e + 1]);
                    else
                        *reinterpret_cast<uint32_t *>(dst + e) = pack2<T>(v[e], v[e + 1]);
                }
                else {
                    dst[e] = from_f<T>(v[e]);
                    dst[e + 1] = from_f<T>(v[e + 1]);
                }
            }
    };
    const int rl = BM / a.cs;  // rows of the tile a CTA merges: r % cs == rank
    float *part = reinterpret_cast<float *>(smem + CF::OFF_PART);
    auto owner = [&](int r) {  // where this CTA's part of row r goes
        return mapa_shared(smem_addr(part + (rank * rl + r / a.cs) * PT::PR), r % a.cs);
    };
    if constexpr (WK > 1) {
        // the warps' parts first, over the stages
        float *mine = reinterpret_cast<float *>(ring);
        __syncthreads();
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int r = g4 + 8 * h;
            float *pr = mine + (wk * BM + r) * PT::PR;
#pragma unroll
            for (int d = 0; d < DT; d++)
                *reinterpret_cast<float2 *>(pr + d * 8 + t4 * 2) = make_float2(o[d][2 * h], o[d][2 * h + 1]);
            if (t4 == 0)
                *reinterpret_cast<float2 *>(pr + HDP) = make_float2(mx[h], sum[h]);
        }
        if (a.cs > 1)
            asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        __syncthreads();
        for (int e = t; e < rows * (HDP / 4); e += kThreads) {
            const int r = e / (HDP / 4), c = (e % (HDP / 4)) * 4;
            float2 ml[WK];
            float m = -INFINITY, l = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int p = 0; p < WK; p++) {
                ml[p] = *reinterpret_cast<const float2 *>(mine + (p * BM + r) * PT::PR + HDP);
                m = fmaxf(m, ml[p].x);
            }
#pragma unroll
            for (int p = 0; p < WK; p++) {
                const bool none = ml[p].x == -INFINITY;
                const float w = none ? 0.0f : exp2f((ml[p].x - m) * a.scale_log2);
                const float4 x = *reinterpret_cast<const float4 *>(mine + (p * BM + r) * PT::PR + c);
                l += none ? (ml[p].y == ml[p].y ? 0.0f : ml[p].y) : ml[p].y * w;
                v[0] = fmaf(x.x, w, v[0]);
                v[1] = fmaf(x.y, w, v[1]);
                v[2] = fmaf(x.z, w, v[2]);
                v[3] = fmaf(x.w, w, v[3]);
            }
            if (a.cs == 1) {
                const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    v[i] = v[i] * inv * unscale;
                store(r, c, v);
            }
            else {
                st_dsmem4(owner(r) + c * 4, v[0], v[1], v[2], v[3]);
                if (c == 0)
                    st_dsmem4(owner(r) + HDP * 4, m, l, unscale, 0.0f);
            }
        }
        if (a.cs == 1)
            return;
    }
    else {
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int r = wm * 16 + g4 + 8 * h;
            if (r >= rows)
                continue;
            const uint32_t dst = owner(r);
#pragma unroll
            for (int d = 0; d < DT; d++)
                st_dsmem2(dst + (d * 8 + t4 * 2) * 4, o[d][2 * h], o[d][2 * h + 1]);
            if (t4 == 0)
                st_dsmem4(dst + HDP * 4, mx[h], sum[h], unscale, 0.0f);
        }
    }
    cluster_sync_all();
    const int live = rows > rank ? (rows - 1 - rank) / a.cs + 1 : 0;
    PT::template merge<kThreads, F32>(part, a.cs, rl, live, a.scale_log2,
                                      [&](int i, int c, float x, float y, float z, float w) {
                                          const float v[4] = {x, y, z, w};
                                          store(i * a.cs + rank, c, v);
                                      });
}

// Few keys (all in one step) and many rows. A CTA reads the keys and values of
// one key head once and walks over tiles of 64 rows, each warp its 16 rows
// through three cp.async buffers of its own (no block barrier in the loop);
// one pass of softmax without a running maximum, row sums as a product with
// ones, -inf of hidden keys as the scores' first accumulator; results go back
// through the rows' buffer so that they are stored as 16-byte vectors. 8 x 5184
// rows x 8 heads of 32 columns over 39 keys: 14.5 us, 2.9 TB/s. No unit is full
// (issue slots 53 %, matrix unit 31 %, half the copy rate): what a warp waits for
// is its own chain of fragment loads, products, maxima, exponentials, products
// and the way out, at 14 warps per SM; the same loop without its arithmetic
// copies at 5.9 TB/s. Key and value fragments kept in registers, 5 or 6 CTAs per SM
// and two row groups per warp were slower (by 3 %, 11 to 20 %, 16 %).
template <typename T, int HDP, int KT>
__global__ void __launch_bounds__(kThreads, HDP <= 64 ? 4 : 3) attn_few_kernel(const __grid_constant__ XaArgs a)
{
    using TL = Tile<T, HDP>;
    constexpr int NK = KT * 16, CPR = TL::CPR, EPC = 8, NT = KT * 2, DT = HDP / 8, QB = 16 * TL::PITCH, ST = 3;
    extern __shared__ __align__(16) uint8_t smem[];
    uint8_t *ks = smem, *vs = ks + NK * TL::PITCH;
    __shared__ uint8_t vis[NK];
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31, g4 = lane >> 2, t4 = lane & 3;
    uint8_t *qs = vs + NK * TL::PITCH + warp * ST * QB;
    const int split = (int)(blockIdx.x % a.cs), bh = (int)(blockIdx.x / a.cs);  // cs: CTAs walking over a head's tiles
    const int b = bh / a.kvheads, kh = bh - b * a.kvheads;

    griddep_wait();

    const T *qb = reinterpret_cast<const T *>(a.q) + b * a.qs0 + (long)kh * a.g * a.qs1;
    T *ob = reinterpret_cast<T *>(a.o) + b * a.os0 + (long)kh * a.g * a.os1;
    const int hdc = a.hd / EPC;
    const int ntile = split < a.nqt ? (a.nqt - 1 - split) / a.cs + 1 : 0;
    auto row_at = [&](uint32_t gr, long ld, long s1) {
        const uint32_t qi = quot(gr, a.dg);
        return qi * ld + (gr - qi * a.dg.d) * s1;
    };
    // A lane's chunks of a tile are RS rows apart. Without shared heads their
    // addresses step by a constant from tile to tile.
    constexpr int NC = 16 * CPR / 32, RS = 32 / CPR;
    const int lr = lane / CPR, lc = lane % CPR;
    const bool plain = a.g == 1, col = lc < hdc;
    const uint32_t w0 = (uint32_t)split * 64 + warp * 16;  // first row of the warp's first tile
    const T *qp = qb + (w0 + lr) * a.qld + lc * EPC;
    T *op = ob + (w0 + lr) * a.old + lc * EPC;
    const long qstep = (long)a.cs * 64 * a.qld, ostep = (long)a.cs * 64 * a.old;
    long qleft = a.rows - w0 - lr;  // rows from the lane's first one to the last
    const uint32_t slot0 = smem_addr(qs);
    int qslot = 0;
    auto load_q = [&](int i) {
        if (i < ntile) {
            uint8_t *buf = qs + qslot * QB;
#pragma unroll
            for (int k = 0; k < NC; k++) {
                const int r = lr + k * RS;
                const bool live = col && qleft > k * RS;
                const T *src = plain ? qp + k * RS * a.qld
                                     : qb + (live ? row_at(w0 + (uint32_t)i * a.cs * 64 + r, a.qld, a.qs1) : 0) + lc * EPC;
                if (a.qvec)
                    cp16(slot0 + qslot * QB + TL::at(r, lc), live ? src : a.q, live);
                else {
                    T w[EPC];
#pragma unroll
                    for (int e = 0; e < EPC; e++)
                        w[e] = live ? src[e] : from_f<T>(0.0f);
                    *reinterpret_cast<uint4 *>(buf + TL::at(r, lc)) = *reinterpret_cast<const uint4 *>(w);
                }
            }
            qp += qstep;
            qleft -= a.cs * 64;
            qslot = qslot + 1 == ST ? 0 : qslot + 1;
        }
        cp_commit();
    };
    int len = a.Nk;
    if (a.klen)
        len = min(max(__ldg(a.klen + b), 0), a.Nk);
    {
        const uint8_t *mask = a.kmask ? a.kmask + (long)b * a.Nk : nullptr;
        const T *kb = reinterpret_cast<const T *>(a.k) + b * a.ks0 + kh * a.ks1;
        const T *vb = reinterpret_cast<const T *>(a.v) + b * a.vs0 + kh * a.vs1;
        for (int x = t; x < NK * CPR; x += kThreads) {
            const int r = x / CPR, c = x % CPR;
            bool see = r < len;
            if (see && mask)
                see = __ldg(mask + r) == 0;
            const bool live = see && c < hdc;
            const T *k1 = kb + r * a.kld + c * EPC, *v1 = vb + r * a.vld + c * EPC;
            uint8_t *kd = ks + TL::at(r, c), *vd = vs + TL::at(r, c);
            if (a.kvec) {
                cp16(smem_addr(kd), live ? k1 : kb, live);
                cp16(smem_addr(vd), live ? v1 : vb, live);
            }
            else {
                T w[EPC], y[EPC];
#pragma unroll
                for (int e = 0; e < EPC; e++) {
                    w[e] = live ? k1[e] : from_f<T>(0.0f);
                    y[e] = live ? v1[e] : from_f<T>(0.0f);
                }
                *reinterpret_cast<uint4 *>(kd) = *reinterpret_cast<const uint4 *>(w);
                *reinterpret_cast<uint4 *>(vd) = *reinterpret_cast<const uint4 *>(y);
            }
            if (c == 0)
                vis[r] = see;
        }
        cp_commit();
    }
    load_q(0);
    load_q(1);
    cp_wait<2>();
    __syncthreads();
    // What a lane's columns of the scores start from: -inf where the key is
    // hidden (its row of K is zero)
    float start[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 2; e++)
            start[n][e] = vis[n * 8 + t4 * 2 + e] ? 0.0f : -INFINITY;
    const uint32_t ka = smem_addr(ks), va = smem_addr(vs);
    constexpr uint32_t kOnes = __is_same(T, __half) ? 0x3c003c00u : 0x3f803f80u;
    const uint64_t sl2x2 = f2_make(a.scale_log2, a.scale_log2), shift2 = f2_make(kWeightShift<T>, kWeightShift<T>);
    auto key_frag = [&](int kk, int n, uint32_t (&f)[4]) {
        ldsm4(ka + TL::at(n * 8 + (lane & 7) + ((lane >> 4) << 3), kk * 2 + ((lane >> 3) & 1)), f);
    };
    auto value_frag = [&](int n, int d, uint32_t (&f)[4]) {
        ldsm4t(va + TL::at(n * 8 + (lane & 15), d + (lane >> 4)), f);
    };
    long left = a.rows - w0 - lr;
    int slot = 0;
    for (int i = 0; i < ntile; i++) {
        load_q(i + 2);
        cp_wait<2>();
        __syncwarp();
        uint8_t *buf = qs + slot * QB;
        slot = slot + 1 == ST ? 0 : slot + 1;
        float sc[NT][4];
#pragma unroll
        for (int kk = 0; kk < HDP / 16; kk++) {
            uint32_t qf[4];
            ldsm4(smem_addr(buf) + TL::at(lane & 15, kk * 2 + (lane >> 4)), qf);
#pragma unroll
            for (int n = 0; n < KT; n++) {
                uint32_t k4[4];
                key_frag(kk, 2 * n, k4);
                if (kk == 0) {
                    mma16_from<T>(sc[2 * n], qf, k4[0], k4[1], start[2 * n][0], start[2 * n][1]);
                    mma16_from<T>(sc[2 * n + 1], qf, k4[2], k4[3], start[2 * n + 1][0], start[2 * n + 1][1]);
                }
                else {
                    mma16<T>(sc[2 * n], qf, k4[0], k4[1]);
                    mma16<T>(sc[2 * n + 1], qf, k4[2], k4[3]);
                }
            }
        }
        __syncwarp();
        float inv[2], m[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            m[h] = -INFINITY;
#pragma unroll
            for (int n = 0; n < NT; n++)
                m[h] = max3f(m[h], sc[n][2 * h], sc[n][2 * h + 1]);
            m[h] = fmaxf(m[h], __shfl_xor_sync(0xffffffffu, m[h], 1));
            m[h] = fmaxf(m[h], __shfl_xor_sync(0xffffffffu, m[h], 2));
        }
        // Infinities of a query times a hidden key's zeros are NaN: where no score
        // is left such keys are hidden again (a score of +inf gives NaN anyway).
        if (__any_sync(0xffffffffu, fminf(m[0], m[1]) == -INFINITY)) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (start[n][e & 1] < 0.0f)
                        sc[n][e] = -INFINITY;
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const float base = m[h] == -INFINITY ? 0.0f : -m[h];
            const uint64_t base2 = f2_make(base, base);
#pragma unroll
            for (int n = 0; n < NT; n++) {
                float x, y;
                f2_split(fma2(add2(f2_make(sc[n][2 * h], sc[n][2 * h + 1]), base2), sl2x2, shift2), x, y);
                sc[n][2 * h] = ex2_approx(x);
                sc[n][2 * h + 1] = ex2_approx(y);
            }
        }
        float o[DT][4], sums[4];  // sums: a row's P times ones
#pragma unroll
        for (int n = 0; n < KT; n++) {
            const uint32_t pf[4] = {pack2<T>(sc[2 * n][0], sc[2 * n][1]), pack2<T>(sc[2 * n][2], sc[2 * n][3]),
                                    pack2<T>(sc[2 * n + 1][0], sc[2 * n + 1][1]),
                                    pack2<T>(sc[2 * n + 1][2], sc[2 * n + 1][3])};
#pragma unroll
            for (int d = 0; d < DT / 2; d++) {
                uint32_t v4[4];
                value_frag(2 * n, 2 * d, v4);
                if (n == 0) {
                    mma16_from<T>(o[2 * d], pf, v4[0], v4[1], 0.0f, 0.0f);
                    mma16_from<T>(o[2 * d + 1], pf, v4[2], v4[3], 0.0f, 0.0f);
                }
                else {
                    mma16<T>(o[2 * d], pf, v4[0], v4[1]);
                    mma16<T>(o[2 * d + 1], pf, v4[2], v4[3]);
                }
            }
            if (n == 0)
                mma16_from<T>(sums, pf, kOnes, kOnes, 0.0f, 0.0f);
            else
                mma16<T>(sums, pf, kOnes, kOnes);
        }
#pragma unroll
        for (int h = 0; h < 2; h++)
            inv[h] = sums[2 * h] > 0.0f || sums[2 * h] != sums[2 * h] ? rcp_approx(sums[2 * h]) : 0.0f;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int h = 0; h < 2; h++)
                *reinterpret_cast<uint32_t *>(buf + TL::at(g4 + 8 * h, d) + t4 * 4) =
                    pack2<T>(o[d][2 * h] * inv[h], o[d][2 * h + 1] * inv[h]);
        __syncwarp();
#pragma unroll
        for (int k = 0; k < NC; k++) {
            const int r = lr + k * RS;
            if (col && left > k * RS) {
                T *dst = plain ? op + k * RS * a.old
                               : ob + row_at(w0 + (uint32_t)i * a.cs * 64 + r, a.old, a.os1) + lc * EPC;
                const uint4 w = *reinterpret_cast<const uint4 *>(buf + TL::at(r, lc));
                if (a.ovec)
                    *reinterpret_cast<uint4 *>(dst) = w;
                else {
                    const T *e8 = reinterpret_cast<const T *>(&w);
#pragma unroll
                    for (int e = 0; e < EPC; e++)
                        dst[e] = e8[e];
                }
            }
        }
        op += ostep;
        left -= a.cs * 64;
        __syncwarp();
    }
    cp_wait<0>();
    griddep_launch();
}

// CTAs of a kernel that run at the same time.
template <auto Kern>
long resident(int smem)
{
    return (long)ctas_of_sm<Kern>(kThreads, smem) * device_sms();
}

template <typename T, int HDP, int KT>
int launch_few(XaArgs &a, int nb, cudaStream_t s)
{
    using TL = Tile<T, HDP>;
    constexpr int smem = 2 * KT * 16 * TL::PITCH + 4 * 3 * 16 * TL::PITCH;
    const cudaError_t e = smem_limit_once<attn_few_kernel<T, HDP, KT>>(smem);
    if (e != cudaSuccess)
        return (int)e;
    a.nqt = (int)((a.rows + 63) / 64);
    // CTAs of a head: all that run at once
    const long heads = (long)nb * a.kvheads, want = resident<attn_few_kernel<T, HDP, KT>>(smem) / heads;
    a.cs = (int)(want < 1 ? 1 : (want < a.nqt ? want : a.nqt));
    if (heads > 0x7fffffffL / a.cs)
        return K_EARG;
    return launch_pdl(attn_few_kernel<T, HDP, KT>, dim3((unsigned)(heads * a.cs)), dim3(kThreads), smem, s,
                      (const XaArgs)a);
}

template <typename T, int HDP>
int launch_few_k(XaArgs &a, int nb, cudaStream_t s)
{
    switch ((a.Nk + 15) / 16) {
    case 1:
        return launch_few<T, HDP, 1>(a, nb, s);
    case 2:
        return launch_few<T, HDP, 2>(a, nb, s);
    case 3:
        return launch_few<T, HDP, 3>(a, nb, s);
    default:
        return launch_few<T, HDP, 4>(a, nb, s);
    }
}

template <typename T, int HDP, int WM>
int launch(XaArgs &a, int nb, cudaStream_t s)
{
    using CF = Cfg<T, HDP, WM>;
    const cudaError_t pe = cluster_prepare_once<attn_cross_kernel<T, HDP, WM>>(CF::SMEM_PARTS);
    if (pe != cudaSuccess)
        return (int)pe;
    constexpr int BM = 16 * WM;
    const long nqt = (a.rows + BM - 1) / BM;
    if (nqt > 0x7fffffffL)
        return K_EARG;
    a.nqt = (int)nqt;
    const long items = (long)nb * a.kvheads * nqt;
    // CTAs sharing a tile's keys: while all run at once, each with at least
    // two steps, and a cluster of them fits the device.
    const long slots = resident<attn_cross_kernel<T, HDP, WM>>(CF::SMEM_PARTS), steps = (a.Nk + CF::BK - 1) / CF::BK;
    a.cs = 1;
    while (a.cs < kMaxCluster && items * a.cs * 2 <= slots && steps >= a.cs * kSplitSteps &&
           clusters_at_once<attn_cross_kernel<T, HDP, WM>>(a.cs * 2, kThreads, CF::SMEM_PARTS) > 0)
        a.cs *= 2;
    if (items > 0x7fffffffL / a.cs)
        return K_EARG;
    const int smem = a.cs > 1 ? CF::SMEM_PARTS : CF::SMEM_WHOLE;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.cs;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(items * a.cs));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = a.cs > 1 ? 2 : 1;
    return (int)cudaLaunchKernelEx(&cfg, attn_cross_kernel<T, HDP, WM>, (const XaArgs)a);
}

template <typename T>
int launch_t(XaArgs &a, int nb, cudaStream_t s)
{
    const bool few = a.rows <= 16;
    if constexpr (sizeof(T) == 2) {
        if (a.Nk <= 64 && !few && a.rows < 0x7fffff00L)
            return a.hd <= 32 ? launch_few_k<T, 32>(a, nb, s)
                              : (a.hd <= 64 ? launch_few_k<T, 64>(a, nb, s) : launch_few_k<T, 128>(a, nb, s));
    }
    if (a.hd <= 32)
        return few ? launch<T, 32, 1>(a, nb, s) : launch<T, 32, 4>(a, nb, s);
    if (a.hd <= 64)
        return few ? launch<T, 64, 1>(a, nb, s) : launch<T, 64, 4>(a, nb, s);
    return few ? launch<T, 128, 1>(a, nb, s) : launch<T, 128, 4>(a, nb, s);
}

}  // namespace
}  // namespace sam3

extern "C" int k_cross_attend(const struct k_rows *Q, const struct k_rows *K, const struct k_rows *V,
                              const struct k_rows *O, int nb, int Nq, int Nk, int heads, int kvheads,
                              int hd, const int *klen, const unsigned char *kmask, float scale,
                              int *err, k_stream s)
{
    using namespace sam3;
    if (nb <= 0 || Nq <= 0 || Nk <= 0 || heads <= 0 || kvheads <= 0 || heads % kvheads || hd <= 0 ||
        hd > 128 || hd % 8)
        return K_EARG;
    const int es = Q->dt == K_F32 ? 4 : 2;
    auto vec = [&](const struct k_rows *x) {
        const long m = 16 / es;
        return !(reinterpret_cast<uintptr_t>(x->p) & 15) && x->ld % m == 0 && x->s0 % m == 0 && x->s1 % m == 0;
    };
    auto pairs = [&](const struct k_rows *x) {
        return !(reinterpret_cast<uintptr_t>(x->p) & (2 * es - 1)) && x->ld % 2 == 0 && x->s0 % 2 == 0 &&
               x->s1 % 2 == 0;
    };
    XaArgs a = {};
    a.q = Q->p;
    a.k = K->p;
    a.v = V->p;
    a.o = O->p;
    a.qld = Q->ld, a.qs0 = Q->s0, a.qs1 = Q->s1;
    a.kld = K->ld, a.ks0 = K->s0, a.ks1 = K->s1;
    a.vld = V->ld, a.vs0 = V->s0, a.vs1 = V->s1;
    a.old = O->ld, a.os0 = O->s0, a.os1 = O->s1;
    a.klen = klen;
    a.kmask = kmask;
    a.Nq = Nq;
    a.Nk = Nk;
    a.heads = heads;
    a.kvheads = kvheads;
    a.g = heads / kvheads;
    a.hd = hd;
    a.rows = (long)Nq * a.g;
    a.qvec = vec(Q);
    a.kvec = vec(K) && vec(V);
    a.ovec = pairs(O);
    a.dg = make_div(a.g);
    if (es == 2 && Nk <= 64 && a.rows > 16)
        a.ovec = vec(O);  // the form for few keys stores 16 bytes
    a.scale_log2 = (float)(scale * 1.4426950408889634);
    a.err = err;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(s);
    // Many rows over many keys: tcgen05. Both forms were measured over 1 to 1024
    // queries and 96 to 4096 keys (us, tcgen05 / this file): 128 columns a head
    // 128 heads, 1 query x 4096 keys 46 / 71 (8 heads, 8192 keys 22.0 / 18.8), 128 x
    // 4096 53 / 145;
    // 64 columns, 32 heads, 48 x 384 7.0 / 8.4, 48 x 1024 11.6 / 12.1 (1.6 M
    // scores), 128 x 1024 14.4 / 12.1 (4.2 M), 256 x 1024 15.1 / 17.0 (8.4 M);
    // 32 columns, 64 heads, 64 x 192 5.6 / 4.8, 64 x 384 7.2 / 7.2, 96 x 1024
    // 14.2 / 13.7 (6.3 M), 96 x 2048 17.1 / 22.7. Heads sharing keys are rows of
    // one tile here, so few queries of theirs stay.
    const double scores = (double)nb * heads * Nq * Nk;
    const bool mid = Nk < 640, big = scores >= 6e6;
    const bool many = hd > 64   ? Nk >= 96 && (Nq >= 16 || (a.g == 1 && (long)nb * heads >= 64))
                      : hd > 32 ? Nq >= 24 && (mid ? Nk >= 96 : big)
                                : (Nq >= 64 && mid && Nk >= 256) || (Nq >= 24 && Nk >= 96 && big);
    if (many && attn_cross_tc_takes(a, nb, Q->dt)) {
        a.ovec = vec(O);
        const int rc = attn_cross_tc(a, nb, Q->dt, st);
        if (rc != K_ETMAP)
            return rc;
        a.ovec = pairs(O);
    }
    if (Q->dt == K_F32)
        return launch_t<float>(a, nb, st);
    if (Q->dt == K_BF16)
        return launch_t<__nv_bfloat16>(a, nb, st);
    return launch_t<__half>(a, nb, st);
}
