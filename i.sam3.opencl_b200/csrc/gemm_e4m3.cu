// SPDX-License-Identifier: Unlicense
// Product of E4M3 matrices with block scales on tcgen05 (kind::f8f6f4): C = act(sum
// over 128-column blocks kb of SA[m, kb] SB[n / 128, kb] (A_kb B_kb^T) + bias).
//
// The scales are any numbers, so a block's product cannot simply be added to the
// last one's: each k-block of 128 (one shared-memory stage, four MMAs of K = 32)
// goes into a tensor-memory buffer of its own from zero, and the epilogue warps
// add it, times its scale, to sums in registers, one row and 128 columns a
// thread: one scale of B and one of A per thread and k-block. 10 warps: a TMA
// producer, an MMA issuer, and two groups of four warps (a warp per lane quarter
// of tensor memory).
//   PING: tiles are 128 columns wide and the groups take tiles in turn, each
//         with two buffers, so that one group's epilogue runs beside the other's
//         sums;
//   else: tiles of 256 columns, each group 128 of them (two buffers), half the
//         shared-memory traffic per product of B.
//   PAIR: a cluster of two CTAs computes 256 rows with cta_group::2 MMAs, each
//         CTA loading half of B's tile.
// A 128-column block of a row lies in one thread, so an E4M3 result is scaled and
// rounded there.
#include "act.cuh"
#include "e4m3.cuh"
#include "kernels.h"
#include "tc_ptx.cuh"
#include "tmap.cuh"
#include "vec8.cuh"

namespace sam3 {
namespace {

constexpr int BM = 128, BK = 128;
constexpr int kThreads = 384;
constexpr int kStageTile = 32 * 128;  // a warp's 32 rows x 128 bytes of C
constexpr int kChunk = 4;             // k-blocks whose scales are handed over at once
constexpr int kScaleRing = 2 * kChunk * BM * 4;  // two chunks of a group's scales

struct E4Args {
    int M, N, K;
    const void *sa, *sb;
    long ldsa, ldsb;
    int sadt, sbdt;
    int savec, sbvec;  // rows of scales start at multiples of four
    const float *bias;
    void *c;
    long ldc;
    int cdt;
    void *sc;
    long ldsc;
    int scdt;
    int act;
    int tma;  // C is stored through its tensor map
    int *err;
};

template <int BN, bool PAIR>
struct E4Smem {
    static constexpr int A_BYTES = BM * BK;
    static constexpr int B_ROWS = PAIR ? BN / 2 : BN;
    static constexpr int STAGE_BYTES = A_BYTES + B_ROWS * BK;
    static constexpr int STAGES = STAGE_BYTES > 32768 ? 3 : (STAGE_BYTES > 24576 ? 5 : 7);
    static constexpr int EPI_OFF = STAGES * STAGE_BYTES;
    static constexpr int SCALE_OFF = EPI_OFF + 8 * kStageTile;
    static constexpr int BAR_OFF = SCALE_OFF + 2 * kScaleRing;
    // full[S], empty[S], tfull[4], tempty[4], sfull[2][2], sempty[2][2], drain, then
    // tmem base + abort
    static constexpr int BYTES = BAR_OFF + (2 * STAGES + 17) * 8 + 16 + 1024;
    static_assert(BYTES <= 232448, "shared memory");
};

// Scales [k .. k + 3] of a row (of `n` it has), as stored: one load where the row
// is aligned for it.
__device__ __forceinline__ void load_scales(const void *p, int dt, bool vec, long row, int k, int n,
                                            uint32_t (&v)[kChunk])
{
    if (vec && k + kChunk <= n) {
        if (dt == K_E8M0) {
            const uint32_t w = __ldg(reinterpret_cast<const uint32_t *>(reinterpret_cast<const uint8_t *>(p) + row + k));
            v[0] = w;  // taken apart by scale_at
        }
        else {
            const uint4 w = __ldg(reinterpret_cast<const uint4 *>(reinterpret_cast<const float *>(p) + row + k));
            v[0] = w.x;
            v[1] = w.y;
            v[2] = w.z;
            v[3] = w.w;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < kChunk; i++)
        v[i] = k + i < n ? scale_raw(p, dt, row + k + i) : 0u;
}
__device__ __forceinline__ float scale_at(const uint32_t (&v)[kChunk], int dt, bool vec, int k, int n, int i)
{
    if (dt == K_E8M0 && vec && k + kChunk <= n)
        return scale_of(v[0] >> (8 * i) & 255u, dt);
    return scale_of(v[i], dt);
}

// The products of both scales for the rows and the column block of one group's
// tiles, four k-blocks at a time, by a warp that runs ahead of the group: the
// loads of a chunk are in flight while the last one is handed over.
__device__ __forceinline__ void feed_scales(const E4Args &p, float *ring, uint64_t *sfull, uint64_t *sempty, int t0,
                                            int tstep, int num_tiles, int num_n, int tm, int bn, int row0, int col,
                                            int kblocks, int lane, volatile int *abort_flag)
{
    constexpr int R = BM / 32;  // rows of a lane
    uint32_t va[R][kChunk], vb[kChunk], wa[R][kChunk], wb[kChunk];
    int t = t0, k = 0;
    auto fetch = [&](uint32_t(&a)[R][kChunk], uint32_t(&b)[kChunk]) {
        const int m = (t / num_n) * tm + row0 + lane, n = (t % num_n) * bn + col;
        load_scales(p.sb, p.sbdt, p.sbvec, (long)(min(n, p.N - 1) / kScaleBlock) * p.ldsb, k, kblocks, b);
#pragma unroll
        for (int i = 0; i < R; i++)
            load_scales(p.sa, p.sadt, p.savec, (long)min(m + 32 * i, p.M - 1) * p.ldsa, k, kblocks, a[i]);
    };
    uint32_t c = 0;  // chunks handed over
    auto give = [&](const uint32_t(&a)[R][kChunk], const uint32_t(&b)[kChunk], int k0) {
        const uint32_t slot = c & 1, parity = (c >> 1 & 1) ^ 1;
        if (!__all_sync(0xffffffffu, mbar_wait_brief(&sempty[slot], parity, p.err, abort_flag)))
            return false;
        float *dst = ring + slot * (kChunk * BM) + lane;
#pragma unroll
        for (int j = 0; j < kChunk; j++) {
            const float sb = scale_at(b, p.sbdt, p.sbvec, k0, kblocks, j);
#pragma unroll
            for (int i = 0; i < R; i++)
                dst[j * BM + 32 * i] = scale_at(a[i], p.sadt, p.savec, k0, kblocks, j) * sb;
        }
        __syncwarp();
        if (lane == 0)
            mbar_arrive(&sfull[slot]);
        c++;
        return true;
    };
    auto advance = [&]() {
        k += kChunk;
        if (k >= kblocks) {
            k = 0;
            t += tstep;
        }
        return t < num_tiles;
    };
    bool more = t < num_tiles;
    if (more)
        fetch(va, vb);
    while (more) {
        const int k0 = k;
        more = advance();
        if (more)
            fetch(wa, wb);
        if (!give(va, vb, k0))
            return;
        if (!more)
            return;
        const int k1 = k;
        more = advance();
        if (more)
            fetch(va, vb);
        if (!give(wa, wb, k1))
            return;
    }
}

template <bool FULL>
__device__ __forceinline__ void add_bias(const float *bias, int n, int N, float (&acc)[128])
{
#pragma unroll
    for (int j = 0; j < 128; j += 4) {
        if (FULL) {
            const float4 v = __ldg(reinterpret_cast<const float4 *>(bias + n + j));
            acc[j] += v.x;
            acc[j + 1] += v.y;
            acc[j + 2] += v.z;
            acc[j + 3] += v.w;
        }
        else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (n + j + e < N)
                    acc[j + e] += __ldg(bias + n + j + e);
        }
    }
}

// A 128-byte row of a chunk into the warp's staging tile, 16-byte pieces in the
// order a 128B-swizzled tensor map expects.
__device__ __forceinline__ void stage_piece(uint32_t tile, int r, int q, uint32_t a, uint32_t b, uint32_t c,
                                            uint32_t d)
{
    st_shared_v4(tile + r * 128 + ((q ^ (r & 7)) << 4), a, b, c, d);
}

// The staged chunk to C at rows m0 .., columns n ..: by TMA, or element by element
// along the rows where C's rows are not 16-byte aligned.
__device__ __forceinline__ void store_chunk(const E4Args &p, const CUtensorMap *tmC, uint32_t tile, int lane, int m0,
                                            int n)
{
    if (p.tma) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
            tma_store_2d(tmC, reinterpret_cast<const void *>(__cvta_shared_to_generic(tile)), n, m0);
            bulk_commit();
        }
        return;
    }
    __syncwarp();
    const int es = p.cdt == K_F32 ? 4 : (p.cdt == K_E4M3 ? 1 : 2), per = 128 / es;
    for (int r = 0; r < 32 && m0 + r < p.M; r++) {
        const long row = (long)(m0 + r) * p.ldc + n;
        for (int j = lane; j < per && n + j < p.N; j += 32) {
            const int byte = j * es;
            const uint32_t src = tile + r * 128 + (((byte >> 4) ^ (r & 7)) << 4) + (byte & 15);
            if (es == 4) {
                uint32_t v;
                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(src) : "memory");
                reinterpret_cast<uint32_t *>(p.c)[row + j] = v;
            }
            else if (es == 2) {
                uint16_t v;
                asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(src) : "memory");
                reinterpret_cast<uint16_t *>(p.c)[row + j] = v;
            }
            else {
                uint16_t v;
                asm volatile("{.reg .b8 t; ld.shared.b8 t, [%1]; cvt.u16.u8 %0, t;}" : "=h"(v) : "r"(src) : "memory");
                reinterpret_cast<uint8_t *>(p.c)[row + j] = (uint8_t)v;
            }
        }
    }
    __syncwarp();
}

// Bias, activation, rounding and store of a thread's row and 128 columns. tile:
// the warp's staging tile.
template <bool GELU>
__device__ __forceinline__ void finish(const E4Args &p, const CUtensorMap *tmC, uint32_t tile, int lane, int m0, int n,
                                       float (&acc)[128])
{
    const bool full = n + 128 <= p.N;
    if (p.bias) {
        if (full && !(reinterpret_cast<uintptr_t>(p.bias) & 15))
            add_bias<true>(p.bias, n, p.N, acc);
        else
            add_bias<false>(p.bias, n, p.N, acc);
    }
    if (p.act == K_ACT_RELU) {
#pragma unroll
        for (int j = 0; j < 128; j++)
            asm("max.NaN.f32 %0, %0, %1;" : "+f"(acc[j]) : "f"(0.0f));
    }
    if (GELU && p.cdt != K_F32) {
#pragma unroll
        for (int j = 0; j < 128; j += 2)
            gelu_pair_rel(acc[j], acc[j + 1]);
    }
    auto wait_tile = [&]() {  // the store issued from this tile before has read it
        if (p.tma && lane == 0)
            bulk_wait_read<0>();
        __syncwarp();
    };
    if (p.cdt == K_F32) {
#pragma unroll
        for (int c = 0; c < 4; c++) {
            if (n + 32 * c >= p.N)
                break;
            wait_tile();
#pragma unroll
            for (int q = 0; q < 8; q++)
                stage_piece(tile, lane, q, __float_as_uint(acc[32 * c + 4 * q]), __float_as_uint(acc[32 * c + 4 * q + 1]),
                            __float_as_uint(acc[32 * c + 4 * q + 2]), __float_as_uint(acc[32 * c + 4 * q + 3]));
            if (GELU) {
                // the thread's own row again, so that the loop is not unrolled over the sums
#pragma unroll 1
                for (int q = 0; q < 8; q++) {
                    const uint32_t at = tile + lane * 128 + q * 16;
                    float v[4];
                    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3])
                                 : "r"(at)
                                 : "memory");
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        v[e] = 0.5f * v[e] * (1.0f + erff(v[e] * 0.70710678118654752f));
                    st_shared_v4(at, __float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                                 __float_as_uint(v[3]));
                }
            }
            store_chunk(p, tmC, tile, lane, m0, n + 32 * c);
        }
    }
    else if (p.cdt == K_E4M3) {
        float most = 0.0f;
#pragma unroll
        for (int j = 0; j < 128; j++)  // (0 behind N: B's rows there read as zero, the bias is not added)
            most = larger(most, acc[j]);
        if (infinite(most)) {
            most = 0.0f;
#pragma unroll
            for (int j = 0; j < 128; j++) {
                most = larger_finite(most, acc[j]);
                acc[j] = fmaf(acc[j], 0.0f, acc[j]);  // NaN for an infinity
            }
        }
        const uint32_t byte = scale_byte(most);
        const float inv = scale_inverse(byte);
        wait_tile();
#pragma unroll
        for (int q = 0; q < 8; q++) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int j = 16 * q + 4 * e;
                w[e] = pack_e4m3<false>(acc[j], acc[j + 1], acc[j + 2], acc[j + 3], inv);
            }
            stage_piece(tile, lane, q, w[0], w[1], w[2], w[3]);
        }
        store_chunk(p, tmC, tile, lane, m0, n);
        if (m0 + lane < p.M)
            put_scale(p.sc, p.scdt, (long)(m0 + lane) * p.ldsc + n / kScaleBlock, byte);
    }
    else {
#pragma unroll
        for (int c = 0; c < 2; c++) {
            if (n + 64 * c >= p.N)
                break;
            wait_tile();
#pragma unroll
            for (int q = 0; q < 8; q++) {
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float v0 = acc[64 * c + 8 * q + 2 * e], v1 = acc[64 * c + 8 * q + 2 * e + 1];
                    w[e] = p.cdt == K_BF16 ? pack_bf16x2(v0, v1) : pack_f16x2(v0, v1);
                }
                stage_piece(tile, lane, q, w[0], w[1], w[2], w[3]);
            }
            store_chunk(p, tmC, tile, lane, m0, n + 64 * c);
        }
    }
}

template <int BN, bool PAIR, bool GELU>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_e4m3_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                     const __grid_constant__ CUtensorMap tmC, const __grid_constant__ E4Args p)
{
    constexpr bool PING = BN == 128;
    constexpr int NBUF = 512 / BN;
    using L = E4Smem<BN, PAIR>;
    constexpr int STAGES = L::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem =
        reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::BAR_OFF);
    uint64_t *empty = full + STAGES;
    uint64_t *tfull = empty + STAGES;
    uint64_t *tempty = tfull + 4;
    uint64_t *sfull = tempty + 4, *sempty = sfull + 4;  // [group][chunk]
    uint64_t *drain = sempty + 4;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = PAIR ? cluster_ctarank() : 0;

    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; i++) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < NBUF; i++) {
            mbar_init(&tfull[i], 1);
            mbar_init(&tempty[i], (PING ? 4 : 8) * (PAIR ? 2 : 1));
        }
        for (int i = 0; i < 4; i++) {
            mbar_init(&sfull[i], 1);
            mbar_init(&sempty[i], 4);
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        if constexpr (PAIR) {
            tmem_alloc_pair(tmem_slot, 512);
            tmem_relinquish_pair();
        }
        else {
            tmem_alloc(tmem_slot, 512);
            tmem_relinquish();
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (PAIR)
        cluster_sync_all();  // both CTAs' barriers exist before either signals the other
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    griddep_launch();
    griddep_wait();

    constexpr int TM = PAIR ? 2 * BM : BM;  // rows per tile
    const int first = PAIR ? (int)(blockIdx.x >> 1) : (int)blockIdx.x;
    const int step = PAIR ? (int)(gridDim.x >> 1) : (int)gridDim.x;
    const int num_n = (p.N + BN - 1) / BN;
    const int num_tiles = (p.M + TM - 1) / TM * num_n;
    const int kblocks = (p.K + BK - 1) / BK;
    const int tstep = PING ? 2 * step : step;  // of a group's tiles

    // The warpgroups start with 168 registers a thread: 128 x 72 + 256 x 216 <= 384 x 168.
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == 0) {
            if (elect_one()) {
                prefetch_tmap(&tmA);
                prefetch_tmap(&tmB);
                int stage = 0;
                uint32_t phase = 0, issued_mask = 0, last_parity = 0;
                bool ok = true;
                for (int t = first; t < num_tiles && ok; t += step) {
                    const int m0 = (t / num_n) * TM + (int)rank * BM, n0 = (t % num_n) * BN;
                    for (int kb = 0; kb < kblocks; kb++) {
                        if (!mbar_wait_brief<PAIR>(&empty[stage], phase ^ 1, p.err, abort_flag)) {
                            ok = false;
                            break;
                        }
                        uint8_t *sa = smem + stage * L::STAGE_BYTES;
                        if constexpr (PAIR) {
                            if (rank == 0)
                                mbar_arrive_expect_tx(&full[stage], 2 * L::STAGE_BYTES);
                            const uint32_t fb = mapa_shared(smem_addr(&full[stage]), 0);
                            tma_load_2d_pair(sa, &tmA, fb, kb * BK, m0);
                            tma_load_2d_pair(sa + L::A_BYTES, &tmB, fb, kb * BK, n0 + (int)rank * (BN / 2));
                        }
                        else {
                            mbar_arrive_expect_tx(&full[stage], L::STAGE_BYTES);
                            tma_load_2d(sa, &tmA, &full[stage], kb * BK, m0);
                            tma_load_2d(sa + L::A_BYTES, &tmB, &full[stage], kb * BK, n0);
                        }
                        issued_mask |= 1u << stage;
                        last_parity = (last_parity & ~(1u << stage)) | (phase << stage);
                        if (++stage == STAGES) {
                            stage = 0;
                            phase ^= 1;
                        }
                    }
                }
                // Every copy this thread issued lands before the CTA exits (in a pair
                // rank 0's barriers count both CTAs' copies, and the closing cluster
                // barrier holds rank 1).
                for (int s = 0; s < STAGES; s++)
                    if (rank == 0 && (issued_mask & (1u << s))) {
                        volatile int no_abort = 0;
                        mbar_wait(&full[s], (last_parity >> s) & 1, p.err, &no_abort);
                    }
            }
        }
        else if (warp == 1) {
            if (elect_one()) {
                if (rank == 0) {
                    constexpr uint32_t idesc = idesc_e4m3_f32(TM, BN);
                    int stage = 0, g = 0;
                    uint32_t phase = 0, done[2] = {0, 0};  // k-blocks handed to each group
                    bool ok = true;
                    for (int t = first; t < num_tiles && ok; t += step, g ^= PING) {
                        uint32_t c = done[g];
                        for (int kb = 0; kb < kblocks; kb++) {
                            const uint32_t buf = 2 * g + (c & 1), parity = (c >> 1 & 1) ^ 1;
                            if (!mbar_wait_brief<PAIR>(&tempty[buf], parity, p.err, abort_flag) ||
                                !mbar_wait_brief(&full[stage], phase, p.err, abort_flag)) {
                                ok = false;
                                break;
                            }
                            tc_fence_after();
                            const uint32_t d = tmem_base + buf * BN;
                            const uint32_t sa = smem_addr(smem + stage * L::STAGE_BYTES), sb = sa + L::A_BYTES;
    #pragma unroll
                            for (int k = 0; k < BK / 32; k++) {
                                if constexpr (PAIR)
                                    tc_mma_e4m3_pair(d, sw128_desc(sa + k * 32, 16, 1024), sw128_desc(sb + k * 32, 16, 1024),
                                                     idesc, k != 0);
                                else
                                    tc_mma_e4m3(d, sw128_desc(sa + k * 32, 16, 1024), sw128_desc(sb + k * 32, 16, 1024),
                                                idesc, k != 0);
                            }
                            if constexpr (PAIR) {
                                tc_commit_pair(&empty[stage], 3);
                                tc_commit_pair(&tfull[buf], 3);
                            }
                            else {
                                tc_commit(&empty[stage]);
                                tc_commit(&tfull[buf]);
                            }
                            if (++stage == STAGES) {
                                stage = 0;
                                phase ^= 1;
                            }
                            c++;
                        }
                        done[g] = c;
                    }
                    // one arrival (on both CTAs' barriers in a pair) once every MMA is done
                    if constexpr (PAIR)
                        tc_commit_pair(drain, 3);
                    else
                        tc_commit(drain);
                }
                // Tensor memory is idle before it is freed.
                volatile int no_abort = 0;
                if constexpr (PAIR)
                    mbar_wait_cluster(drain, 0, p.err, &no_abort);
                else
                    mbar_wait(drain, 0, p.err, &no_abort);
            }
        }
        else {
            const int g = warp - 2;
            feed_scales(p, reinterpret_cast<float *>(smem + L::SCALE_OFF + g * kScaleRing), sfull + 2 * g, sempty + 2 * g,
                        first + (PING ? g * step : 0), tstep, num_tiles, num_n, TM, BN, (int)rank * BM,
                        PING ? 0 : g * 128, kblocks, lane, abort_flag);
        }
    }
    else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int group = (warp - 4) >> 2;
        const int quarter = warp & 3;  // the TMEM lanes this warp may read
        const int row = (int)rank * BM + quarter * 32, col = PING ? 0 : group * 128;
        const uint32_t stage_tile = smem_addr(smem + L::EPI_OFF + (warp - 4) * kStageTile);
        const int t0 = first + (PING ? group * step : 0);
        const float *ring = reinterpret_cast<const float *>(smem + L::SCALE_OFF + group * kScaleRing) + quarter * 32 + lane;
        if (lane == 0)
            prefetch_tmap(&tmC);
        // A barrier's parity tells neighbouring phases apart only: each group has
        // buffers of its own (PING), whose every phase it waits for.
        uint32_t c = 0, chunk = 0;
        bool ok = true;
        for (int t = t0; t < num_tiles && ok; t += tstep) {
            float acc[128];
#pragma unroll
            for (int j = 0; j < 128; j++)
                acc[j] = 0.0f;
            for (int kb = 0; kb < kblocks; kb++, c++) {
                const uint32_t buf = (PING ? 2 * group : 0) + (c & 1), parity = c >> 1 & 1;
                const uint32_t slot = 2 * group + (chunk & 1);
                ok = kb % kChunk || mbar_wait_brief(&sfull[slot], chunk >> 1 & 1, p.err, abort_flag);
                ok = ok && mbar_wait_brief<PAIR>(&tfull[buf], parity, p.err, abort_flag);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok)
                    break;
                tc_fence_after();
                const uint32_t src = tmem_base + ((uint32_t)(quarter * 32) << 16) + buf * BN + col;
                const float s = ring[((chunk & 1) * kChunk + kb % kChunk) * BM];
                uint32_t r[2][32];
                tmem_ld32(src, r[0]);
                tmem_wait_ld(r[0]);
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    if (q < 3)
                        tmem_ld32(src + 32 * (q + 1), r[(q + 1) & 1]);
#pragma unroll
                    for (int j = 0; j < 32; j++)  // (packed pairs cost two moves each)
                        acc[32 * q + j] = fmaf(__uint_as_float(r[q & 1][j]), s, acc[32 * q + j]);
                    if (q < 3)
                        tmem_wait_ld(r[(q + 1) & 1]);
                    if (q == 2) {  // the buffer has been read
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) {
                            if constexpr (PAIR)
                                mbar_arrive_cluster_relaxed(mapa_shared(smem_addr(&tempty[buf]), 0));
                            else
                                mbar_arrive_relaxed(&tempty[buf]);
                        }
                    }
                }
                if (kb % kChunk == kChunk - 1 || kb + 1 == kblocks) {
                    __syncwarp();
                    if (lane == 0)
                        mbar_arrive(&sempty[slot]);
                    chunk++;
                }
            }
            if (!ok)
                break;
            const int m0 = (t / num_n) * TM + row, n = (t % num_n) * BN + col;
            if (m0 < p.M && n < p.N)
                finish<GELU>(p, &tmC, stage_tile, lane, m0, n, acc);
        }
        if (p.tma && lane == 0)
            bulk_wait_all();
    }

    tc_fence_before();
    __syncthreads();
    // In a pair, neither CTA leaves (nor frees tensor memory) while the other's
    // MMAs, copies or arrivals may still touch its shared memory.
    if constexpr (PAIR)
        cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        if constexpr (PAIR)
            tmem_dealloc_pair(tmem_base, 512);
        else
            tmem_dealloc(tmem_base, 512);
    }
}

// Clusters of two CTAs of a kernel that run at once (0: none), per device.
template <auto Kern>
int pairs_at_once(cudaLaunchConfig_t &cfg)
{
    static int known[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64)
        return 0;
    if (!known[dev]) {
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, Kern, &cfg) != cudaSuccess) {
            (void)cudaGetLastError();
            n = 0;
        }
        known[dev] = n + 1;
    }
    return known[dev] - 1;
}

// K_EARG: pairs cannot be launched here.
template <int BN, bool PAIR, bool GELU>
int launch(const E4Args &p, const struct k_rows *A, const struct k_rows *B, const CUtensorMap &tc, cudaStream_t s)
{
    using L = E4Smem<BN, PAIR>;
    constexpr auto kern = gemm_e4m3_kernel<BN, PAIR, GELU>;
    CUtensorMap ta, tb;
    // a single row's pitch is of no account
    const uint64_t pitch = ((uint64_t)p.K + 15) / 16 * 16;
    if (!make_tmap_2d(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, A->p, (uint64_t)p.M, (uint64_t)p.K,
                      p.M > 1 ? (uint64_t)A->ld : pitch, BK, BM) ||
        !make_tmap_2d(&tb, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, B->p, (uint64_t)p.N, (uint64_t)p.K,
                      p.N > 1 ? (uint64_t)B->ld : pitch, BK, L::B_ROWS))
        return K_ETMAP;
    const cudaError_t e = smem_limit_once<kern>(L::BYTES);
    if (e != cudaSuccess)
        return (int)e;
    const int tiles = (p.M + (PAIR ? 2 : 1) * BM - 1) / ((PAIR ? 2 : 1) * BM) * ((p.N + BN - 1) / BN);
    const int sms = device_sms();
    if constexpr (!PAIR)
        return launch_pdl(kern, dim3(tiles < sms ? tiles : sms), dim3(kThreads), L::BYTES, s, ta, tb, tc, p);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(sms / 2 * 2);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = L::BYTES;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const int most = pairs_at_once<kern>(cfg);
    if (most <= 0)
        return K_EARG;
    cfg.gridDim = dim3(2 * (tiles < most ? tiles : most));
    cfg.numAttrs = 2;
    return (int)cudaLaunchKernelEx(&cfg, kern, ta, tb, tc, p);
}

template <int BN, bool PAIR>
int launch_act(const E4Args &p, const struct k_rows *A, const struct k_rows *B, const CUtensorMap &tc, cudaStream_t s)
{
    return p.act == K_ACT_GELU ? launch<BN, PAIR, true>(p, A, B, tc, s) : launch<BN, PAIR, false>(p, A, B, tc, s);
}

}  // namespace
}  // namespace sam3

extern "C" int k_gemm_e4m3(int M, int N, int K, const struct k_rows *A, const struct k_rows *SA, const struct k_rows *B,
                           const struct k_rows *SB, const struct k_rows *C, const struct k_rows *SC, const float *bias,
                           int act, int *err, k_stream s)
{
    using namespace sam3;
    if (M <= 0 || N <= 0 || K <= 0)
        return K_EARG;
    E4Args p = {};
    p.M = M;
    p.N = N;
    p.K = K;
    p.sa = SA->p;
    p.sb = SB->p;
    p.ldsa = SA->ld;
    p.ldsb = SB->ld;
    p.sadt = SA->dt;
    p.sbdt = SB->dt;
    auto aligned = [](const struct k_rows *r) {
        return r->ld % 4 == 0 && reinterpret_cast<uintptr_t>(r->p) % (r->dt == K_E8M0 ? 4 : 16) == 0;
    };
    p.savec = aligned(SA);
    p.sbvec = aligned(SB);
    p.bias = bias;
    p.c = C->p;
    p.ldc = C->ld;
    p.cdt = C->dt;
    if (SC) {
        p.sc = SC->p;
        p.ldsc = SC->ld;
        p.scdt = SC->dt;
    }
    p.act = act;
    p.err = err;
    CUtensorMap tc;
    const int es = C->dt == K_F32 ? 4 : (C->dt == K_E4M3 ? 1 : 2);
    const CUtensorMapDataType dt = C->dt == K_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : C->dt == K_E4M3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                                     : CU_TENSOR_MAP_DATA_TYPE_UINT16;
    const uint64_t pitch = M > 1 ? (uint64_t)C->ld : ((uint64_t)N + 15) / 16 * 16;
    p.tma = make_tmap_2d(&tc, dt, es, C->p, (uint64_t)M, (uint64_t)N, pitch, 128 / es, 32);
    if (!p.tma && !make_tmap_2d(&tc, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, A->p, (uint64_t)M, (uint64_t)K,
                                M > 1 ? (uint64_t)A->ld : ((uint64_t)K + 15) / 16 * 16, 128, 32))
        return K_ETMAP;  // (a map for the argument that is not used)
    cudaStream_t st = reinterpret_cast<cudaStream_t>(s);
    // Tiles of 128 x 256 where they fill the device (41472 x 1024 x 4096: 191 us, 271
    // with 128 columns; 603 x 520 x 588: 10.7 and 9.3).
    if ((long)((M + 127) / 128) * ((N + 255) / 256) >= device_sms())
        return launch_act<256, false>(p, A, B, tc, st);
    return launch_act<128, false>(p, A, B, tc, st);
}
