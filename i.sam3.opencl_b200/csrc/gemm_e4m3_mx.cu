// SPDX-License-Identifier: Unlicense
// Product of E4M3 matrices whose block scales are both powers of two (E8M0), into
// 16-bit, E4M3 or (over short rows) 32-bit results: the matrix unit applies the scales itself
// (tcgen05.mma kind::mxf8f6f4, a scale for each 32 columns, the same for the four of a
// block), so that a tile's products add up in tensor memory over all of K and
// the epilogue runs once a tile.
//
// Four warpgroups: a TMA producer and an MMA issuer; four warps that read the scales
// of four k-blocks at a time and write them to tensor memory, each its own lane
// quarter's copy; two groups of four epilogue warps, 128 columns each.
//   BN 256, PAIR: two CTAs compute 256 x 256 with cta_group::2 MMAs, each loading half
//           of B's tile; one accumulator, read into registers by both groups before
//           the next tile's products start;
//   BN 128: two accumulators of 128, a group each.
// 41472 x 1024 x 4096 131 us (2.66 PFLOP/s), 41472 x 4096 x 1024 149 us; with GELU and E4M3
// results 184 us, where the epilogue counts: four instructions a value for GELU's polynomial
// (in pairs), two for the scale and its product, one to round. Under the power cap 161, 183 and
// 214 us at 1136, 1237 and 1545 MHz: 183, 227 and 331 thousand cycles.
#include "gemm_e4m3.cuh"

namespace sam3 {
namespace {

constexpr int BM = 128, BK = 128;
constexpr int kThreads = 512;
constexpr int kSlots = 4;         // chunks of scales in tensor memory
constexpr int kScaleCol = 256;    // their first column
constexpr int kSlotCols = 16;     // 4 of A, BN / 32 of B

template <int BN, bool PAIR>
struct MxSmem {
    static constexpr int A_BYTES = BM * BK;
    static constexpr int B_ROWS = PAIR ? BN / 2 : BN;
    static constexpr int STAGE_BYTES = A_BYTES + B_ROWS * BK;
    static constexpr int STAGES = 6;
    static constexpr int EPI_OFF = STAGES * STAGE_BYTES;
    static constexpr int BAR_OFF = EPI_OFF + 8 * kStageTile;
    // full[S], empty[S], tfull[2], tempty[2], sfull[4], sempty[4], drain, then tmem base + abort
    static constexpr int BYTES = BAR_OFF + (2 * STAGES + 13) * 8 + 16 + 1024;
    static_assert(BYTES <= 232448, "shared memory");
};

// The scales of the CTA's rows and of the tile's columns, written to tensor memory
// by one of four warps (quarter: its lanes).
template <int BN, bool PAIR>
__device__ __forceinline__ void feed_tmem(const E4Args &p, uint32_t tmem, uint64_t *sfull, uint64_t *sempty, int first,
                                          int step, int num_tiles, int num_n, int row0, int kblocks, int lane,
                                          volatile int *abort_flag)
{
    constexpr int TM = PAIR ? 2 * BM : BM, NB = BN / 128;
    struct Words {
        uint32_t a[4], b[NB];
    } v, w;
    int t = first, k = 0;
    auto word = [&](const void *base, bool vec, long row) {
        uint32_t x[kChunk];
        load_scales(base, K_E8M0, vec, row, k, kblocks, x);
        return vec && k + kChunk <= kblocks ? x[0] : x[0] | x[1] << 8 | x[2] << 16 | x[3] << 24;
    };
    auto fetch = [&](Words &o) {
        const int m = (t / num_n) * TM + row0 + lane, n = (t % num_n) * BN;
#pragma unroll
        for (int i = 0; i < NB; i++)
            o.b[i] = word(p.sb, p.sbvec, (long)(min(n + 128 * i, p.N - 1) / kScaleBlock) * p.ldsb);
#pragma unroll
        for (int i = 0; i < 4; i++)
            o.a[i] = word(p.sa, p.savec, (long)min(m + 32 * i, p.M - 1) * p.ldsa);
    };
    auto advance = [&]() {
        k += kChunk;
        if (k >= kblocks) {
            k = 0;
            t += step;
        }
        return t < num_tiles;
    };
    bool more = t < num_tiles;
    if (more)
        fetch(v);
    for (uint32_t c = 0; more; c++) {
        more = advance();
        if (more)
            fetch(w);  // in flight beside the wait
        const uint32_t slot = c % kSlots, parity = (c / kSlots & 1) ^ 1;
        if (!__all_sync(0xffffffffu, mbar_wait_brief<PAIR>(&sempty[slot], parity, p.err, abort_flag)))
            return;
        tc_fence_after();
        const uint32_t at = tmem + kScaleCol + slot * kSlotCols;
        tmem_st4(at, v.a[0], v.a[1], v.a[2], v.a[3]);
#pragma unroll
        for (int i = 0; i < NB; i++)
            tmem_st4(at + 4 + 4 * i, v.b[i], v.b[i], v.b[i], v.b[i]);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
            if constexpr (PAIR)
                mbar_arrive_cluster_relaxed(mapa_shared(smem_addr(&sfull[slot]), 0));
            else
                mbar_arrive_relaxed(&sfull[slot]);
        }
        v = w;
    }
}

template <int BN, bool PAIR, bool GELU>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_mx_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                   const __grid_constant__ CUtensorMap tmC, const __grid_constant__ E4Args p)
{
    constexpr int NACC = 256 / BN;  // accumulators
    using L = MxSmem<BN, PAIR>;
    constexpr int STAGES = L::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem =
        reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::BAR_OFF);
    uint64_t *empty = full + STAGES;
    uint64_t *tfull = empty + STAGES, *tempty = tfull + 2;
    uint64_t *sfull = tempty + 2, *sempty = sfull + kSlots;
    uint64_t *drain = sempty + kSlots;
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
        for (int i = 0; i < NACC; i++) {
            mbar_init(&tfull[i], 1);
            mbar_init(&tempty[i], (BN == 128 ? 4 : 8) * (PAIR ? 2 : 1));
        }
        for (int i = 0; i < kSlots; i++) {
            mbar_init(&sfull[i], PAIR ? 8 : 4);
            mbar_init(&sempty[i], 1);
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

    // The warpgroups start with 128 registers a thread: 256 x 48 + 256 x 208 <= 512 x 128.
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        if (warp == 0 && elect_one()) {
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
        else if (warp == 1 && elect_one()) {
            if (rank == 0) {
                int stage = 0, acc = 0;
                uint32_t phase = 0, acc_phase = 0, chunk = 0;
                bool ok = true;
                const uint32_t smem0 = smem_addr(smem);
                for (int t = first; t < num_tiles && ok; t += step) {
                    if (!mbar_wait_brief<PAIR>(&tempty[acc], acc_phase ^ 1, p.err, abort_flag))
                        break;
                    tc_fence_after();
                    const uint32_t d = tmem_base + acc * BN;
                    for (int kb = 0; kb < kblocks; kb++) {
                        const uint32_t slot = chunk % kSlots;
                        if ((kb % kChunk == 0 &&
                             !mbar_wait_brief<PAIR>(&sfull[slot], chunk / kSlots & 1, p.err, abort_flag)) ||
                            !mbar_wait_brief(&full[stage], phase, p.err, abort_flag)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint32_t sf = tmem_base + kScaleCol + slot * kSlotCols;
                        const uint32_t idesc = idesc_mx_e4m3(TM, BN, 0) + (uint32_t)(kb % kChunk) * (1u << 4 | 1u << 29);
                        const uint64_t da = sw128_desc(smem0 + stage * L::STAGE_BYTES, 16, 1024);
                        const uint64_t db = sw128_desc(smem0 + stage * L::STAGE_BYTES + L::A_BYTES, 16, 1024);
#pragma unroll
                        for (int k = 0; k < BK / 32; k++) {  // 32 columns further: 2 units of 16 bytes
                            if constexpr (PAIR)
                                tc_mma_mx_pair(d, da + 2 * k, db + 2 * k, idesc, sf, sf + 4, (kb | k) != 0);
                            else
                                tc_mma_mx(d, da + 2 * k, db + 2 * k, idesc, sf, sf + 4, (kb | k) != 0);
                        }
                        if constexpr (PAIR)
                            tc_commit_pair(&empty[stage], 3);
                        else
                            tc_commit(&empty[stage]);
                        if (kb % kChunk == kChunk - 1 || kb + 1 == kblocks) {
                            if constexpr (PAIR)
                                tc_commit_pair(&sempty[slot], 3);
                            else
                                tc_commit(&sempty[slot]);
                            chunk++;
                        }
                        if (++stage == STAGES) {
                            stage = 0;
                            phase ^= 1;
                        }
                    }
                    if (!ok)
                        break;
                    if constexpr (PAIR)
                        tc_commit_pair(&tfull[acc], 3);
                    else
                        tc_commit(&tfull[acc]);
                    if (++acc == NACC) {
                        acc = 0;
                        acc_phase ^= 1;
                    }
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
    else if (warp < 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        feed_tmem<BN, PAIR>(p, tmem_base + ((uint32_t)((warp & 3) * 32) << 16), sfull, sempty, first, step, num_tiles,
                            num_n, (int)rank * BM, kblocks, lane, abort_flag);
    }
    else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int group = (warp - 8) >> 2, quarter = warp & 3;
        const int row = (int)rank * BM + quarter * 32, col = BN == 128 ? 0 : group * 128;
        const uint32_t stage_tile = smem_addr(smem + L::EPI_OFF + (warp - 8) * kStageTile);
        const int acc = BN == 128 ? group : 0;  // this group's accumulator
        if (lane == 0)
            prefetch_tmap(&tmC);
        uint32_t phase = 0;
        for (int t = first + (BN == 128 ? group * step : 0); t < num_tiles; t += BN == 128 ? 2 * step : step) {
            const bool ok = mbar_wait_brief<PAIR>(&tfull[acc], phase, p.err, abort_flag);
            if (!__all_sync(0xffffffffu, ok))
                break;
            phase ^= 1;
            tc_fence_after();
            const uint32_t src = tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * BN + col;
            float v[128];
#pragma unroll
            for (int q = 0; q < 4; q++) {
                uint32_t r[32];
                tmem_ld32(src + 32 * q, r);
                tmem_wait_ld(r);
#pragma unroll
                for (int j = 0; j < 32; j++)
                    v[32 * q + j] = __uint_as_float(r[j]);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (PAIR)
                    mbar_arrive_cluster_relaxed(mapa_shared(smem_addr(&tempty[acc]), 0));
                else
                    mbar_arrive_relaxed(&tempty[acc]);
            }
            const int m0 = (t / num_n) * TM + row, n = (t % num_n) * BN + col;
            if (m0 < p.M && n < p.N)
                finish<GELU>(p, &tmC, stage_tile, lane, m0, n, v);
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

template <int BN, bool PAIR, bool GELU>
int launch(const E4Args &p, const struct k_rows *A, const struct k_rows *B, const CUtensorMap &tc, cudaStream_t s)
{
    using L = MxSmem<BN, PAIR>;
    return launch_tiles<gemm_mx_kernel<BN, PAIR, GELU>, BN, PAIR, L::B_ROWS, kThreads, L::BYTES>(p, A, B, tc, s);
}

template <int BN, bool PAIR>
int launch_act(const E4Args &p, const struct k_rows *A, const struct k_rows *B, const CUtensorMap &tc, cudaStream_t s)
{
    return p.act == K_ACT_GELU ? launch<BN, PAIR, true>(p, A, B, tc, s) : launch<BN, PAIR, false>(p, A, B, tc, s);
}

}  // namespace

// Cycles of the waves of tiles, from measured times: 500 a k-block and 500 for tiles
// of 128 x 128, 840 and 1000 for pairs' tiles of 256 x 256 (41472 x 1024 x 4096: 162 and 133
// us; 5184 x 1024 x 1024: 10.4 and 12.3).
static long small_tiles(const E4Args &p)
{
    const long sms = device_sms(), kb = (p.K + BK - 1) / BK;
    return ((long)((p.M + 127) / 128) * ((p.N + 127) / 128) + sms - 1) / sms * (500 * kb + 500);
}
static long large_tiles(const E4Args &p)
{
    const long pairs = device_sms() > 1 ? device_sms() / 2 : 1, kb = (p.K + BK - 1) / BK;
    return ((long)((p.M + 255) / 256) * ((p.N + 255) / 256) + pairs - 1) / pairs * (840 * kb + 1000);
}

long cost_mx(const E4Args &p)
{
    const long a = small_tiles(p), b = large_tiles(p), kb = (p.K + BK - 1) / BK;
    // a wave of its own: 0.17 us a k-block (8 x 4096 x 1024 6.0 us, 256 x 4096 x 4096 11.5)
    if ((long)((p.M + 127) / 128) * ((p.N + 127) / 128) <= device_sms())
        return 460 + 17 * kb;
    return 400 + (a < b ? a : b) / 19;
}

int launch_mx(const E4Args &p, const struct k_rows *A, const struct k_rows *B, const CUtensorMap &tc, cudaStream_t s)
{
    if (large_tiles(p) < small_tiles(p)) {
        const int rc = launch_act<256, true>(p, A, B, tc, s);
        if (rc != K_EARG)
            return rc;
    }
    return launch_act<128, false>(p, A, B, tc, s);
}

}  // namespace sam3
