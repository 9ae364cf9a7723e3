// SPDX-License-Identifier: Unlicense
// Product of E4M3 matrices with block scales on tcgen05 (kind::f8f6f4): C = act(sum
// over 128-column blocks kb of SA[m, kb] SB[n / 128, kb] (A_kb B_kb^T) + bias).
//
// The scales are any numbers, so a block's product cannot simply be added to the
// last one's: each k-block of 128 (one shared-memory stage, four MMAs of K = 32)
// goes into a tensor-memory buffer of its own from zero, and the epilogue warps
// add it, times its scale, to sums in registers, one row and 128 columns a
// thread: one scale of B and one of A per thread and k-block. That also keeps long
// sums of 32-bit results out of the matrix unit, which truncates. Three
// warpgroups: a TMA producer, an MMA issuer and two warps that read scales in the
// first, two groups of four warps (a warp per lane quarter of tensor memory), which
// take over most of its registers.
//   BN 256: tiles of 128 x 256, each group 128 columns of them;
//   BN 128: tiles of 128 x 128, the groups take k-blocks in turn (twice as many are
//           under way, for problems of few tiles) and join their sums at the end.
// What bounds a tile is the way of a k-block through its buffer: about 900 cycles from
// the issue of its MMAs to the epilogue's first load, 250 for loads and sums, 250
// until the buffer is given back (41472 x 1024 x 4096: 187 us in a burst, 218 at the 1511 MHz that
// the power cap leaves; two buffers of 256 columns or four of 128 make no difference).
// A 128-column block of a row lies in one thread, so an E4M3 result is scaled and
// rounded there.
#include "gemm_e4m3.cuh"

#include <type_traits>

namespace sam3 {
namespace {

constexpr int BM = 128, BK = 128;
constexpr int kThreads = 384;
constexpr int kChunks = 4;                             // chunks of a group's scales in its ring
constexpr int kScaleRing = kChunks * kChunk * BM * 4;  // bytes

// Keeps the sums in front of the wait that follows.
__device__ __forceinline__ void hold32(float *a)
{
#pragma unroll
    for (int j = 0; j < 32; j += 8)
        asm volatile("" : "+f"(a[j]), "+f"(a[j + 1]), "+f"(a[j + 2]), "+f"(a[j + 3]), "+f"(a[j + 4]), "+f"(a[j + 5]),
                          "+f"(a[j + 6]), "+f"(a[j + 7]));
}

template <int BN>
struct E4Smem {
    static constexpr int A_BYTES = BM * BK;
    static constexpr int STAGE_BYTES = A_BYTES + BN * BK;
    static constexpr int STAGES = BN == 256 ? 3 : 4;
    static constexpr int EPI_OFF = STAGES * STAGE_BYTES;
    static constexpr int SCALE_OFF = EPI_OFF + (BN == 128 ? 4 : 8) * kStageTile;  // BN 128: one group stores
    static constexpr int JOIN_OFF = SCALE_OFF + 2 * kScaleRing;  // BN 128: the second group's sums
    static constexpr int BAR_OFF = JOIN_OFF + (BN == 128 ? BM * 128 * 4 : 0);
    // full[S], empty[S], tfull[4], tempty[4], sfull[2][4], sempty[2][4], drain, then
    // tmem base + abort
    static constexpr int BYTES = BAR_OFF + (2 * STAGES + 9 + 4 * kChunks) * 8 + 16 + 1024;
    static_assert(BYTES <= 232448, "shared memory");
};

// The products of both scales for the rows and the column block of one group's
// k-blocks (BN 128: every second one), four of them at a time, by a warp that runs
// ahead of the group: the loads of a chunk are in flight while the last one is
// handed over.
template <int BN>
__device__ __forceinline__ void feed_scales(const E4Args &p, float *ring, uint64_t *sfull, uint64_t *sempty, int group,
                                            int first, int step, int num_tiles, int num_n, int kblocks, int lane,
                                            volatile int *abort_flag)
{
    constexpr int R = BM / 32;  // rows of a lane
    constexpr int S = BN == 128 ? 2 : 1;
    struct Chunk {
        uint32_t a[R][kChunk], b[kChunk];
        int k;
    } v, w;
    const int k0 = BN == 128 ? group : 0, col = BN == 128 ? 0 : group * 128;
    int t = first, k = k0;
    auto fetch = [&](Chunk &o) {
        const int m = (t / num_n) * BM + lane, n = (t % num_n) * BN + col;
        const long rb = (long)(min(n, p.N - 1) / kScaleBlock) * p.ldsb;
        o.k = k;
        if constexpr (S == 1) {
            load_scales(p.sb, p.sbdt, p.sbvec, rb, k, kblocks, o.b);
#pragma unroll
            for (int i = 0; i < R; i++)
                load_scales(p.sa, p.sadt, p.savec, (long)min(m + 32 * i, p.M - 1) * p.ldsa, k, kblocks, o.a[i]);
        }
        else {
#pragma unroll
            for (int j = 0; j < kChunk; j++) {
                const bool in = k + S * j < kblocks;
                o.b[j] = in ? scale_raw(p.sb, p.sbdt, rb + k + S * j) : 0u;
#pragma unroll
                for (int i = 0; i < R; i++)
                    o.a[i][j] = in ? scale_raw(p.sa, p.sadt, (long)min(m + 32 * i, p.M - 1) * p.ldsa + k + S * j) : 0u;
            }
        }
    };
    uint32_t c = 0;  // chunks handed over
    auto put = [&](const Chunk &o, auto at, auto bt) {
        constexpr int AT = decltype(at)::value, BT = decltype(bt)::value;
        float *dst = ring + (c % kChunks) * (kChunk * BM) + lane;
        const bool va = S == 1 && p.savec, vb = S == 1 && p.sbvec;
#pragma unroll
        for (int j = 0; j < kChunk; j++) {
            const float sb = scale_at(o.b, BT, vb, o.k, kblocks, j);
#pragma unroll
            for (int i = 0; i < R; i++)
                dst[j * BM + 32 * i] = scale_at(o.a[i], AT, va, o.k, kblocks, j) * sb;
        }
    };
    auto give = [&](const Chunk &o) {
        const uint32_t slot = c % kChunks, parity = (c / kChunks & 1) ^ 1;
        if (!__all_sync(0xffffffffu, mbar_wait_brief(&sempty[slot], parity, p.err, abort_flag)))
            return false;
        using E = std::integral_constant<int, K_E8M0>;
        using F = std::integral_constant<int, K_F32>;
        if (p.sadt == K_E8M0)
            p.sbdt == K_E8M0 ? put(o, E{}, E{}) : put(o, E{}, F{});
        else
            p.sbdt == K_E8M0 ? put(o, F{}, E{}) : put(o, F{}, F{});
        __syncwarp();
        if (lane == 0)
            mbar_arrive(&sfull[slot]);
        c++;
        return true;
    };
    auto advance = [&]() {
        k += S * kChunk;
        if (k >= kblocks) {
            k = k0;
            t += step;
        }
        return t < num_tiles;
    };
    bool more = t < num_tiles && k0 < kblocks;
    if (more)
        fetch(v);
    while (more) {
        more = advance();
        if (more)
            fetch(w);
        if (!give(v) || !more)
            return;
        more = advance();
        if (more)
            fetch(v);
        if (!give(w))
            return;
    }
}

template <int BN, bool GELU>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_e4m3_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                     const __grid_constant__ CUtensorMap tmC, const __grid_constant__ E4Args p)
{
    constexpr bool TURNS = BN == 128;          // the groups take k-blocks in turn
    constexpr int KS = TURNS ? 2 : 1;
    using L = E4Smem<BN>;
    constexpr int STAGES = L::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem =
        reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::BAR_OFF);
    uint64_t *empty = full + STAGES;
    uint64_t *tfull = empty + STAGES;                   // [group][buffer] (TURNS), [buffer]
    uint64_t *tempty = tfull + 4;
    uint64_t *sfull = tempty + 4, *sempty = sfull + 2 * kChunks;  // [group][chunk]
    uint64_t *drain = sempty + 2 * kChunks;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; i++) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 4; i++) {
            mbar_init(&tfull[i], 1);
            mbar_init(&tempty[i], TURNS ? 4 : 8);
        }
        for (int i = 0; i < 2 * kChunks; i++) {
            mbar_init(&sfull[i], 1);
            mbar_init(&sempty[i], 4);
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    griddep_launch();
    griddep_wait();

    const int first = (int)blockIdx.x, step = (int)gridDim.x;
    const int num_n = (p.N + BN - 1) / BN;
    const int num_tiles = (p.M + BM - 1) / BM * num_n;
    const int kblocks = (p.K + BK - 1) / BK;

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
                    const int m0 = (t / num_n) * BM, n0 = (t % num_n) * BN;
                    for (int kb = 0; kb < kblocks; kb++) {
                        if (!mbar_wait_brief(&empty[stage], phase ^ 1, p.err, abort_flag)) {
                            ok = false;
                            break;
                        }
                        uint8_t *sa = smem + stage * L::STAGE_BYTES;
                        mbar_arrive_expect_tx(&full[stage], L::STAGE_BYTES);
                        tma_load_2d(sa, &tmA, &full[stage], kb * BK, m0);
                        tma_load_2d(sa + L::A_BYTES, &tmB, &full[stage], kb * BK, n0);
                        issued_mask |= 1u << stage;
                        last_parity = (last_parity & ~(1u << stage)) | (phase << stage);
                        if (++stage == STAGES) {
                            stage = 0;
                            phase ^= 1;
                        }
                    }
                }
                // Every copy this thread issued lands before the CTA exits.
                for (int s = 0; s < STAGES; s++)
                    if (issued_mask & (1u << s)) {
                        volatile int no_abort = 0;
                        mbar_wait(&full[s], (last_parity >> s) & 1, p.err, &no_abort);
                    }
            }
        }
        else if (warp == 1) {
            if (elect_one()) {
                constexpr uint32_t idesc = idesc_e4m3_f32(BM, BN);
                const uint32_t smem0 = smem_addr(smem);
                int stage = 0;
                uint32_t phase = 0, c0 = 0, c1 = 0;  // k-blocks handed to each group
                bool ok = true, loaded = false, free = false;
                // The barriers of the next k-block are asked while this one's MMAs run (an
                // answer takes about 150 cycles). Its commit tells the epilogue, which
                // gives the stage back: a second commit would take 300.
                for (int t = first; t < num_tiles && ok; t += step)
                    for (int kb = 0; kb < kblocks; kb++) {
                        const int g = TURNS ? kb & 1 : 0;
                        const uint32_t c = g ? c1++ : c0++, b = 2 * g + (c & 1), parity = (c >> 1 & 1) ^ 1;
                        ok = (loaded || mbar_wait_brief(&full[stage], phase, p.err, abort_flag)) &&
                             (free || mbar_wait_brief(&tempty[b], parity, p.err, abort_flag));
                        if (!ok)
                            break;
                        tc_fence_after();
                        const uint32_t sa = smem0 + stage * L::STAGE_BYTES;
                        const uint64_t da = sw128_desc(sa, 16, 1024), db = sw128_desc(sa + L::A_BYTES, 16, 1024);
                        const uint32_t d = tmem_base + b * BN;
#pragma unroll
                        for (int k = 0; k < BK / 32; k++)  // 32 columns further: 2 units of 16 bytes
                            tc_mma_e4m3(d, da + 2 * k, db + 2 * k, idesc, k != 0);
                        tc_commit(&tfull[b]);
                        if (++stage == STAGES) {
                            stage = 0;
                            phase ^= 1;
                        }
                        const int g1 = TURNS && kb + 1 < kblocks ? (kb + 1) & 1 : 0;
                        const uint32_t cn = g1 ? c1 : c0;
                        loaded = mbar_test_wait(smem_addr(&full[stage]), phase);
                        free = mbar_test_wait(smem_addr(&tempty[2 * g1 + (cn & 1)]), (cn >> 1 & 1) ^ 1);
                    }
                tc_commit(drain);  // one arrival once every MMA is done
                // Tensor memory is idle before it is freed.
                volatile int no_abort = 0;
                mbar_wait(drain, 0, p.err, &no_abort);
            }
        }
        else {
            const int g = warp - 2;
            feed_scales<BN>(p, reinterpret_cast<float *>(smem + L::SCALE_OFF + g * kScaleRing), sfull + kChunks * g,
                            sempty + kChunks * g, g, first, step, num_tiles, num_n, kblocks, lane, abort_flag);
        }
    }
    else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int group = (warp - 4) >> 2;
        const int quarter = warp & 3;  // the TMEM lanes this warp may read
        const int row = quarter * 32, col = TURNS ? 0 : group * 128;
        const uint32_t stage_tile = smem_addr(smem + L::EPI_OFF + (TURNS ? quarter : warp - 4) * kStageTile);
        const float *ring = reinterpret_cast<const float *>(smem + L::SCALE_OFF + group * kScaleRing) + row + lane;
        if (lane == 0)
            prefetch_tmap(&tmC);
        // A barrier's parity tells neighbouring phases apart only: a group waits for
        // every phase of its buffers.
        uint32_t c = 0, chunk = 0, before = 0;  // before: k-blocks of the tiles before
        bool ok = true, ready = false;
        for (int t = first; t < num_tiles && ok; t += step, before += kblocks) {
            float acc[128];
#pragma unroll
            for (int j = 0; j < 128; j++)
                acc[j] = 0.0f;
            for (int kb = TURNS ? group : 0, i = 0; kb < kblocks; kb += KS, i++, c++) {
                const uint32_t buf = (TURNS ? 2 * group : 0) + (c & 1), slot = kChunks * group + chunk % kChunks;
                if (!__all_sync(0xffffffffu, ready)) {
                    ok = mbar_wait_brief(&sfull[slot], chunk / kChunks & 1, p.err, abort_flag) &&
                         mbar_wait_brief(&tfull[buf], c >> 1 & 1, p.err, abort_flag);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok)
                        break;
                }
                tc_fence_after();
                if (quarter == 0 && (TURNS || group == 0) && lane == 0)
                    mbar_arrive(&empty[(before + kb) % STAGES]);  // the MMAs have read the stage
                const uint32_t src = tmem_base + ((uint32_t)row << 16) + buf * BN + col;
                const float s = ring[(chunk % kChunks * kChunk + i % kChunk) * BM];
                const bool last = i % kChunk == kChunk - 1 || kb + KS >= kblocks;
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
                    hold32(&acc[32 * q]);
                    if (q < 3)
                        tmem_wait_ld(r[(q + 1) & 1]);
                    if (q == 2) {  // the buffer has been read
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) {
                            mbar_arrive_relaxed(&tempty[buf]);
                            if (last)  // the chunk's scales are in registers
                                mbar_arrive(&sempty[slot]);
                        }
                        // the next block's barriers, asked beside the last sums
                        const uint32_t cn = c + 1, chn = chunk + last;
                        ready = mbar_test_wait(smem_addr(&tfull[(TURNS ? 2 * group : 0) + (cn & 1)]), cn >> 1 & 1);
                        if (last)
                            ready = mbar_test_wait(smem_addr(&sfull[kChunks * group + chn % kChunks]), chn / kChunks & 1) && ready;
                    }
                }
                chunk += last;
            }
            if constexpr (TURNS) {
                // The second group's sums through shared memory to the first: 16 bytes of
                // a thread, threads side by side.
                float4 *join = reinterpret_cast<float4 *>(smem + L::JOIN_OFF) + row + lane;
                if (group == 1) {
#pragma unroll
                    for (int j = 0; j < 32; j++)
                        join[j * BM] = make_float4(acc[4 * j], acc[4 * j + 1], acc[4 * j + 2], acc[4 * j + 3]);
                }
                // the two warps of the rows, which go on or give up together
                uint32_t both;
                asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
                             "bar.red.and.pred p, %2, 64, q;\n\tselp.b32 %0, 1, 0, p;\n\t}"
                             : "=r"(both)
                             : "r"((uint32_t)ok), "r"(1 + quarter)
                             : "memory");
                ok = both != 0;
                if (group == 0) {
#pragma unroll
                    for (int j = 0; j < 32; j++) {
                        const float4 v = join[j * BM];
                        acc[4 * j] += v.x;
                        acc[4 * j + 1] += v.y;
                        acc[4 * j + 2] += v.z;
                        acc[4 * j + 3] += v.w;
                    }
                }
                asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");  // read before the next tile's are written
            }
            if (!ok)
                break;
            const int m0 = (t / num_n) * BM + row, n = (t % num_n) * BN + col;
            if (m0 < p.M && n < p.N && (!TURNS || group == 0))
                finish<GELU>(p, &tmC, stage_tile, lane, m0, n, acc);
        }
        if (p.tma && lane == 0)
            bulk_wait_all();
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
}

template <int BN, bool GELU>
int launch(const E4Args &p, const struct k_rows *A, const struct k_rows *B, const CUtensorMap &tc, cudaStream_t s)
{
    return launch_tiles<gemm_e4m3_kernel<BN, GELU>, BN, false, BN, kThreads, E4Smem<BN>::BYTES>(p, A, B, tc, s);
}

template <int BN>
int launch_act(const E4Args &p, const struct k_rows *A, const struct k_rows *B, const CUtensorMap &tc, cudaStream_t s)
{
    return p.act == K_ACT_GELU ? launch<BN, true>(p, A, B, tc, s) : launch<BN, false>(p, A, B, tc, s);
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
    cudaStream_t st = reinterpret_cast<cudaStream_t>(s);
    // Of the forms that take the call, the one whose time, from measured ones, is the
    // smallest (in 1/100 us). Tiles of the form below: 0.40 us a k-block and 2 a wave for 128
    // columns, 0.55 and 2.5 for 256 (256 x 4096 x 4096: 17.8 and 22.6 us, 41472 x 1024 x 4096:
    // 245 and 182); 32 rows of the form for few: 0.62 us for 2^20 weights (32 x 4096 x 4096: 13.1
    // us, 10.4 by gemm_e4m3_mx.cu; 32 x 4096 x 1024: 4.8 and 6.1).
    const long sms = device_sms(), kb = (K + BK - 1) / BK;
    const long t1 = (long)((M + 127) / 128) * ((N + 127) / 128), t2 = (long)((M + 127) / 128) * ((N + 255) / 256);
    const long c1 = (t1 + sms - 1) / sms * (40 * kb + 200), c2 = (t2 + sms - 1) / sms * (55 * kb + 250);
    // Scales the matrix unit can apply, results that do not show its truncation: errors
    // against 64 bits 7e-8 of 32-bit results over 1024 columns (4e-8 by the form below), 2.8e-7
    // over 4096 (7e-8).
    const bool mx = p.sadt == K_E8M0 && p.sbdt == K_E8M0 && (p.cdt != K_F32 || kb <= 8);
    const long tiles = mx ? cost_mx(p) : 270 + (c1 < c2 ? c1 : c2);
    if (C->dt != K_E4M3 && M <= 256 && 250 + (long)((M + 31) / 32) * N * K / 16900 < tiles)
        return launch_few(p, A, B, st);
    CUtensorMap tc;
    const int es = C->dt == K_F32 ? 4 : (C->dt == K_E4M3 ? 1 : 2);
    const CUtensorMapDataType dt = C->dt == K_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : C->dt == K_E4M3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                                     : CU_TENSOR_MAP_DATA_TYPE_UINT16;
    const uint64_t pitch = M > 1 ? (uint64_t)C->ld : ((uint64_t)N + 15) / 16 * 16;
    p.ntma = N - N % (16 / es);
    p.tma = p.ntma > 0 && make_tmap_2d(&tc, dt, es, C->p, (uint64_t)M, (uint64_t)p.ntma, pitch, 128 / es, 32);
    if (!p.tma && !make_tmap_2d(&tc, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, A->p, (uint64_t)M, (uint64_t)K,
                                M > 1 ? (uint64_t)A->ld : ((uint64_t)K + 15) / 16 * 16, 128, 32))
        return K_ETMAP;  // (a map for the argument that is not used)
    if (mx)
        return launch_mx(p, A, B, tc, st);
    return c2 < c1 ? launch_act<256>(p, A, B, tc, st) : launch_act<128>(p, A, B, tc, st);
}
