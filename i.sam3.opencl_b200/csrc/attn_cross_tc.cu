// SPDX-License-Identifier: Unlicense
// Cross attention (see attn_cross.cu) of many query rows over many keys on
// tcgen05 tensor cores, bf16 and f16. The pipeline is that of attn_tc.cu:
// work items (sequence, head, 128 query rows), two persistent CTAs per SM, one
// thread per query row in warps 0-3, TMA producers in warp 4 (lane 0: Q and K,
// lane 1: V), MMA issuer in warp 5; scores of two key tiles in tensor memory,
// P written over the scores it came from, P.V reading it from there. Here
//   - operands come through 4-D maps (column, row, head, sequence), so any
//     order and stride of the operand works and columns past hd read as zero:
//     heads of up to 64 columns run as 64, up to 128 as two 64-column panels
//     (64 keys a tile instead of 96, one Q buffer and two stages a ring, which
//     keeps two CTAs per SM);
//   - a sequence's key count bounds its tiles; in a tile with keys that are
//     masked or past the count their scores become -inf, and the softmax warps
//     zero their V rows in shared memory before they hand P over (0 * NaN would
//     reach the sum); the mask bytes of a tile are read one tile ahead;
//   - when the items leave CTA slots free, a cluster of 2 to 8 CTAs shares an
//     item's key tiles and merges (max, sum, output) through distributed
//     shared memory: no workspace, one launch.
// Softmax as in attn_tc.cu: the row's offset is the maximum of its first tile
// with a visible key, exponentials of later tiles are taken against it, and a
// tile whose sum reaches kOverflowSum (or is not a number; the polynomial
// exponential makes 2^125 of one) is taken again with a raised offset, without
// the polynomial, so that infinities and NaN of visible keys come out as such.
// Measured: 8 x 5184 queries x 5184 keys x 16 heads of 64 columns 1028 us, 857
// TFLOP/s (the softmax warps bound it as in attn_tc.cu: 879), with a key mask, every
// tile in the rolled path, 1173 us; 4 x 4096 x 4096 x 16 heads of 128 columns 483
// us, 1138 TFLOP/s (tensor pipe 60 %); 32 x 1 query over 2048 keys of 8 heads of 128
// columns 45 us, 5.9 TB/s.
#include "attn_cross.cuh"
#include "cluster.cuh"
#include "kernels.h"
#include "pdl.cuh"
#include "tc_ptx.cuh"
#include "tmap.cuh"

namespace sam3 {
namespace {

constexpr int BQ = 128;
constexpr int kProducerWarp = 4;
constexpr int kMmaWarp = 5;
constexpr int kThreads = 32 * 6;
constexpr int kCtasPerSm = 2;
constexpr int kMaxSplit = 8;
constexpr int kPolyPairsPer8 = 2;  // of 8 pairs, on the FMA pipe (attn_tc.cu)
// Weights times 2^kShift (as kWeightShift, attn_cross.cuh), and the sum of a tile's
// from which it is taken again. f16: 96 weights of the first tile, 2^9 at most,
// stay below the limit and each weight below it fits the type: whole down to
// 2^-23 of the offset's weight and rounded by 2^-34 below. bf16: weights stay
// below 1, so that their sums with values are finite as far as the plain ones
// are, and 2^-13 of the smallest normal value still has the type's bits.
template <typename T>
constexpr float kShift = __is_same(T, __half) ? 9.0f : -13.0f;
template <typename T>
constexpr float kOverflowSum = __is_same(T, __half) ? 61440.0f : 1.0f;
// An offset is a score; its product with the scale is rounded, which leaves a
// power of two of that rounding in every weight of the row. Products below this
// leave 2^-12 at most, less than the weights' own rounding; beyond it a tile
// goes through again, where differences are taken before they are scaled.
constexpr float kFarOffset = 4096.0f;

template <int HDP>
struct Geo {
    static constexpr int BKV = HDP == 64 ? 96 : 64;
    static constexpr int KST = HDP == 64 ? 3 : 2;
    static constexpr int NQ = HDP == 64 ? 2 : 1;  // Q buffers
    static constexpr int NP = HDP / 64;           // 64-column panels
    static constexpr int Q_BYTES = BQ * HDP * 2;
    static constexpr int KV_BYTES = BKV * HDP * 2;
    static constexpr int OFF_Q = 0;
    static constexpr int OFF_K = OFF_Q + NQ * Q_BYTES;
    static constexpr int OFF_V = OFF_K + KST * KV_BYTES;
    static constexpr int OFF_BAR = OFF_V + KST * KV_BYTES;
    static constexpr int NBAR = 2 * NQ + 4 * KST + 2 + 2 + 2 + 1;
    static constexpr int SMEM = OFF_BAR + NBAR * 8 + 16 + 1024;
    static constexpr uint32_t TM_O = 2 * BKV, TM_COLS = 256;
    static_assert(kCtasPerSm * SMEM <= 232448 - 2048, "two CTAs per SM");
    static_assert(TM_O + HDP <= TM_COLS, "tensor memory");
    static_assert(BQ * Parts<HDP>::PR * 4 <= OFF_BAR, "partial rows");
};

template <typename T>
__host__ __device__ constexpr uint32_t idesc(int M, int N, int b_mn_major)
{
    // kind::f16 with fp32 accumulation; A and B of one type
    const uint32_t f = sizeof(T) == 2 && !__is_same(T, __half) ? 1u : 0u;
    return (1u << 4) | (f << 7) | (f << 10) | ((uint32_t)b_mn_major << 16) |
           ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

struct TcArgs {
    XaArgs x;
    int nitems;
    int qb0, qb1, kb0, kb1, vb0, vb1;  // 1: the map has that dimension (stride not 0)
};

template <typename T, int HDP, bool SPLIT, bool MASK>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
    attn_cross_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                         const __grid_constant__ CUtensorMap tmV, const __grid_constant__ TcArgs ta)
{
    using G = Geo<HDP>;
    constexpr int BKV = G::BKV, KST = G::KST, NQ = G::NQ, NP = G::NP, NW = BKV / 32;
    const XaArgs &a = ta.x;
    extern __shared__ uint8_t smem_raw[];
    // Same offset in every CTA of a cluster: dynamic shared memory starts at
    // the same address in all of them.
    uint8_t *smem = reinterpret_cast<uint8_t *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + G::OFF_BAR);
    uint64_t *q_full = bars, *q_empty = q_full + NQ;
    uint64_t *k_full = q_empty + NQ, *k_empty = k_full + KST;
    uint64_t *v_full = k_empty + KST, *v_empty = v_full + KST;
    uint64_t *s_full = v_empty + KST, *p_ready = s_full + 2, *pv_full = p_ready + 2;
    uint64_t *drain = pv_full + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + G::NBAR);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = SPLIT ? (int)(blockIdx.x % a.cs) : 0;
    const int first = SPLIT ? (int)(blockIdx.x / a.cs) : (int)blockIdx.x;
    const int stride = SPLIT ? ta.nitems : (int)gridDim.x;

    if (threadIdx.x == 0) {
        for (int i = 0; i < NQ; i++) {
            mbar_init(&q_full[i], 1);
            mbar_init(&q_empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_ready[i], 4);
            mbar_init(&pv_full[i], 1);
        }
        for (int i = 0; i < KST; i++) {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_full[i], 1);
            mbar_init(&v_empty[i], 1);
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == kMmaWarp) {
        tmem_alloc(tmem_slot, G::TM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    griddep_launch();
    griddep_wait();

    // item = (sequence * heads + head) * nqt + query tile; its key tiles
    // [j0, j0 + n) of this CTA
    struct Item {
        int seq, head, qt, len, j0, n;
    };
    auto item_at = [&](int u) {
        Item it;
        it.qt = u % a.nqt;
        const int sh = u / a.nqt;
        it.head = sh % a.heads;
        it.seq = sh / a.heads;
        it.len = a.klen ? min(max(__ldg(a.klen + it.seq), 0), a.Nk) : a.Nk;
        const int nt = (it.len + BKV - 1) / BKV;
        it.j0 = SPLIT ? (int)((long)nt * rank / a.cs) : 0;
        it.n = (SPLIT ? (int)((long)nt * (rank + 1) / a.cs) : nt) - it.j0;
        return it;
    };

    // what a split item's rows leave for the merge
    float part_max = -INFINITY, part_sum = 0.0f;
    int part_tiles = 0;

    if (warp == kProducerWarp) {
        if (lane < 2) {
            const bool is_k = lane == 0;
            const CUtensorMap *tmX = is_k ? &tmK : &tmV;
            if (is_k)
                prefetch_tmap(&tmQ);
            prefetch_tmap(tmX);
            uint64_t *full = is_k ? k_full : v_full;
            uint64_t *empty = is_k ? k_empty : v_empty;
            uint8_t *ring = smem + (is_k ? G::OFF_K : G::OFF_V);
            int qn = 0, g = 0, st = 0, use = 0;
            bool ok = true;
            for (int u = first; u < ta.nitems && ok; u += stride) {
                const Item it = item_at(u);
                if (it.n == 0)
                    continue;
                if (is_k) {
                    const int qb = qn % NQ;
                    if (!mbar_wait(&q_empty[qb], ((qn / NQ) & 1) ^ 1, a.err, abort_flag))
                        break;
                    mbar_arrive_expect_tx(&q_full[qb], G::Q_BYTES);
                    for (int p = 0; p < NP; p++)
                        tma_load_4d(smem + G::OFF_Q + qb * G::Q_BYTES + p * BQ * 128, &tmQ, &q_full[qb],
                                    p * 64, it.qt * BQ, it.head * ta.qb1, it.seq * ta.qb0);
                    qn++;
                }
                const int kh = it.head / a.g;
                const int ch = kh * (is_k ? ta.kb1 : ta.vb1), cb = it.seq * (is_k ? ta.kb0 : ta.vb0);
                for (int j = 0; j < it.n; j++) {
                    if (!mbar_wait(&empty[st], (use & 1) ^ 1, a.err, abort_flag)) {
                        ok = false;
                        break;
                    }
                    mbar_arrive_expect_tx(&full[st], G::KV_BYTES);
                    for (int p = 0; p < NP; p++)
                        tma_load_4d(ring + st * G::KV_BYTES + p * BKV * 128, tmX, &full[st], p * 64,
                                    (it.j0 + j) * BKV, ch, cb);
                    g++;
                    if (++st == KST) {
                        st = 0;
                        use++;
                    }
                }
            }
            // no copy may be in flight when the CTA ends
            volatile int no_abort = 0;
            for (int k = qn - NQ; is_k && k < qn; k++)
                if (k >= 0)
                    mbar_wait(&q_full[k % NQ], (k / NQ) & 1, a.err, &no_abort);
            for (int k = g - KST; k < g; k++)
                if (k >= 0)
                    mbar_wait(&full[k % KST], (k / KST) & 1, a.err, &no_abort);
        }
    }
    else if (warp == kMmaWarp) {
        if (elect_one()) {
            constexpr uint32_t idS = idesc<T>(BQ, BKV, 0);
            constexpr uint32_t idPV = idesc<T>(BQ, HDP, 1);
            const uint64_t dQ = sw128_desc(smem_addr(smem + G::OFF_Q), 16, 1024);
            const uint64_t dK = sw128_desc(smem_addr(smem + G::OFF_K), 16, 1024);
            const uint64_t dV = sw128_desc(smem_addr(smem + G::OFF_V), BKV * 128, 1024);
            struct Cur {
                int u, n, j, g, qn, st, ph;
            };
            auto settle = [&](Cur &c) {  // to the next item with tiles
                while (c.u < ta.nitems) {
                    c.n = item_at(c.u).n;
                    if (c.n > 0)
                        return;
                    c.u += stride;
                }
            };
            auto adv = [&](Cur &c) {
                c.g++;
                if (++c.st == KST) {
                    c.st = 0;
                    c.ph ^= 1;
                }
                if (++c.j == c.n) {
                    c.j = 0;
                    c.qn++;
                    c.u += stride;
                    settle(c);
                }
            };
            auto issue_s = [&](const Cur &c) -> bool {
                const int st = c.st, qb = c.qn & (NQ - 1);
                if (!mbar_wait(&k_full[st], c.ph, a.err, abort_flag))
                    return false;
                if (c.j == 0 && !mbar_wait(&q_full[qb], (c.qn / NQ) & 1, a.err, abort_flag))
                    return false;
                tc_fence_after();
                const uint32_t dS = tmem_base + (c.g & 1) * BKV;
                const uint64_t qd = dQ + (uint64_t)((qb * G::Q_BYTES) >> 4);
                const uint64_t kd = dK + (uint64_t)((st * G::KV_BYTES) >> 4);
#pragma unroll
                for (int kq = 0; kq < HDP / 16; kq++)
                    tc_mma(dS, qd + (((kq / 4) * BQ * 128 + (kq % 4) * 32) >> 4),
                           kd + (((kq / 4) * BKV * 128 + (kq % 4) * 32) >> 4), idS, kq != 0);
                tc_commit(&s_full[c.g & 1]);
                tc_commit(&k_empty[st]);
                if (c.j == c.n - 1)
                    tc_commit(&q_empty[qb]);
                return true;
            };
            auto issue_pv = [&](const Cur &c) -> bool {
                const int st = c.st;
                if (!mbar_wait(&v_full[st], c.ph, a.err, abort_flag))
                    return false;
                if (!mbar_wait(&p_ready[c.g & 1], (c.g >> 1) & 1, a.err, abort_flag))
                    return false;
                tc_fence_after();
                const uint32_t aP = tmem_base + (c.g & 1) * BKV;
                const uint64_t vd = dV + (uint64_t)((st * G::KV_BYTES) >> 4);
#pragma unroll
                for (int kk = 0; kk < BKV / 16; kk++)
                    tc_mma_ts(tmem_base + G::TM_O, aP + kk * 8, vd + 128 * kk, idPV, (c.j | kk) != 0);
                tc_commit(&pv_full[c.g & 1]);
                tc_commit(&v_empty[st]);
                return true;
            };
            Cur ahead = {first, 0, 0, 0, 0, 0, 0};
            settle(ahead);
            Cur cur = ahead;
            bool ok = true;
            for (int i = 0; ok && i < 2 && ahead.u < ta.nitems; i++) {
                ok = issue_s(ahead);
                adv(ahead);
            }
            while (ok && cur.u < ta.nitems) {
                ok = issue_pv(cur);
                if (ok && ahead.u < ta.nitems) {
                    ok = issue_s(ahead);
                    adv(ahead);
                }
                adv(cur);
            }
            tc_commit(drain);
            volatile int no_abort = 0;
            mbar_wait(drain, 0, a.err, &no_abort);
        }
    }
    else {  // softmax warps 0-3, warp = TMEM lane quarter
        const int quarter = warp;
        const int r = quarter * 32 + lane;
        const uint32_t tL = tmem_base + ((uint32_t)(quarter * 32) << 16);
        const uint32_t tO = tL + G::TM_O;
        const uint64_t sl2x2 = f2_make(a.scale_log2, a.scale_log2);
        bool ok = true;
        int g = 0;
        for (int u = first; u < ta.nitems && ok; u += stride) {
            const Item it = item_at(u);
            const bool rows_live = it.qt * BQ + quarter * 32 < a.Nq;
            const int q = it.qt * BQ + r;
            const uint8_t *mask = MASK ? a.kmask + (long)it.seq * a.Nk : nullptr;
            float m_used = -INFINITY;  // offset, a score before scaling
            uint64_t lsum0 = 0, lsum1 = 0;
            uint8_t ahead[NW];  // mask bytes of the next tile, a key per lane
            auto look = [&](int j) {
#pragma unroll
                for (int w = 0; w < NW; w++) {
                    const int key = (it.j0 + j) * BKV + w * 32 + lane;
                    ahead[w] = MASK && j < it.n && key < it.len ? __ldg(mask + key) : 0;
                }
            };
            look(0);
            for (int j = 0; j < it.n; j++, g++) {
                const int b = g & 1;
                // visible keys of the tile; without a mask only the last tile
                // can hold hidden ones
                uint32_t vis[NW];
                bool whole = MASK || j < it.n - 1 || (it.j0 + it.n) * BKV <= it.len;
                if (MASK || !whole) {
#pragma unroll
                    for (int w = 0; w < NW; w++) {
                        const int left = it.len - (it.j0 + j) * BKV - w * 32;
                        vis[w] = left >= 32 ? 0xffffffffu : (left > 0 ? (1u << left) - 1 : 0u);
                        if (MASK) {
                            vis[w] &= __ballot_sync(0xffffffffu, ahead[w] == 0);
                            whole = whole && vis[w] == 0xffffffffu;
                        }
                    }
                    if (MASK)
                        look(j + 1);
                }
                ok = __all_sync(0xffffffffu, mbar_wait(&s_full[b], (g >> 1) & 1, a.err, abort_flag));
                if (!ok)
                    break;
                tc_fence_after();
                // The hidden keys' rows of V, a thread per key. Only after the
                // scores: S(g) follows P.V(g - 2), so the load of this stage
                // before this one is complete and the wait below cannot take it
                // for this one's (two stages a ring; a parity names every other
                // load of a stage).
                if (!whole) {
                    const int st = g % KST;
                    ok = __all_sync(0xffffffffu, mbar_wait(&v_full[st], (g / KST) & 1, a.err, abort_flag));
                    if (!ok)
                        break;
                    const int key = r;
                    uint32_t word = 0xffffffffu;
#pragma unroll
                    for (int w = 0; w < NW; w++)
                        if (key / 32 == w)
                            word = vis[w];
                    if (key < BKV && !((word >> (key & 31)) & 1)) {
                        uint8_t *row = smem + G::OFF_V + st * G::KV_BYTES + key * 128;
#pragma unroll
                        for (int p = 0; p < NP; p++)
#pragma unroll
                            for (int c = 0; c < 8; c++)
                                *reinterpret_cast<uint4 *>(row + p * BKV * 128 + c * 16) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async_smem();
                }
                const uint32_t tS = tL + b * BKV;
                bool resc = false;
                float factor = 1.0f;
                if (rows_live) {
                    uint64_t t0 = 0, t1 = 0;
                    bool over = true;
                    if (whole) {
                        uint32_t s[BKV];
#pragma unroll
                        for (int c = 0; c < NW; c++)
                            tmem_ld32(tS + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(s + 32 * c));
                        tmem_wait_ld();
                        if (m_used == -INFINITY) {
                            float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
                            for (int e = 0; e < BKV; e += 4) {
                                mx0 = max3f(mx0, __uint_as_float(s[e]), __uint_as_float(s[e + 1]));
                                mx1 = max3f(mx1, __uint_as_float(s[e + 2]), __uint_as_float(s[e + 3]));
                            }
                            m_used = fmaxf(mx0, mx1);
                        }
                        const float top = m_used == -INFINITY ? 0.0f : m_used * a.scale_log2;
                        const uint64_t negm = f2_make(kShift<T> - top, kShift<T> - top);
#pragma unroll
                        for (int e = 0; e < BKV; e += 2) {
                            const uint64_t x2 = fma2(f2_make(__uint_as_float(s[e]), __uint_as_float(s[e + 1])),
                                                     sl2x2, negm);
                            float x0, x1, p0, p1;
                            f2_split(x2, x0, x1);
                            if (((e >> 1) & 7) >= 8 - kPolyPairsPer8)
                                exp2_poly2(x0, x1, p0, p1);
                            else {
                                p0 = ex2_approx(x0);
                                p1 = ex2_approx(x1);
                            }
                            if ((e >> 1) & 1)
                                t1 = add2(t1, f2_make(p0, p1));
                            else
                                t0 = add2(t0, f2_make(p0, p1));
                            s[e >> 1] = pack2<T>(p0, p1);
                        }
                        float u0, u1, u2, u3;
                        f2_split(t0, u0, u1);
                        f2_split(t1, u2, u3);
                        over = __any_sync(0xffffffffu,
                                          !(((u0 + u1) + (u2 + u3)) < kOverflowSum<T> &&
                                            fabsf(top) < kFarOffset));
                        if (!over) {
                            tmem_st32(tS, *reinterpret_cast<const uint32_t(*)[32]>(s));
                            if constexpr (BKV == 96)
                                tmem_st16(tS + 32, *reinterpret_cast<const uint32_t(*)[16]>(s + 32));
                        }
                    }
                    if (over) {
                        // A tile with hidden keys, or one to take again: 32 columns
                        // at a time in rolled loops (the unrolled code above has to
                        // stay in the instruction cache), its maximum, then the
                        // exponentials, P of a chunk written below the scores not
                        // yet read.
                        auto chunk = [&](int c, uint32_t (&s)[32]) {
                            tmem_ld32(tS + 32 * c, s);
                            tmem_wait_ld();
                            uint32_t seen = 0xffffffffu;
                            if (!whole) {
#pragma unroll
                                for (int w = 0; w < NW; w++)
                                    seen = c == w ? vis[w] : seen;
                            }
#pragma unroll
                            for (int e = 0; e < 32; e++)
                                if (!((seen >> e) & 1))
                                    s[e] = __float_as_uint(-INFINITY);
                        };
                        float mx = -INFINITY;
#pragma unroll 1
                        for (int c = 0; c < NW; c++) {
                            uint32_t s[32];
                            chunk(c, s);
#pragma unroll
                            for (int e = 0; e < 32; e += 2)
                                mx = max3f(mx, __uint_as_float(s[e]), __uint_as_float(s[e + 1]));
                        }
                        if (m_used == -INFINITY)
                            m_used = mx;
                        else if (mx > m_used) {
                            resc = true;
                            factor = ex2_approx((m_used - mx) * a.scale_log2);
                            m_used = mx;
                            lsum0 = mul2(lsum0, f2_make(factor, factor));
                            lsum1 = mul2(lsum1, f2_make(factor, factor));
                        }
                        const float base = m_used == -INFINITY ? 0.0f : -m_used;
                        const uint64_t base2 = f2_make(base, base), shift2 = f2_make(kShift<T>, kShift<T>);
                        t0 = t1 = 0;
#pragma unroll 1
                        for (int c = 0; c < NW; c++) {
                            uint32_t s[32], p[16];
                            chunk(c, s);
#pragma unroll
                            for (int e = 0; e < 32; e += 2) {
                                float x0, x1;
                                f2_split(fma2(add2(f2_make(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), base2),
                                              sl2x2, shift2),
                                         x0, x1);
                                const float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
                                t0 = add2(t0, f2_make(p0, p1));
                                p[e >> 1] = pack2<T>(p0, p1);
                            }
                            tmem_st16(tS + 16 * c, p);
                        }
                    }
                    lsum0 = add2(lsum0, t0);
                    lsum1 = add2(lsum1, t1);
                }
                if (__any_sync(0xffffffffu, resc)) {
                    const int gp = g - 1;
                    ok = __all_sync(0xffffffffu, mbar_wait(&pv_full[gp & 1], (gp >> 1) & 1, a.err,
                                                           abort_flag));
                    if (!ok)
                        break;
                    tc_fence_after();
                    const uint64_t f2v = f2_make(factor, factor);
#pragma unroll 1
                    for (int c = 0; c < HDP / 32; c++) {
                        uint32_t o[32];
                        tmem_ld32(tO + c * 32, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            float o0, o1;
                            f2_split(mul2(f2_make(__uint_as_float(o[e]), __uint_as_float(o[e + 1])), f2v),
                                     o0, o1);
                            o[e] = __float_as_uint(o0);
                            o[e + 1] = __float_as_uint(o1);
                        }
                        tmem_st32(tO + c * 32, o);
                    }
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0)
                    mbar_arrive(&p_ready[b]);
            }
            if (!ok)
                break;
            if (it.n > 0) {
                const int gl = g - 1;
                ok = __all_sync(0xffffffffu, mbar_wait(&pv_full[gl & 1], (gl >> 1) & 1, a.err, abort_flag));
                if (!ok)
                    break;
                tc_fence_after();
            }
            if (SPLIT) {  // pushed behind the cluster barrier below
                float la, lb, lc, ld;
                f2_split(lsum0, la, lb);
                f2_split(lsum1, lc, ld);
                part_max = m_used;
                part_sum = (la + lb) + (lc + ld);
                part_tiles = it.n;
            }
            else if (rows_live) {
                float la, lb, lc, ld;
                f2_split(lsum0, la, lb);
                f2_split(lsum1, lc, ld);
                const float lsum = (la + lb) + (lc + ld);
                const float inv = m_used == -INFINITY && lsum == lsum ? 0.0f : 1.0f / lsum;
                T *dst = reinterpret_cast<T *>(a.o) + it.seq * a.os0 + (long)q * a.old + it.head * a.os1;
#pragma unroll
                for (int c = 0; c < HDP; c += 32) {
                    uint32_t ov[32];
                    if (it.n > 0) {
                        tmem_ld32(tO + c, ov);
                        tmem_wait_ld();
                    }
                    else {
#pragma unroll
                        for (int e = 0; e < 32; e++)
                            ov[e] = 0;
                    }
                    if (q < a.Nq) {
#pragma unroll
                        for (int e = 0; e < 32; e += 8) {
                            if (c + e >= a.hd)
                                break;
                            uint32_t w[4];
#pragma unroll
                            for (int i = 0; i < 4; i++)
                                w[i] = pack2<T>(__uint_as_float(ov[e + 2 * i]) * inv,
                                                __uint_as_float(ov[e + 2 * i + 1]) * inv);
                            if (a.ovec)
                                *reinterpret_cast<uint4 *>(dst + c + e) = make_uint4(w[0], w[1], w[2], w[3]);
                            else {
#pragma unroll
                                for (int i = 0; i < 8; i++)
                                    dst[c + e + i] = from_f<T>(__uint_as_float(ov[e + i]) * inv);
                            }
                        }
                    }
                }
                tc_fence_before();
            }
        }
    }
    if constexpr (SPLIT) {
        using PT = Parts<HDP>;
        const Item it = item_at(first);
        const int live = min(BQ, a.Nq - it.qt * BQ), rl = BQ / a.cs;
        float *part = reinterpret_cast<float *>(smem);
        __syncwarp();
        cluster_sync_all();  // every copy has landed and every product is done in all CTAs: the stages are free
        if (warp < kProducerWarp && warp * 32 < live) {
            const int r = warp * 32 + lane;
            const uint32_t tO = tmem_base + ((uint32_t)(warp * 32) << 16) + G::TM_O;
            const uint32_t dst =
                mapa_shared(smem_addr(part + (rank * rl + r / a.cs) * PT::PR), r % a.cs);
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < HDP; c += 32) {
                uint32_t ov[32];
                if (part_tiles > 0) {
                    tmem_ld32(tO + c, ov);
                    tmem_wait_ld();
                }
                else {
#pragma unroll
                    for (int e = 0; e < 32; e++)
                        ov[e] = 0;
                }
#pragma unroll
                for (int e = 0; e < 32; e += 4)
                    st_dsmem4(dst + (c + e) * 4, __uint_as_float(ov[e]), __uint_as_float(ov[e + 1]),
                              __uint_as_float(ov[e + 2]), __uint_as_float(ov[e + 3]));
            }
            st_dsmem2(dst + HDP * 4, part_max, part_sum);
        }
        __syncwarp();
        cluster_sync_all();
        const int mine = live > rank ? (live - 1 - rank) / a.cs + 1 : 0;
        T *ob = reinterpret_cast<T *>(a.o) + it.seq * a.os0 + it.head * a.os1;
        PT::template merge<kThreads, false>(part, a.cs, rl, mine, a.scale_log2, [&](int i, int c, float x, float y, float z, float w) {
            if (c >= a.hd)
                return;
            T *dst = ob + (long)(it.qt * BQ + i * a.cs + rank) * a.old + c;
            if (a.ovec)
                *reinterpret_cast<uint2 *>(dst) = make_uint2(pack2<T>(x, y), pack2<T>(z, w));
            else {
                dst[0] = from_f<T>(x);
                dst[1] = from_f<T>(y);
                dst[2] = from_f<T>(z);
                dst[3] = from_f<T>(w);
            }
        });
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem_base, G::TM_COLS);
    }
}

// 4-D map (column, row, head, sequence) of an operand, box 64 columns x
// box_rows; dimensions that repeat (stride 0) or have one step are dropped.
bool make_map(CUtensorMap *map, bool bf16, const void *p, int hd, long rows, int heads, int nb, long ld, long s1,
              long s0, int box_rows, int &has1, int &has0)
{
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn)
        return false;
    has1 = heads > 1 && s1 != 0;
    has0 = nb > 1 && s0 != 0;
    cuuint64_t dims[4] = {(cuuint64_t)hd, (cuuint64_t)rows, (cuuint64_t)(has1 ? heads : 1), (cuuint64_t)(has0 ? nb : 1)};
    const cuuint64_t one = (cuuint64_t)hd * 2;  // a multiple of 16
    cuuint64_t strides[3] = {rows > 1 ? (cuuint64_t)ld * 2 : one, has1 ? (cuuint64_t)s1 * 2 : one,
                             has0 ? (cuuint64_t)s0 * 2 : one};
    cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void *>(p),
              dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int HDP, bool SPLIT, bool MASK>
int launch(TcArgs &ta, const CUtensorMap &tq, const CUtensorMap &tk, const CUtensorMap &tv, int grid, cudaStream_t s)
{
    const cudaError_t e = cluster_prepare_once<attn_cross_tc_kernel<T, HDP, SPLIT, MASK>>(Geo<HDP>::SMEM);
    if (e != cudaSuccess)
        return (int)e;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ta.x.cs;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Geo<HDP>::SMEM;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = SPLIT ? 2 : 1;
    return (int)cudaLaunchKernelEx(&cfg, attn_cross_tc_kernel<T, HDP, SPLIT, MASK>, tq, tk, tv, (const TcArgs)ta);
}

// Whether a cluster of c CTAs fits the device.
template <typename T, int HDP, bool MASK>
bool cluster_fits(int c)
{
    return cluster_prepare_once<attn_cross_tc_kernel<T, HDP, true, MASK>>(Geo<HDP>::SMEM) == cudaSuccess &&
           clusters_at_once<attn_cross_tc_kernel<T, HDP, true, MASK>>(c, kThreads, Geo<HDP>::SMEM) > 0;
}

template <typename T, int HDP>
int run(XaArgs &x, int nb, bool bf16, cudaStream_t s)
{
    constexpr int BKV = Geo<HDP>::BKV;
    TcArgs ta = {};
    CUtensorMap tq, tk, tv;
    if (!make_map(&tq, bf16, x.q, x.hd, x.Nq, x.heads, nb, x.qld, x.qs1, x.qs0, BQ, ta.qb1, ta.qb0) ||
        !make_map(&tk, bf16, x.k, x.hd, x.Nk, x.kvheads, nb, x.kld, x.ks1, x.ks0, BKV, ta.kb1, ta.kb0) ||
        !make_map(&tv, bf16, x.v, x.hd, x.Nk, x.kvheads, nb, x.vld, x.vs1, x.vs0, BKV, ta.vb1, ta.vb0))
        return K_ETMAP;
    x.nqt = (x.Nq + BQ - 1) / BQ;
    const long items = (long)nb * x.heads * x.nqt;
    const int slots = kCtasPerSm * device_sms(), nkv = (x.Nk + BKV - 1) / BKV;
    if (items > 0x3fffffffL)
        return K_EARG;
    ta.nitems = (int)items;
    // CTAs sharing an item's keys: as many as run at once (cluster scheduling
    // leaves a few slots), from ten tiles on: a tile takes about 0.75 us alone, the
    // merge 3.5 us (64 (sequence, head) pairs x 128 queries, cs 1 and 4: 8
    // tiles 11.8 and 12.6 us, 11 tiles 14.6 and 13.7 us).
    int cs = 1;
    while (nkv >= 10 && cs < kMaxSplit && items * cs * 2 <= slots - slots / 16 &&
           (x.kmask ? cluster_fits<T, HDP, true>(cs * 2) : cluster_fits<T, HDP, false>(cs * 2)))
        cs *= 2;
    x.cs = cs;
    ta.x = x;
    const int grid = cs > 1 ? (int)items * cs : (items < slots ? (int)items : slots);
    if (cs > 1)
        return x.kmask ? launch<T, HDP, true, true>(ta, tq, tk, tv, grid, s)
                       : launch<T, HDP, true, false>(ta, tq, tk, tv, grid, s);
    return x.kmask ? launch<T, HDP, false, true>(ta, tq, tk, tv, grid, s)
                   : launch<T, HDP, false, false>(ta, tq, tk, tv, grid, s);
}

}  // namespace

bool attn_cross_tc_takes(const XaArgs &a, int nb, int dt)
{
    if (dt == K_F32)
        return false;
    // a map wants 16-byte aligned starts and strides below 2^40 bytes
    auto fits = [&](const void *p, long ld, long s1, long s0, long rows, int heads) {
        auto ok = [](long st, long n) { return n == 1 || (st % 8 == 0 && st < (1L << 38)); };
        return !(reinterpret_cast<uintptr_t>(p) & 15) && ok(ld, rows) && (rows == 1 || ld > 0) && ok(s1, heads) &&
               ok(s0, nb);
    };
    return fits(a.q, a.qld, a.qs1, a.qs0, a.Nq, a.heads) && fits(a.k, a.kld, a.ks1, a.ks0, a.Nk, a.kvheads) &&
           fits(a.v, a.vld, a.vs1, a.vs0, a.Nk, a.kvheads);
}

int attn_cross_tc(XaArgs &a, int nb, int dt, cudaStream_t s)
{
    if (dt == K_BF16)
        return a.hd <= 64 ? run<__nv_bfloat16, 64>(a, nb, true, s) : run<__nv_bfloat16, 128>(a, nb, true, s);
    return a.hd <= 64 ? run<__half, 64>(a, nb, false, s) : run<__half, 128>(a, nb, false, s);
}

}  // namespace sam3
