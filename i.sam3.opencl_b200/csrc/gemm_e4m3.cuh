// SPDX-License-Identifier: Unlicense
// What the forms of the E4M3 product share: arguments, the reading of scales, and
// the epilogue of a thread that holds 128 columns of a row.
#pragma once

#include "act.cuh"
#include "e4m3.cuh"
#include "kernels.h"
#include "tc_ptx.cuh"
#include "tmap.cuh"
#include "vec8.cuh"

namespace sam3 {

constexpr int kStageTile = 32 * 128;  // a warp's 32 rows x 128 bytes of C
constexpr int kChunk = 4;             // k-blocks whose scales are handed over at once

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
    int tma;   // C is stored through its tensor map:
    int ntma;  // its columns up to here, the others by elements
    int *err;
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

// Element j of row r of the staged chunk to element i of C; es: bytes of an element.
__device__ __forceinline__ void copy_staged(const E4Args &p, int es, uint32_t tile, int r, int j, long i)
{
    const int byte = j * es;
    const uint32_t src = tile + r * 128 + (((byte >> 4) ^ (r & 7)) << 4) + (byte & 15);
    if (es == 4) {
        uint32_t v;
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(src) : "memory");
        reinterpret_cast<uint32_t *>(p.c)[i] = v;
    }
    else if (es == 2) {
        uint16_t v;
        asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(src) : "memory");
        reinterpret_cast<uint16_t *>(p.c)[i] = v;
    }
    else {
        uint16_t v;
        asm volatile("{.reg .b8 t; ld.shared.b8 t, [%1]; cvt.u16.u8 %0, t;}" : "=h"(v) : "r"(src) : "memory");
        reinterpret_cast<uint8_t *>(p.c)[i] = (uint8_t)v;
    }
}

// The staged chunk to C at rows m0 .., columns n ..: by TMA, or element by element
// along the rows where C's rows are not 16-byte aligned. TMA writes whole 16-byte
// pieces, past the end of its map's rows too: the map ends with the row's last whole
// piece, the elements behind it each lane copies from the row that it staged.
__device__ __forceinline__ void store_chunk(const E4Args &p, const CUtensorMap *tmC, uint32_t tile, int lane, int m0,
                                            int n)
{
    const int es = p.cdt == K_F32 ? 4 : (p.cdt == K_E4M3 ? 1 : 2), per = 128 / es;
    if (p.tma) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 && n < p.ntma) {
            tma_store_2d(tmC, reinterpret_cast<const void *>(__cvta_shared_to_generic(tile)), n, m0);
            bulk_commit();
        }
        if (m0 + lane < p.M) {
#pragma unroll 1
            for (int j = max(p.ntma, n); j < min(p.N, n + per); j++)
                copy_staged(p, es, tile, lane, j - n, (long)(m0 + lane) * p.ldc + j);
        }
        return;
    }
    __syncwarp();
    for (int r = 0; r < 32 && m0 + r < p.M; r++) {
        const long row = (long)(m0 + r) * p.ldc + n;
        for (int j = lane; j < per && n + j < p.N; j += 32)
            copy_staged(p, es, tile, r, j, row + j);
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
            gelu_pair_exp(acc[j], acc[j + 1]);
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

// A kernel over tiles of 128 (PAIR: 256) x BN, one CTA or pair to an SM or two;
// K_EARG: pairs cannot be launched here.
template <auto Kern, int BN, bool PAIR, int B_ROWS, int THREADS, int SMEM>
inline int launch_tiles(const E4Args &p, const struct k_rows *A, const struct k_rows *B, const CUtensorMap &tc,
                        cudaStream_t s)
{
    constexpr int BM = 128, BK = 128;
    CUtensorMap ta, tb;
    // a single row's pitch is of no account
    const uint64_t pitch = ((uint64_t)p.K + 15) / 16 * 16;
    if (!make_tmap_2d(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, A->p, (uint64_t)p.M, (uint64_t)p.K,
                      p.M > 1 ? (uint64_t)A->ld : pitch, BK, BM) ||
        !make_tmap_2d(&tb, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, B->p, (uint64_t)p.N, (uint64_t)p.K,
                      p.N > 1 ? (uint64_t)B->ld : pitch, BK, B_ROWS))
        return K_ETMAP;
    const cudaError_t e = smem_limit_once<Kern>(SMEM);
    if (e != cudaSuccess)
        return (int)e;
    const int tiles = (p.M + (PAIR ? 2 : 1) * BM - 1) / ((PAIR ? 2 : 1) * BM) * ((p.N + BN - 1) / BN);
    const int sms = device_sms();
    if constexpr (!PAIR)
        return launch_pdl(Kern, dim3(tiles < sms ? tiles : sms), dim3(THREADS), SMEM, s, ta, tb, tc, p);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(sms / 2 * 2);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = SMEM;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    static PerDevice pairs;
    const int most = clusters_of<Kern>(pairs, cfg);
    if (most <= 0)
        return K_EARG;
    cfg.gridDim = dim3(2 * (tiles < most ? tiles : most));
    cfg.numAttrs = 2;
    return (int)cudaLaunchKernelEx(&cfg, Kern, ta, tb, tc, p);
}

// The form for few rows of A and results that are not E4M3 (gemm_e4m3_few.cu).
int launch_few(const E4Args &p, const struct k_rows *A, const struct k_rows *B, cudaStream_t s);

// The form for E8M0 scales (gemm_e4m3_mx.cu), and its time in 1/100 us.
long cost_mx(const E4Args &p);
int launch_mx(const E4Args &p, const struct k_rows *A, const struct k_rows *B, const CUtensorMap &tc, cudaStream_t s);

}  // namespace sam3
