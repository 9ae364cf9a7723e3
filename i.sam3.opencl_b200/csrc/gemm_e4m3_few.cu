// SPDX-License-Identifier: Unlicense
// Product of E4M3 matrices with block scales for few rows of A (single tokens of some
// sequences): the weights are read once for 32 rows, from memory into the operand
// registers of mma.sync (m16n8k32), with no stage in between; what counts is how many
// loads are in flight. A CTA takes 16 rows of B (columns of C), its warps k-blocks of
// 128 in turn; the warps' sums meet in shared memory, added in their order. A block's
// product starts from zero and is added times its scales, as in the other forms.
// 8 x 4096 x 1024 and 8 x 1024 x 4096: the launch (4.7 us a call in a row of calls, 6.0 and
// 10.0 by tcgen05 tiles); 32 x 4096 x 4096 13.1 us.
//
// A lane reads 16 adjacent bytes of its rows of B and of A. The instruction wants
// columns 4 t .. and 16 + 4 t .. of lane t; a sum over columns may take them in any
// order that is the same for both operands.
#include "gemm_e4m3.cuh"
#include "pdl.cuh"

namespace sam3 {
namespace {

constexpr int kRowsB = 16;

struct FewArgs {
    E4Args p;
    const uint8_t *a, *b;
    long lda, ldb;
};

__device__ __forceinline__ void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes of a row at column k, zeros behind its K columns (and for in false).
__device__ __forceinline__ uint4 row16(const uint8_t *row, int k, int K, bool in)
{
    if (in && k + 16 <= K)
        return __ldg(reinterpret_cast<const uint4 *>(row + k));
    uint32_t w[4] = {0, 0, 0, 0};
    if (in && k < K) {
#pragma unroll
        for (int e = 0; e < 16; e++)
            if (k + e < K)
                w[e / 4] |= (uint32_t)__ldg(row + k + e) << (8 * (e & 3));
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// MT: groups of eight rows of A; W: warps.
template <int MT, int W>
__global__ void __launch_bounds__(32 * W) gemm_few_kernel(const __grid_constant__ FewArgs f)
{
    constexpr int kPad = 8 * MT + 1;
    __shared__ float sums[W][kRowsB * kPad];
    const E4Args &p = f.p;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * kRowsB, m0 = blockIdx.y * 8 * MT;
    const int kblocks = (p.K + kScaleBlock - 1) / kScaleBlock;
    const uint8_t *b0 = f.b + (long)(n0 + g) * f.ldb, *b1 = f.b + (long)(n0 + g + 8) * f.ldb;
    const bool in0 = n0 + g < p.N, in1 = n0 + g + 8 < p.N;
    const long rb = (long)(n0 / kScaleBlock) * p.ldsb;
    float acc[MT][4];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int e = 0; e < 4; e++)
            acc[i][e] = 0.0f;
    griddep_wait();
    griddep_launch();
#pragma unroll 2
    for (int kb = warp; kb < kblocks; kb += W) {
        const int k = kb * kScaleBlock + t * 16;
        uint4 w0[2], w1[2], x[MT][2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            w0[h] = row16(b0, k + 64 * h, p.K, in0);
            w1[h] = row16(b1, k + 64 * h, p.K, in1);
        }
        const uint32_t sb = scale_raw(p.sb, p.sbdt, rb + kb);
        uint32_t sa[MT][2];
#pragma unroll
        for (int i = 0; i < MT; i++) {
#pragma unroll
            for (int h = 0; h < 2; h++)
                x[i][h] = row16(f.a + (long)(m0 + 8 * i + g) * f.lda, k + 64 * h, p.K, m0 + 8 * i + g < p.M);
#pragma unroll
            for (int e = 0; e < 2; e++)
                sa[i][e] = scale_raw(p.sa, p.sadt, (long)min(m0 + 8 * i + 2 * t + e, p.M - 1) * p.ldsa + kb);
        }
        const float sbv = scale_of(sb, p.sbdt);
#pragma unroll
        for (int i = 0; i < MT; i++) {
            float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int h = 0; h < 2; h++) {
                mma_e4m3(d, w0[h].x, w1[h].x, w0[h].y, w1[h].y, x[i][h].x, x[i][h].y);
                mma_e4m3(d, w0[h].z, w1[h].z, w0[h].w, w1[h].w, x[i][h].z, x[i][h].w);
            }
            const float s0 = scale_of(sa[i][0], p.sadt) * sbv, s1 = scale_of(sa[i][1], p.sadt) * sbv;
            acc[i][0] = fmaf(d[0], s0, acc[i][0]);
            acc[i][1] = fmaf(d[1], s1, acc[i][1]);
            acc[i][2] = fmaf(d[2], s0, acc[i][2]);
            acc[i][3] = fmaf(d[3], s1, acc[i][3]);
        }
    }
    // element (row of B, row of A) of a warp's sums
#pragma unroll
    for (int i = 0; i < MT; i++) {
        float *s = &sums[warp][g * kPad + 8 * i + 2 * t];
        s[0] = acc[i][0];
        s[1] = acc[i][1];
        s[8 * kPad] = acc[i][2];
        s[8 * kPad + 1] = acc[i][3];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kRowsB * 8 * MT; i += 32 * W) {
        const int j = i % kRowsB, r = i / kRowsB, m = m0 + r, n = n0 + j;
        if (n >= p.N || m >= p.M)
            continue;
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < W; w++)
            v += sums[w][j * kPad + r];
        if (p.bias)
            v += __ldg(p.bias + n);
        if (p.act == K_ACT_GELU) {
            float u = 0.0f;
            if (p.cdt == K_F32)
                v = 0.5f * v * (1.0f + erff(v * 0.70710678118654752f));
            else
                gelu_pair_exp(v, u);
        }
        else if (p.act == K_ACT_RELU)
            asm("max.NaN.f32 %0, %0, %1;" : "+f"(v) : "f"(0.0f));
        store1(p.c, p.cdt, (long)m * p.ldc + n, v);
    }
}

template <int MT>
int launch_w(const FewArgs &f, int kblocks, cudaStream_t s)
{
    const dim3 grid((f.p.N + kRowsB - 1) / kRowsB, (f.p.M + 8 * MT - 1) / (8 * MT));
    // A warp for two k-blocks, up to 16.
    if (kblocks > 16)
        return launch_pdl(gemm_few_kernel<MT, 16>, grid, dim3(512), 0, s, f);
    if (kblocks > 4)
        return launch_pdl(gemm_few_kernel<MT, 8>, grid, dim3(256), 0, s, f);
    return launch_pdl(gemm_few_kernel<MT, 4>, grid, dim3(128), 0, s, f);
}

}  // namespace

int launch_few(const E4Args &p, const struct k_rows *A, const struct k_rows *B, cudaStream_t s)
{
    const FewArgs f = {p, reinterpret_cast<const uint8_t *>(A->p), reinterpret_cast<const uint8_t *>(B->p), A->ld, B->ld};
    const int kb = (p.K + kScaleBlock - 1) / kScaleBlock;
    if (p.M <= 8)
        return launch_w<1>(f, kb, s);
    return p.M <= 16 ? launch_w<2>(f, kb, s) : launch_w<4>(f, kb, s);
}

}  // namespace sam3
