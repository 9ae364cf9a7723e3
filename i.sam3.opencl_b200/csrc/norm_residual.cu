// SPDX-License-Identifier: Unlicense
// What stands between two blocks of a transformer, one pass over the residual
// stream: h = post(H), r = X + alpha ls gate h, R = r, Y = pre(r) (1 + scale) +
// shift, in 32 bits; Y rounded to its type or quantised to E4M3 (blocks of 128
// columns are the 16 lanes of a half-warp, eight adjacent columns a lane). Memory
// bound: X and H read, R and Y written once.
//
// T threads hold a row in registers, 8 V columns a thread, so that mean and
// variance are two sums over values at hand (no E[x^2] - E[x]^2); rows wider than
// that are read again for each sum, from L2.
#include "div.cuh"
#include "e4m3.cuh"
#include "kernels.h"
#include "pdl.cuh"
#include "tmap.cuh"
#include "vec8.cuh"

#include <type_traits>

namespace sam3 {
namespace {

struct NormArgs {
    k_norm_args p;
    Div dN;
    long rows;
    long chunk;   // rows of a CTA (SHARED)
    float share;  // 1 / C
    int gaterow, scalerow, shiftrow;  // the operand is read with each row, not kept with a sample's vectors
};

// Sum over the T threads of a row in a fixed order; every thread gets it. A row of
// more than one warp is a CTA's: smem holds two rounds of its warps' sums, used in
// turn, so that one barrier a sum is enough.
template <int T>
__device__ __forceinline__ float row_sum(float v, float *smem, int &turn)
{
#pragma unroll
    for (int o = (T < 32 ? T : 32) / 2; o; o >>= 1)
        v += __shfl_xor_sync(0xffffffffu, v, o);
    if constexpr (T > 32) {
        float *s = smem + turn * 32;
        turn ^= 1;
        if ((threadIdx.x & 31) == 0)
            s[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < T / 32; w++)
            v += s[w];
    }
    return v;
}

__device__ __forceinline__ long at_row(const k_rows &k, long b, long n)
{
    return b * k.s0 + n * k.ld;
}

// The columns of a thread: eight adjacent ones of every 8 T (VEC: aligned rows of a
// multiple of eight), or
// every 32nd of a warp's 256 V (rows that are not aligned: 32 adjacent elements to
// an access). Either way 128-column blocks lie within a warp.
template <int T, int V, bool VEC>
struct Cols {
    int first;
    __device__ __forceinline__ Cols()
    {
        const int lane = threadIdx.x & (T - 1);
        first = VEC ? lane * 8 : (lane >> 5) * (256 * V) + (lane & 31);
    }
    // VEC: C is a multiple of eight, so that eight columns end together
    __device__ __forceinline__ bool in(int j, int e, int C) const { return at(j, VEC ? 0 : e) < C; }
    __device__ __forceinline__ int at(int j, int e) const
    {
        return VEC ? first + j * 8 * T + e : first + (j * 8 + e) * 32;
    }
};

// go(element type as a constant): one branch for a loop over elements.
template <typename F>
__device__ __forceinline__ void typed(int dt, const F &go)
{
    if (dt == K_F32)
        go(std::integral_constant<int, K_F32>{});
    else if (dt == K_BF16)
        go(std::integral_constant<int, K_BF16>{});
    else
        go(std::integral_constant<int, K_F16>{});
}

// The values of a row of X or H (either may be R or Y too), as stored where they are
// vectors. DT: its type, or kAnyType for the type that the operand names.
constexpr int kAnyType = -1;
template <int V, bool VEC, int DT>
struct Row {
    static constexpr bool NARROW = DT == K_BF16 || DT == K_F16;
    uint4 w[VEC ? V : 1][NARROW ? 1 : 2];
    float f[VEC ? 1 : V][8];

    template <int T>
    __device__ __forceinline__ void load(const k_rows &k, long base, const Cols<T, V, VEC> &c, int C)
    {
        const int dt = DT == kAnyType ? k.dt : DT;
        if constexpr (VEC) {
#pragma unroll
            for (int j = 0; j < V; j++) {
                const Raw8 r = c.in(j, 0, C) ? load8<true>(k.p, dt, base + c.at(j, 0), 8) : Raw8{};
                w[j][0] = r.a;
                if constexpr (!NARROW)
                    w[j][1] = r.b;
            }
        }
        else {
            typed(dt, [&](auto t) {
#pragma unroll
                for (int j = 0; j < V; j++)
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        f[j][e] = c.in(j, e, C) ? elem<true>(k.p, decltype(t)::value, base + c.at(j, e)) : 0.0f;
            });
        }
    }
    __device__ __forceinline__ void get(int any, int j, float (&v)[8]) const
    {
        const int dt = DT == kAnyType ? any : DT;
        if constexpr (VEC) {
            Raw8 r;
            r.a = w[j][0];
            if constexpr (NARROW)
                r.b = make_uint4(0, 0, 0, 0);
            else
                r.b = w[j][1];
            unpack8(r, dt, v);
        }
        else {
#pragma unroll
            for (int e = 0; e < 8; e++)
                v[e] = f[j][e];
        }
    }
};

// Eight values of a 32-bit vector of C columns (NULL: `none`) in global memory.
template <int T, int V, bool VEC>
__device__ __forceinline__ void param8(const float *p, const Cols<T, V, VEC> &c, int j, int C, float none, float (&v)[8])
{
#pragma unroll
    for (int e = 0; e < 8; e++)
        v[e] = none;
    if (!p)
        return;
    if constexpr (VEC) {
        if (!c.in(j, 0, C))
            return;
        const float4 a = __ldg(reinterpret_cast<const float4 *>(p + c.at(j, 0)));
        const float4 b = __ldg(reinterpret_cast<const float4 *>(p + c.at(j, 4)));
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
        v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    }
    else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (c.in(j, e, C))
                v[e] = __ldg(p + c.at(j, e));
    }
}

// Eight values of an operand's row.
template <int T, int V, bool VEC>
__device__ __forceinline__ void operand8(const k_rows &k, long base, const Cols<T, V, VEC> &c, int j, int C, float (&v)[8])
{
    if constexpr (VEC)
        unpack8(c.in(j, 0, C) ? load8<true>(k.p, k.dt, base + c.at(j, 0), 8) : Raw8{}, k.dt, v);
    else
        typed(k.dt, [&](auto t) {
#pragma unroll
            for (int e = 0; e < 8; e++)
                v[e] = c.in(j, e, C) ? elem(k.p, decltype(t)::value, base + c.at(j, e)) : 0.0f;
        });
}

// What multiplies and is added to a normalised row: one vector each, kept in shared
// memory for the rows of a sample (SHARED); VEC: in two halves of four columns of
// every eight, so that a warp's 16-byte reads meet no bank twice.
template <int T, int V, bool VEC>
__device__ __forceinline__ void shared8(const float *s, const Cols<T, V, VEC> &c, int j, int half, float (&v)[8])
{
    if constexpr (VEC) {
        const float4 a = *reinterpret_cast<const float4 *>(s + c.at(j, 0) / 2);
        const float4 b = *reinterpret_cast<const float4 *>(s + half + c.at(j, 0) / 2);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
        v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    }
    else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            v[e] = s[c.at(j, e)];
    }
}

template <int V>
__device__ __forceinline__ float sum_of(const float (&v)[V][8])
{
    float s[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        s[e] = v[0][e];
#pragma unroll
        for (int j = 1; j < V; j++)
            s[e] += v[j][e];
    }
    return ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
}

// v becomes (v - mean) / sqrt(variance + eps) (RMS: mean 0); columns behind C hold 0
// and count for nothing.
template <int T, int V, bool VEC>
__device__ __forceinline__ void normalise(const k_norm &k, const Cols<T, V, VEC> &c, int C, float share, float *smem,
                                          int &turn, float (&v)[V][8])
{
    if (k.kind == K_NORM_LAYER) {
        const float mean = row_sum<T>(sum_of(v), smem, turn) * share;
#pragma unroll
        for (int j = 0; j < V; j++)
#pragma unroll
            for (int e = 0; e < 8; e++)
                v[j][e] = c.in(j, e, C) ? v[j][e] - mean : 0.0f;
    }
    float q[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        q[e] = v[0][e] * v[0][e];
#pragma unroll
        for (int j = 1; j < V; j++)
            q[e] = fmaf(v[j][e], v[j][e], q[e]);
    }
    const float q1 = ((q[0] + q[1]) + (q[2] + q[3])) + ((q[4] + q[5]) + (q[6] + q[7]));
    const float rstd = rsqrtf(fmaf(row_sum<T>(q1, smem, turn), share, k.eps));
#pragma unroll
    for (int j = 0; j < V; j++)
#pragma unroll
        for (int e = 0; e < 8; e++)
            v[j][e] *= rstd;
}

// Y's eight values (and, of E4M3, their block's scale).
template <int T, int V, bool VEC, int XT>
__device__ __forceinline__ void put8(const k_norm_args &p, long y, long s, const Cols<T, V, VEC> &c, int j,
                                     bool write, const float (&v)[8])
{
    const int dt = XT == K_BF16 || XT == K_F16 ? XT : p.Y.dt;  // where it is not E4M3
    if (p.Y.dt != K_E4M3) {
        if constexpr (VEC) {
            if (write && c.in(j, 0, p.C))
                store8<true>(p.Y.p, dt, y + c.at(j, 0), 8, v);
        }
        else if (write)
            typed(dt, [&](auto t) {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (c.in(j, e, p.C))
                        store1(p.Y.p, decltype(t)::value, y + c.at(j, e), v[e]);
            });
        return;
    }
    // a half-warp holds a block of 128 columns (VEC), else four values of each lane
    constexpr int G = VEC ? 8 : 4;
    auto largest = [&](int g, bool finite) {
        float m = 0.0f;
#pragma unroll
        for (int e = g; e < g + G; e++)
            if (c.in(j, e, p.C))
                m = finite ? larger_finite(m, v[e]) : larger(m, v[e]);
#pragma unroll
        for (int o = VEC ? (T < 16 ? T / 2 : 8) : 16; o; o >>= 1)
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        return m;
    };
#pragma unroll
    for (int g = 0; g < 8; g += G) {
        float m = largest(g, false);
        const bool inf = __any_sync(0xffffffffu, infinite(m));
        if (inf)
            m = largest(g, true);
        const uint32_t byte = scale_byte(m);
        const float inv = scale_inverse(byte);
        if constexpr (VEC) {
            if (write && c.in(j, 0, p.C))
                store8_e4m3<true>(p.Y.p, y + c.at(j, 0), 8, pack8_e4m3(v, inv, inf));
        }
        else {
            const uint32_t w = inf ? pack_e4m3<true>(v[g], v[g + 1], v[g + 2], v[g + 3], inv)
                                   : pack_e4m3<false>(v[g], v[g + 1], v[g + 2], v[g + 3], inv);
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (c.in(j, g + e, p.C))
                    reinterpret_cast<uint8_t *>(p.Y.p)[y + c.at(j, g + e)] = (uint8_t)(w >> (8 * e));
        }
        if ((threadIdx.x & (VEC ? (T < 16 ? T - 1 : 15) : 31)) == 0 && write && c.in(j, g, p.C))
            put_scale(p.S.p, p.S.dt, s + c.at(j, VEC ? 0 : g) / kScaleBlock, byte);
    }
}

__host__ __device__ constexpr int cta_threads(int T) { return T < 256 ? (T > 32 ? T : 256) : T; }

// CTAs an SM is to hold (0: left to the compiler). Of wide rows without the shared vectors as many as 64
// registers a thread allow (4000 rows of 6000 fp32: 159 us with one CTA, 113 with two); with
// them the next row's loads would be spilled (20000 rows of 2048 fp32: 107 and 160).
template <int T, int V, bool VEC, bool SHARED>
__host__ __device__ constexpr int ctas_wanted()
{
    return VEC && !SHARED && T > 32 && V == 2 ? 1024 / T : 0;
}

// T threads to a row. SHARED: a CTA takes a range of rows and keeps the vectors of
// their sample in shared memory; else every row reads them (few rows).
// XT, HT: the types of X (and R) and of H.
template <int T, int V, bool VEC, int XT, int HT, bool SHARED>
__global__ void __launch_bounds__(cta_threads(T), ctas_wanted<T, V, VEC, SHARED>()) norm_rows_kernel(const __grid_constant__ NormArgs a)
{
    constexpr int kRows = cta_threads(T) / T;  // rows of a CTA at a time
    constexpr int kHalf = V * T * 4;           // floats of half a vector
    extern __shared__ float vectors[];         // FG, FB, PG, PB: r = x + (FG h + FB), y = PG r + PB
    __shared__ float smem[64];
    int turn = 0;
    const k_norm_args &p = a.p;
    const Cols<T, V, VEC> c;
    griddep_wait();
    griddep_launch();
    const int sub = threadIdx.x / T;
    const bool post = p.post.kind != K_NORM_NONE, pre = p.Y.p && p.pre.kind != K_NORM_NONE;
    const bool useFB = post && p.post.b;
    const bool usePG = p.Y.p && (p.pre.g || (p.scale.p && !a.scalerow));
    const bool usePB = p.Y.p && ((pre && p.pre.b) || (p.shift.p && !a.shiftrow));
    long row = SHARED ? (long)blockIdx.x * a.chunk : (long)blockIdx.x * kRows + sub;
    const long end = SHARED ? min(row + a.chunk, a.rows) : a.rows;
    // Rows of one warp step together (T < 32): one behind the last is read again, not
    // written.
    constexpr int kTogether = T < 32 ? 32 / T : 1;
    while ((SHARED ? row : row - sub % kTogether) < end) {
        const bool last = !SHARED && row >= end;
        const long here = last ? end - 1 : row;
        const long b = quot((uint32_t)here, a.dN);
        long stop = here + 1, step = 1L << 40;
        if constexpr (SHARED) {
            stop = min(end, (b + 1) * p.N);
            step = kRows;
            __syncthreads();  // the last sample's rows are done with the vectors
            for (int i = threadIdx.x; i < p.C; i += blockDim.x) {
                const int at = VEC ? (i & 4 ? kHalf : 0) + (i >> 3) * 4 + (i & 3) : i;
                float f = p.alpha;
                if (p.ls)
                    f *= __ldg(p.ls + i);
                if (p.gate.p && !a.gaterow)
                    f *= elem(p.gate.p, p.gate.dt, b * p.gate.s0 + i);
                vectors[at] = post && p.post.g ? f * __ldg(p.post.g + i) : f;
                if (useFB)
                    vectors[2 * kHalf + at] = f * __ldg(p.post.b + i);
                const float s = p.scale.p && !a.scalerow ? 1.0f + elem(p.scale.p, p.scale.dt, b * p.scale.s0 + i) : 1.0f;
                if (usePG)
                    vectors[4 * kHalf + at] = pre && p.pre.g ? s * __ldg(p.pre.g + i) : s;
                if (usePB)
                    vectors[6 * kHalf + at] = (pre && p.pre.b ? s * __ldg(p.pre.b + i) : 0.0f) +
                                              (p.shift.p && !a.shiftrow ? elem(p.shift.p, p.shift.dt, b * p.shift.s0 + i) : 0.0f);
            }
            __syncthreads();
        }
        // The next row's loads are in flight beside this one's arithmetic.
        Row<V, VEC, XT> x, xnext;
        Row<V, VEC, HT> hnext;
        auto fetch = [&](long q) {
            xnext.load(p.X, at_row(p.X, b, q - b * p.N), c, p.C);
            if (p.H.p)
                hnext.load(p.H, at_row(p.H, b, q - b * p.N), c, p.C);
        };
        long q = SHARED ? row + sub : here;
        auto held = [&](long q) { return kTogether > 1 ? min(q, stop - 1) : q; };
        auto goes = [&](long q) { return (SHARED ? q - sub % kTogether : q) < stop; };
        if (goes(q))
            fetch(held(q));
#pragma unroll 1
        for (long at = q; goes(at); at += step) {
            q = held(at);
            const bool write = !last && at < stop;
            const long n = q - b * p.N;
            float r[V][8];
            x = xnext;
            if (p.H.p) {
#pragma unroll
                for (int j = 0; j < V; j++)
                    hnext.get(p.H.dt, j, r[j]);
            }
            if (SHARED && goes(at + step))
                fetch(held(at + step));
            if (p.H.p) {
                if (post)
                    normalise<T, V, VEC>(p.post, c, p.C, a.share, smem, turn, r);
#pragma unroll
                for (int j = 0; j < V; j++) {
                    float f[8], xv[8], t[8];
                    if constexpr (SHARED) {
                        shared8<T, V, VEC>(vectors, c, j, kHalf, f);
#pragma unroll
                        for (int e = 0; e < 8; e++)
                            t[e] = f[e] * r[j][e];
                        if (useFB) {
                            shared8<T, V, VEC>(vectors + 2 * kHalf, c, j, kHalf, f);
#pragma unroll
                            for (int e = 0; e < 8; e++)
                                t[e] += f[e];
                        }
                        if (p.gate.p && a.gaterow) {
                            operand8<T, V, VEC>(p.gate, at_row(p.gate, b, n), c, j, p.C, f);
#pragma unroll
                            for (int e = 0; e < 8; e++)
                                t[e] *= f[e];
                        }
                    }
                    else {
                        float g[8];
                        if (post) {
                            param8<T, V, VEC>(p.post.g, c, j, p.C, 1.0f, f);
                            param8<T, V, VEC>(p.post.b, c, j, p.C, 0.0f, g);
#pragma unroll
                            for (int e = 0; e < 8; e++)
                                r[j][e] = fmaf(r[j][e], f[e], g[e]);
                        }
                        param8<T, V, VEC>(p.ls, c, j, p.C, 1.0f, f);
#pragma unroll
                        for (int e = 0; e < 8; e++)
                            t[e] = r[j][e] * (p.alpha * f[e]);
                        if (p.gate.p) {
                            operand8<T, V, VEC>(p.gate, at_row(p.gate, b, n), c, j, p.C, g);
#pragma unroll
                            for (int e = 0; e < 8; e++)
                                t[e] *= g[e];
                        }
                    }
                    x.get(p.X.dt, j, xv);
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        r[j][e] = c.in(j, e, p.C) ? xv[e] + t[e] : 0.0f;
                }
            }
            else {
#pragma unroll
                for (int j = 0; j < V; j++)
                    x.get(p.X.dt, j, r[j]);
            }
            if (p.R.p && write) {
                const long at = at_row(p.R, b, n);
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const int dt = XT == kAnyType ? p.R.dt : XT;
                    if constexpr (VEC) {
                        if (c.in(j, 0, p.C))
                            store8<true>(p.R.p, dt, at + c.at(j, 0), 8, r[j]);
                    }
                    else
                        typed(dt, [&](auto t) {
#pragma unroll
                            for (int e = 0; e < 8; e++)
                                if (c.in(j, e, p.C))
                                    store1(p.R.p, decltype(t)::value, at + c.at(j, e), r[j][e]);
                        });
                }
            }
            if (!p.Y.p)
                continue;
            if (pre)
                normalise<T, V, VEC>(p.pre, c, p.C, a.share, smem, turn, r);
#pragma unroll
            for (int j = 0; j < V; j++) {
                float f[8];
                if constexpr (SHARED) {
                    if (usePG) {
                        shared8<T, V, VEC>(vectors + 4 * kHalf, c, j, kHalf, f);
#pragma unroll
                        for (int e = 0; e < 8; e++)
                            r[j][e] *= f[e];
                    }
                    if (usePB) {
                        shared8<T, V, VEC>(vectors + 6 * kHalf, c, j, kHalf, f);
#pragma unroll
                        for (int e = 0; e < 8; e++)
                            r[j][e] += f[e];
                    }
                }
                else if (pre) {
                    float g[8];
                    param8<T, V, VEC>(p.pre.g, c, j, p.C, 1.0f, f);
                    param8<T, V, VEC>(p.pre.b, c, j, p.C, 0.0f, g);
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        r[j][e] = fmaf(r[j][e], f[e], g[e]);
                }
                if (p.scale.p && (!SHARED || a.scalerow)) {
                    operand8<T, V, VEC>(p.scale, at_row(p.scale, b, n), c, j, p.C, f);
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        r[j][e] = fmaf(r[j][e], f[e], r[j][e]);
                }
                if (p.shift.p && (!SHARED || a.shiftrow)) {
                    operand8<T, V, VEC>(p.shift, at_row(p.shift, b, n), c, j, p.C, f);
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        r[j][e] += f[e];
                }
                put8<T, V, VEC, XT>(p, at_row(p.Y, b, n), at_row(p.S, b, n), c, j, write, r[j]);
            }
        }
        row = SHARED ? stop : row + (long)gridDim.x * kRows;
    }
}

// Where a thread's columns of a row lie.
struct At {
    long x, h, gate, r, scale, shift, y, s;
};

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
                                      const float (&h)[8], float (&r)[8])
{
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; e++)
        f[e] = p.ls && e < n ? p.alpha * __ldg(p.ls + c + e) : p.alpha;
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
    float m[8];
    if (p.pre.kind != K_NORM_NONE)
        affine8(p.pre, c, n, mean, rstd, v);
    if (p.scale.p) {
        unpack8(load8<VEC>(p.scale.p, p.scale.dt, at.scale + c, n), p.scale.dt, m);
#pragma unroll
        for (int e = 0; e < 8; e++)
            v[e] = fmaf(v[e], m[e], v[e]);
    }
    if (p.shift.p) {
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
    auto largest = [&](bool finite) {
        float r = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (e < n)
                r = finite ? larger_finite(r, v[e]) : larger(r, v[e]);
#pragma unroll
        for (int o = 8; o; o >>= 1)
            r = fmaxf(r, __shfl_xor_sync(0xffffffffu, r, o));
        return r;
    };
    float most = largest(false);
    const bool inf = __any_sync(0xffffffffu, infinite(most));
    if (inf)
        most = largest(true);
    const uint32_t byte = scale_byte(most);
    store8_e4m3<VEC>(p.Y.p, at.y + c, n, pack8_e4m3(v, scale_inverse(byte), inf));
    if ((threadIdx.x & 15) == 0 && n > 0)
        put_scale(p.S.p, p.S.dt, at.s + c / kScaleBlock, byte);
}

// Rows of any width: each sum and the result read the row again, and what stands in front of
// the second norm is computed for each. 4096 rows of 12288 bf16 with the vectors of a sample 478 us
// (61.5 us at the rate of a copy), with a norm of H too 830; 9001 columns 711 us.
template <int T, bool VEC>
__global__ void __launch_bounds__(T) norm_wide_kernel(const __grid_constant__ NormArgs a)
{
    __shared__ float smem[64];
    const k_norm_args &p = a.p;
    griddep_wait();
    griddep_launch();
    for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const long b = quot((uint32_t)row, a.dN), nn = row - b * p.N;
        const At at = {at_row(p.X, b, nn), at_row(p.H, b, nn), at_row(p.gate, b, nn), at_row(p.R, b, nn),
                       at_row(p.scale, b, nn), at_row(p.shift, b, nn), at_row(p.Y, b, nn), at_row(p.S, b, nn)};
        float hm = 0.0f, hs = 1.0f, mean = 0.0f, rstd = 1.0f;
        int turn = 0;
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
                m = row_sum<T>(s, smem, turn) * a.share;
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
            rs = rsqrtf(fmaf(row_sum<T>(q, smem, turn), a.share, k.eps));
        };
        if (p.H.p && p.post.kind != K_NORM_NONE)
            sums(p.post, false, hm, hs);
        if (p.Y.p && p.pre.kind != K_NORM_NONE)
            sums(p.pre, true, mean, rstd);
        __syncthreads();  // the next row starts with the first round again
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

// The device's CTAs share the rows evenly, in one wave.
template <int T, int V, bool VEC, int XT, int HT>
int launch_shared(NormArgs &a, cudaStream_t st)
{
    constexpr auto kern = norm_rows_kernel<T, V, VEC, XT, HT, true>;
    constexpr int threads = cta_threads(T), kRows = threads / T, smem = 4 * V * T * 8 * 4;
    if (smem > 48 * 1024) {
        const cudaError_t e = smem_limit_once<kern>(smem);
        if (e != cudaSuccess)
            return (int)e;
    }
    const long ctas = (long)device_sms() * ctas_of_sm<kern>(threads, smem);
    a.chunk = (a.rows + ctas - 1) / ctas;
    a.chunk = (a.chunk + kRows - 1) / kRows * kRows;
    const dim3 grid((unsigned)((a.rows + a.chunk - 1) / a.chunk));
    return launch_pdl(kern, grid, dim3(threads), smem, st, (const NormArgs)a);
}

// Rows an SM from which it pays that CTAs keep their sample's vectors in shared memory.
// Measured on 148 SMs, us with and without them, below and above the border (residual scale,
// gate, LayerNorm, shift and scale; fewer vectors move a border by up to a half either way):
//   aligned rows, bf16 to E4M3 (1024 columns by CTAs fp32)   not aligned, fp32
//     64: 15000 rows 8.4, 7.2     20000 8.5, 9.4              77: 20000 rows 15.6, 14.9   60000 36, 41
//    128:  5000      7.8, 6.7     10000 9.3, 9.6             500: 2500       13.0, 11.8   10000 26, 37
//    256: 10000     11.6, 11.0    20000 16.0, 18.6           601: 10000      41, 34       60000 130, 161
//    512:  5000     14.0, 12.2    15000 24, 32
//   1024: 30000     116, 115      60000 193, 227
//   2048: 30000     174, 161      60000 272, 316            2047: 10000      133, 101     60000 385, 456
//   4096: 10000     140, 119      20000 198, 225            3001: 5000       103, 91      10000 149, 165
//   8192: 10000     274, 253      15000 360, 377            5001: 1000       64, 45       5000 154, 192
// Rows that are not aligned with 16-bit X or H never (60000 x 77 bf16 66 and 50, 20000 x 2047 287
// and 202, 10000 x 7001 587 and 545). A sample needs rows too, two steps of the CTA's and
// at least 32 (20480 x 4096 bf16 in samples of 32 rows 217 and 252, of 16 255 and 253, of 2 949 and 277).
template <int T, int V, bool VEC>
__host__ __device__ constexpr int shared_rows()
{
    if (T <= 32)
        return VEC ? (T == 8 ? 128 : (T == 32 ? (V == 1 ? 80 : 48) : 64)) : (V == 1 ? 256 : 32);
    if (T == 128)
        return VEC ? (V == 1 ? 288 : 256) : (V == 1 ? 224 : 128);
    return VEC ? (T == 256 ? 112 : 84) : (T == 256 ? 48 : 14);
}

template <int T, int V, bool VEC>
int launch(NormArgs &a, cudaStream_t st)
{
    constexpr int kRows = cta_threads(T) / T;
    const int sms = device_sms(), xt = a.p.X.dt, ht = a.p.H.p ? a.p.H.dt : xt;
    if (a.rows >= (long)sms * shared_rows<T, V, VEC>() && a.p.N >= (kRows > 16 ? 2 * kRows : 32)) {
        if (xt == K_F32 && ht == K_F32)
            return launch_shared<T, V, VEC, K_F32, K_F32>(a, st);
        if constexpr (VEC) {
            if (xt == K_BF16)
                return launch_shared<T, V, VEC, K_BF16, K_BF16>(a, st);
            if (xt == K_F16)
                return launch_shared<T, V, VEC, K_F16, K_F16>(a, st);
            return launch_shared<T, V, VEC, K_F32, kAnyType>(a, st);
        }
    }
    const long need = (a.rows + kRows - 1) / kRows, most = (long)sms * 16;
    return launch_pdl(norm_rows_kernel<T, V, VEC, kAnyType, kAnyType, false>, dim3((unsigned)(need < most ? need : most)),
                      dim3(cta_threads(T)), 0, st, (const NormArgs)a);
}

template <int T, int V>
int launch(NormArgs &a, bool vec, cudaStream_t st)
{
    return vec ? launch<T, V, true>(a, st) : launch<T, V, false>(a, st);
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
    auto by_row = [&](const struct k_rows &r) { return r.p && r.ld != 0 && p->N > 1; };
    a.gaterow = by_row(p->gate);
    a.scalerow = by_row(p->scale);
    // (a sample's shift beside a scale of the rows' own is added behind that scale)
    a.shiftrow = by_row(p->shift) || (p->shift.p && a.scalerow);
    auto whole = [](const float *v) { return reinterpret_cast<uintptr_t>(v) % 16 == 0; };
    const bool vec = p->C % 8 == 0 && rows_vec8(p->X) && rows_vec8(p->H) && rows_vec8(p->gate) && rows_vec8(p->R) &&
                     rows_vec8(p->scale) && rows_vec8(p->shift) && rows_vec8(p->Y) && whole(p->ls) &&
                     whole(p->post.g) && whole(p->post.b) && whole(p->pre.g) && whole(p->pre.b);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(s);
    const int v = p->C / 8 + (p->C % 8 != 0);  // eights of a row
    // A warp to a row up to 512 columns (part of one for narrow rows), then a CTA;
    // up to 1024 a warp too where its values fit the registers twice over (16-bit
    // vectors) and there are rows enough to fill the device with warps.
    if (vec && v <= 8)
        return launch<8, 1, true>(a, st);
    if (vec && v <= 16)
        return launch<16, 1, true>(a, st);
    if (v <= 32)
        return launch<32, 1>(a, vec, st);
    if (v <= 64)
        return launch<32, 2>(a, vec, st);
    if (v <= 128) {
        const bool narrow = p->X.dt != K_F32;
        if (vec && narrow && a.rows >= (long)device_sms() * 64)
            return launch<32, 4, true>(a, st);
        return launch<128, 1>(a, vec, st);
    }
    if (v <= 256)
        return launch<128, 2>(a, vec, st);
    if (v <= 512)
        return launch<256, 2>(a, vec, st);
    if (v <= 1024)
        return launch<512, 2>(a, vec, st);
    const long most = (long)device_sms() * 2;
    const dim3 grid((unsigned)(a.rows < most ? a.rows : most));
    return vec ? launch_pdl(norm_wide_kernel<1024, true>, grid, dim3(1024), 0, st, (const NormArgs)a)
               : launch_pdl(norm_wide_kernel<1024, false>, grid, dim3(1024), 0, st, (const NormArgs)a);
}
