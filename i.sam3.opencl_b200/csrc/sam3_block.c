/* SPDX-License-Identifier: Unlicense */
/* Operators around attention in a transformer block (include/sam3_cuda.h):
 * E4M3 quantisation, products of E4M3 operands with block scales, norms around
 * the residual stream. Each checks its arguments in full, then enqueues its
 * kernel on the backend stream; none uses the scratch buffer. */
#include <math.h>
#include <string.h>

#include "operand.h"

#define BLOCK 128
#define T_SCALE (T_(CB_F32) | T_(CB_E8M0))

static int blocks(int n)
{
    return n / BLOCK + (n % BLOCK != 0);
}

int cb_quantize_e4m3(cb_backend *b, int nb, int N, int K, int brows, struct cb_opnd X,
                     struct cb_opnd Q, struct cb_opnd S)
{
    struct rows x, q, s;
    int rc;

    if (!b || nb <= 0 || N <= 0 || N > MAX_ROWS || K <= 0 || K > MAX_ROWS || (int64_t)nb * N > INT32_MAX ||
        (brows != 1 && brows != BLOCK) || X.s1 || Q.s1 || S.s1)
        return cbi_fail(b, CB_EARG, "quantize_e4m3");
    if ((rc = take(&X, nb, N, 1, K, T_FLOAT, 0, &x)) != CB_OK ||
        (rc = take(&Q, nb, N, 1, K, T_(CB_E4M3), 1, &q)) != CB_OK ||
        (rc = take(&S, nb, brows == 1 ? N : blocks(N), 1, blocks(K), T_SCALE, 1, &s)) != CB_OK)
        return cbi_fail(b, rc, "quantize_e4m3: operand");
    if (overlap(&q, x.lo, x.hi) || overlap(&s, x.lo, x.hi) || overlap(&q, s.lo, s.hi))
        return cbi_fail(b, CB_EARG, "quantize_e4m3: an output overlaps");
    CB_TRY(cbi_enter(b));
    cbi_prof_begin(b, "quantize_e4m3", 2.0 * nb * N * K,
                   (double)nb * N * K * (cbi_dtype_size(x.k.dt) + 1.0));
    rc = cbi_kstatus(b, k_quantize_e4m3(&x.k, &q.k, &s.k, nb, N, K, brows, (k_stream)b->stream),
                     "quantize_e4m3");
    cbi_prof_end(b);
    return rc;
}

int cb_gemm_e4m3(cb_backend *b, int M, int N, int K, struct cb_opnd A, struct cb_opnd SA,
                 struct cb_opnd B, struct cb_opnd SB, struct cb_opnd C, const struct cb_opnd *SC,
                 cb_mem bias, int act)
{
    struct rows a, sa, w, sb, c, sc;
    const int kb = K > 0 ? blocks(K) : 0;
    int rc;

    if (!b || M <= 0 || M > MAX_ROWS || N <= 0 || N > MAX_ROWS || K <= 0 || K > MAX_ROWS || A.s1 || SA.s1 || B.s1 ||
        SB.s1 || C.s1 || (SC && SC->s1) ||
        (act != CB_ACT_NONE && act != CB_ACT_GELU && act != CB_ACT_RELU) ||
        (bias && !vec_ok(bias, CB_F32, N)))
        return cbi_fail(b, CB_EARG, "gemm_e4m3");
    memset(&sc, 0, sizeof(sc));
    if ((rc = take(&A, 1, M, 1, K, T_(CB_E4M3), 0, &a)) != CB_OK ||
        (rc = take(&B, 1, N, 1, K, T_(CB_E4M3), 0, &w)) != CB_OK ||
        (rc = take(&SA, 1, M, 1, kb, T_SCALE, 0, &sa)) != CB_OK ||
        (rc = take(&SB, 1, blocks(N), 1, kb, T_SCALE, 0, &sb)) != CB_OK ||
        (rc = take(&C, 1, M, 1, N, T_FLOAT | T_(CB_E4M3), 1, &c)) != CB_OK ||
        (SC && (rc = take(SC, 1, M, 1, blocks(N), T_SCALE, 1, &sc)) != CB_OK))
        return cbi_fail(b, rc, "gemm_e4m3: operand");
    if ((c.k.dt == CB_E4M3) != (SC != NULL))
        return cbi_fail(b, CB_EARG, "gemm_e4m3: scales of the result");
    if ((uintptr_t)a.k.p % 16 || (uintptr_t)w.k.p % 16 || (M > 1 && (a.k.ld % 16 || a.k.ld < K)) ||
        (N > 1 && (w.k.ld % 16 || w.k.ld < K)))
        return cbi_fail(b, CB_EARG, "gemm_e4m3: rows of A and B start at multiples of 16 bytes");
    if (overlap(&c, a.lo, a.hi) || overlap(&c, w.lo, w.hi) || overlap(&c, sa.lo, sa.hi) ||
        overlap(&c, sb.lo, sb.hi) || vec_overlap(&c, bias, N) ||
        (SC && (overlap(&c, sc.lo, sc.hi) || overlap(&sc, a.lo, a.hi) || overlap(&sc, w.lo, w.hi) ||
                overlap(&sc, sa.lo, sa.hi) || overlap(&sc, sb.lo, sb.hi) || vec_overlap(&sc, bias, N))))
        return cbi_fail(b, CB_EARG, "gemm_e4m3: an output overlaps");
    CB_TRY(cbi_enter(b));
    cbi_prof_begin(b, "gemm_e4m3", 2.0 * M * N * K,
                   (double)M * K + (double)N * K + (double)M * N * cbi_dtype_size(c.k.dt));
    rc = cbi_kstatus(b,
                     k_gemm_e4m3(M, N, K, &a.k, &sa.k, &w.k, &sb.k, &c.k, SC ? &sc.k : NULL,
                                 bias ? (const float *)bias->ptr : NULL, act, b->d_err,
                                 (k_stream)b->stream),
                     "gemm_e4m3");
    cbi_prof_end(b);
    return rc;
}

/* Norm n of C channels, kind none when n is NULL; CB_EARG. */
static int take_norm(const struct cb_norm *n, int C, struct k_norm *k)
{
    memset(k, 0, sizeof(*k));
    if (!n || n->kind == CB_NORM_NONE)
        return n && (n->g || n->bias) ? CB_EARG : CB_OK;
    if ((n->kind != CB_NORM_LAYER && n->kind != CB_NORM_RMS) || !(n->eps >= 0.0f) || !isfinite(n->eps) ||
        (n->g && !vec_ok(n->g, CB_F32, C)) || (n->bias && !vec_ok(n->bias, CB_F32, C)))
        return CB_EARG;
    k->kind = n->kind;
    k->eps = n->eps;
    k->g = n->g ? (const float *)n->g->ptr : NULL;
    k->b = n->bias ? (const float *)n->bias->ptr : NULL;
    return CB_OK;
}

int cb_norm_residual(cb_backend *b, int nb, int N, int C, struct cb_opnd X, const struct cb_opnd *H,
                     const struct cb_norm *post, float alpha, cb_mem ls, const struct cb_opnd *gate,
                     const struct cb_opnd *R, const struct cb_norm *pre, const struct cb_opnd *scale,
                     const struct cb_opnd *shift, const struct cb_opnd *Y, const struct cb_opnd *S)
{
    const struct cb_opnd *in[5], *out[3];
    struct rows x, ri[5], ro[3];
    struct k_norm_args k;
    const struct cb_norm *norms[2] = {post, pre};
    unsigned ty;
    int rc, i, j;

    in[0] = H, in[1] = gate, in[2] = scale, in[3] = shift, in[4] = &X;
    out[0] = R, out[1] = Y, out[2] = S;
    memset(&k, 0, sizeof(k));
    memset(ri, 0, sizeof(ri));
    memset(ro, 0, sizeof(ro));
    if (!b || nb <= 0 || N <= 0 || N > MAX_ROWS || C <= 0 || C > MAX_ROWS || (int64_t)nb * N > INT32_MAX ||
        !isfinite(alpha) || (ls && !vec_ok(ls, CB_F32, C)) || (!R && !Y) ||
        (!H && (gate || ls || (post && post->kind != CB_NORM_NONE) || alpha != 1.0f)) ||
        (!Y && ((pre && pre->kind != CB_NORM_NONE) || scale || shift || S)))
        return cbi_fail(b, CB_EARG, "norm_residual");
    if (take_norm(post, C, &k.post) != CB_OK || take_norm(pre, C, &k.pre) != CB_OK)
        return cbi_fail(b, CB_EARG, "norm_residual: norm");
    for (i = 0; i < 5; i++)
        if (in[i] && in[i]->s1)
            return cbi_fail(b, CB_EARG, "norm_residual: channel stride");
    for (i = 0; i < 3; i++)
        if (out[i] && out[i]->s1)
            return cbi_fail(b, CB_EARG, "norm_residual: channel stride");
    for (i = 4; i >= 0; i--) /* X first */
        if (in[i] && (rc = take(in[i], nb, N, 1, C, T_FLOAT, 0, &ri[i])) != CB_OK)
            return cbi_fail(b, rc, "norm_residual: operand");
    x = ri[4];
    ty = T_(x.k.dt) | T_(CB_E4M3) | (x.k.dt == CB_F32 ? T_FLOAT : 0);
    if ((R && (rc = take(R, nb, N, 1, C, T_(x.k.dt), 1, &ro[0])) != CB_OK) ||
        (Y && (rc = take(Y, nb, N, 1, C, ty, 1, &ro[1])) != CB_OK) ||
        (S && (rc = take(S, nb, N, 1, blocks(C), T_SCALE, 1, &ro[2])) != CB_OK))
        return cbi_fail(b, rc, "norm_residual: output");
    if (H && ri[0].k.dt != x.k.dt && x.k.dt != CB_F32)
        return cbi_fail(b, CB_EDTYPE, "norm_residual: the block's output");
    if ((Y && ro[1].k.dt == CB_E4M3) != (S != NULL))
        return cbi_fail(b, CB_EARG, "norm_residual: scales of the result");
    for (i = 0; i < 3; i++) {
        if (!out[i])
            continue;
        for (j = 0; j < 5; j++)
            if (in[j] && overlap(&ro[i], ri[j].lo, ri[j].hi) &&
                (i == 2 || (j != 0 && j != 4) || !same_place(&ri[j], &ro[i], nb, N, 1)))
                return cbi_fail(b, CB_EARG, "norm_residual: an output overlaps an input");
        for (j = 0; j < i; j++)
            if (out[j] && overlap(&ro[i], ro[j].lo, ro[j].hi))
                return cbi_fail(b, CB_EARG, "norm_residual: outputs overlap");
        if (vec_overlap(&ro[i], ls, C))
            return cbi_fail(b, CB_EARG, "norm_residual: an output overlaps an input");
        for (j = 0; j < 2; j++)
            if (norms[j] && norms[j]->kind != CB_NORM_NONE &&
                (vec_overlap(&ro[i], norms[j]->g, C) || vec_overlap(&ro[i], norms[j]->bias, C)))
                return cbi_fail(b, CB_EARG, "norm_residual: an output overlaps an input");
    }
    k.nb = nb;
    k.N = N;
    k.C = C;
    k.X = x.k;
    k.H = ri[0].k;
    k.gate = ri[1].k;
    k.scale = ri[2].k;
    k.shift = ri[3].k;
    k.R = ro[0].k;
    k.Y = ro[1].k;
    k.S = ro[2].k;
    k.alpha = alpha;
    k.ls = ls ? (const float *)ls->ptr : NULL;
    CB_TRY(cbi_enter(b));
    cbi_prof_begin(b, "norm_residual", 12.0 * nb * N * C,
                   (double)nb * N * C *
                       ((double)cbi_dtype_size(x.k.dt) * (R ? 2 : 1) +
                        (H ? cbi_dtype_size(ri[0].k.dt) : 0) + (Y ? cbi_dtype_size(ro[1].k.dt) : 0)));
    rc = cbi_kstatus(b, k_norm_residual(&k, (k_stream)b->stream), "norm_residual");
    cbi_prof_end(b);
    return rc;
}
