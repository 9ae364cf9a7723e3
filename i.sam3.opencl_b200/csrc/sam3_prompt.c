/* SPDX-License-Identifier: Unlicense */
/* Operators of the prompt-conditioned path (include/sam3_cuda.h): rotary
 * positions for rows of any layout, cross attention over an encoder's states
 * with their own lengths, group norm. Each checks its arguments in full, then
 * enqueues one kernel on the backend stream; none uses the scratch buffer, so
 * captured graphs and other calls share no memory with them. */
#include <math.h>
#include <string.h>

#include "backend_internal.h"

#define MAX_ROWS (1 << 30) /* rows of one sequence */

/* Elements an operand of counts n (strides st) and hd adjacent columns spans;
 * -1 when a stride is negative or the span passes 2^62. */
static int64_t span(const int64_t *n, const int64_t *st, int k, int64_t hd)
{
    __int128 s = hd;
    int i;

    for (i = 0; i < k; i++) {
        if (st[i] < 0)
            return -1;
        s += (__int128)(n[i] - 1) * st[i];
        if (s > ((__int128)1 << 62))
            return -1;
    }
    return (int64_t)s;
}

/* Whether no two of the operand's elements share an address. */
static int distinct(const int64_t *n, const int64_t *st, int k, int64_t hd)
{
    int64_t extent = hd;
    int done[3] = {0, 0, 0}, i, step;

    for (step = 0; step < k; step++) {
        int best = -1;

        for (i = 0; i < k; i++)
            if (!done[i] && (best < 0 || (n[i] > 1 ? st[i] : 0) < (n[best] > 1 ? st[best] : 0)))
                best = i;
        done[best] = 1;
        if (n[best] == 1)
            continue;
        if (st[best] < extent)
            return 0;
        extent += (n[best] - 1) * st[best];
    }
    return 1;
}

struct rows {
    struct k_rows k;
    const char *lo, *hi; /* bytes it spans */
};

static int float_dt(int dt)
{
    return dt == CB_F32 || dt == CB_BF16 || dt == CB_F16;
}

/* Checks [nb, rows, heads, hd] at o and fills r; CB_EARG / CB_EDTYPE. */
static int take(const struct cb_opnd *o, int64_t nb, int64_t rows, int64_t heads, int64_t hd,
                int output, struct rows *r)
{
    const int64_t n[3] = {nb, rows, heads}, st[3] = {o->s0, o->ld, o->s1};
    int64_t sp, es;

    if (!o->buf || !o->buf->ptr)
        return CB_EARG;
    if (!float_dt(o->buf->dtype))
        return CB_EDTYPE;
    es = (int64_t)cbi_dtype_size(o->buf->dtype);
    sp = span(n, st, 3, hd);
    if (sp < 0 || o->off < 0 || o->off > (INT64_C(1) << 62) ||
        (uint64_t)(o->off + sp) > (uint64_t)o->buf->bytes / (uint64_t)es ||
        ((uintptr_t)o->buf->ptr % (uintptr_t)es) || (output && !distinct(n, st, 3, hd)))
        return CB_EARG;
    r->k.p = (char *)o->buf->ptr + o->off * es;
    r->k.dt = o->buf->dtype;
    r->k.ld = o->ld;
    r->k.s0 = o->s0;
    r->k.s1 = o->s1;
    r->lo = (const char *)r->k.p;
    r->hi = r->lo + sp * es;
    return CB_OK;
}

static int overlap(const struct rows *a, const char *lo, const char *hi)
{
    return a->lo < hi && lo < a->hi;
}

/* Same type, address and layout (of the dimensions that have a second step). */
static int same_place(const struct rows *a, const struct rows *b, int64_t nb, int64_t n,
                      int64_t heads)
{
    return a->k.p == b->k.p && a->k.dt == b->k.dt && (nb == 1 || a->k.s0 == b->k.s0) &&
           (n == 1 || a->k.ld == b->k.ld) && (heads == 1 || a->k.s1 == b->k.s1);
}

/* A vector of n elements of type dt (4-byte types on a 4-byte boundary). */
static int vec_ok(cb_mem m, int dt, int64_t n)
{
    const uint64_t es = cbi_dtype_size(dt);

    return m && m->ptr && m->dtype == dt && n >= 0 && (uint64_t)n <= (uint64_t)m->bytes / es &&
           (uintptr_t)m->ptr % es == 0;
}

static int vec_overlap(const struct rows *a, cb_mem m, int64_t n)
{
    return m && overlap(a, (const char *)m->ptr,
                        (const char *)m->ptr + n * (int64_t)cbi_dtype_size(m->dtype));
}

int cb_rope_table(cb_backend *b, int npos, int rot, int64_t first,
                  const struct cb_rope_scaling *scaling, cb_mem cs)
{
    static const struct cb_rope_scaling plain = {10000.0, CB_ROPE_SCALE_NONE, 1.0, 0.0, 0.0, 0.0, 1.0};
    const struct cb_rope_scaling *sc = scaling ? scaling : &plain;
    const double two_pi = 6.283185307179586476925286766559;
    double turns[K_ROPE_MAX / 2], theta = sc->theta, lo = 0.0, hi = 0.0;
    int j;

    if (!b || npos <= 0 || rot <= 0 || rot % 2 || rot > K_ROPE_MAX ||
        first < -((int64_t)1 << 31) || first > ((int64_t)1 << 31) - npos ||
        !vec_ok(cs, CB_F32, (int64_t)npos * rot) || (uintptr_t)cs->ptr % 8 ||
        !(theta > 1.0) || !isfinite(theta) || !(sc->amplitude > 0.0) || !isfinite((float)sc->amplitude))
        return cbi_fail(b, CB_EARG, "rope_table");
    if (sc->kind != CB_ROPE_SCALE_NONE && (!(sc->factor >= 1.0) || !isfinite(sc->factor)))
        return cbi_fail(b, CB_EARG, "rope_table: factor");
    switch (sc->kind) {
    case CB_ROPE_SCALE_NONE:
    case CB_ROPE_SCALE_LINEAR:
        break;
    case CB_ROPE_SCALE_BASE:
        if (rot > 2)
            theta *= pow(sc->factor, rot / (rot - 2.0));
        break;
    case CB_ROPE_SCALE_RAMP:
        if (!(sc->orig_len > 0.0) || !isfinite(sc->orig_len) || !(sc->turns_slow > 0.0) ||
            !(sc->turns_fast > sc->turns_slow) || !isfinite(sc->turns_fast))
            return cbi_fail(b, CB_EARG, "rope_table: ramp");
        /* the pair that makes `turns` turns over orig_len positions */
        lo = floor(rot * log(sc->orig_len / (two_pi * sc->turns_fast)) / (2.0 * log(theta)));
        hi = ceil(rot * log(sc->orig_len / (two_pi * sc->turns_slow)) / (2.0 * log(theta)));
        lo = lo < 0.0 ? 0.0 : lo;
        hi = hi > rot - 1.0 ? rot - 1.0 : hi;
        break;
    default:
        return cbi_fail(b, CB_EARG, "rope_table: kind");
    }
    for (j = 0; j < rot / 2; j++) {
        double w = pow(theta, -2.0 * j / rot);

        if (sc->kind == CB_ROPE_SCALE_LINEAR)
            w /= sc->factor;
        else if (sc->kind == CB_ROPE_SCALE_RAMP) {
            const double d = hi - lo > 1e-3 ? hi - lo : 1e-3;
            double r = (j - lo) / d;

            r = r < 0.0 ? 0.0 : (r > 1.0 ? 1.0 : r);
            w = w * (1.0 - r) + w / sc->factor * r;
        }
        turns[j] = w / two_pi;
    }
    CB_TRY(cbi_enter(b));
    cbi_prof_begin(b, "rope_table", (double)npos * rot, 4.0 * npos * rot);
    j = cbi_kstatus(b,
                    k_rope_table(npos, rot, (long)first, turns, (float)sc->amplitude,
                                 (float *)cs->ptr, (k_stream)b->stream),
                    "rope_table");
    cbi_prof_end(b);
    return j;
}

int cb_rope_rotate(cb_backend *b, int nb, int N, int heads, int hd, int rot, int layout,
                   struct cb_opnd X, struct cb_opnd Y, cb_mem cs, int npos, cb_mem pos, int pos0)
{
    struct rows x, y;
    int rc;

    if (!b || nb <= 0 || N <= 0 || N > MAX_ROWS || (int64_t)nb * N > INT32_MAX || heads <= 0 ||
        hd <= 0 || hd > (1 << 16) || heads > (1 << 14) || rot <= 0 || rot % 2 || rot > hd ||
        npos <= 0 || (layout != CB_ROPE_PAIRS && layout != CB_ROPE_HALVES) ||
        !vec_ok(cs, CB_F32, (int64_t)npos * rot) || (uintptr_t)cs->ptr % 8)
        return cbi_fail(b, CB_EARG, "rope_rotate");
    if (pos ? (pos0 != 0 || !vec_ok(pos, CB_I32, (int64_t)nb * N))
            : (pos0 < 0 || (int64_t)pos0 + N > npos))
        return cbi_fail(b, CB_EARG, "rope_rotate: positions");
    if ((rc = take(&X, nb, N, heads, hd, 0, &x)) != CB_OK ||
        (rc = take(&Y, nb, N, heads, hd, 1, &y)) != CB_OK)
        return cbi_fail(b, rc, "rope_rotate: operand");
    if (y.k.dt != x.k.dt && x.k.dt != CB_F32)
        return cbi_fail(b, CB_EDTYPE, "rope_rotate: output type");
    if ((overlap(&y, x.lo, x.hi) && !same_place(&x, &y, nb, N, heads)) ||
        vec_overlap(&y, cs, (int64_t)npos * rot) || vec_overlap(&y, pos, (int64_t)nb * N))
        return cbi_fail(b, CB_EARG, "rope_rotate: output overlaps an input");
    CB_TRY(cbi_enter(b));
    cbi_prof_begin(b, "rope_rotate", 3.0 * nb * N * heads * rot,
                   (double)nb * N * heads * hd *
                       (cbi_dtype_size(x.k.dt) + cbi_dtype_size(y.k.dt)));
    rc = cbi_kstatus(b,
                     k_rope_rotate(&x.k, &y.k, nb, N, heads, hd, rot, layout,
                                   pos ? (const int *)pos->ptr : NULL, pos0, npos,
                                   (const float *)cs->ptr, (k_stream)b->stream),
                     "rope_rotate");
    cbi_prof_end(b);
    return rc;
}

int cb_cross_attend(cb_backend *b, int nb, int Nq, int Nk, int heads, int kvheads, int hd,
                    struct cb_opnd Q, struct cb_opnd K, struct cb_opnd V, struct cb_opnd O,
                    cb_mem klen, cb_mem kmask, float scale)
{
    struct rows q, k, v, o;
    int rc;

    if (!b || nb <= 0 || Nq <= 0 || Nq > MAX_ROWS || Nk <= 0 || Nk > MAX_ROWS || heads <= 0 ||
        kvheads <= 0 || heads % kvheads || hd <= 0 || hd > 128 || hd % 8 || !(scale > 0.0f) ||
        scale > 1e38f) /* its product with log2(e) is formed in 32 bits */
        return cbi_fail(b, CB_EARG, "cross_attend");
    if ((klen && !vec_ok(klen, CB_I32, nb)) || (kmask && !vec_ok(kmask, CB_U8, (int64_t)nb * Nk)))
        return cbi_fail(b, CB_EARG, "cross_attend: key lengths or mask");
    if ((rc = take(&Q, nb, Nq, heads, hd, 0, &q)) != CB_OK ||
        (rc = take(&K, nb, Nk, kvheads, hd, 0, &k)) != CB_OK ||
        (rc = take(&V, nb, Nk, kvheads, hd, 0, &v)) != CB_OK ||
        (rc = take(&O, nb, Nq, heads, hd, 1, &o)) != CB_OK)
        return cbi_fail(b, rc, "cross_attend: operand");
    if (k.k.dt != q.k.dt || v.k.dt != q.k.dt || o.k.dt != q.k.dt)
        return cbi_fail(b, CB_EDTYPE, "cross_attend: operands of different types");
    if (overlap(&o, q.lo, q.hi) || overlap(&o, k.lo, k.hi) || overlap(&o, v.lo, v.hi) ||
        vec_overlap(&o, klen, nb) || vec_overlap(&o, kmask, (int64_t)nb * Nk))
        return cbi_fail(b, CB_EARG, "cross_attend: output overlaps an input");
    CB_TRY(cbi_enter(b));
    cbi_prof_begin(b, "cross_attend", 4.0 * nb * heads * hd * (double)Nq * Nk,
                   (double)cbi_dtype_size(q.k.dt) * nb * hd *
                       (2.0 * Nq * heads + 2.0 * Nk * kvheads));
    rc = cbi_kstatus(b,
                     k_cross_attend(&q.k, &k.k, &v.k, &o.k, nb, Nq, Nk, heads, kvheads, hd,
                                    klen ? (const int *)klen->ptr : NULL,
                                    kmask ? (const unsigned char *)kmask->ptr : NULL, scale,
                                    b->d_err, (k_stream)b->stream),
                     "cross_attend");
    cbi_prof_end(b);
    return rc;
}

int cb_groupnorm(cb_backend *b, int nb, int64_t npix, int C, int groups, struct cb_opnd X,
                 struct cb_opnd Y, cb_mem g, cb_mem bias, float eps, int act)
{
    struct rows x, y;
    int rc;

    if (!b || nb <= 0 || npix <= 0 || npix > ((int64_t)1 << 40) || C <= 0 || groups <= 0 ||
        C % groups || !vec_ok(g, CB_F32, C) || !vec_ok(bias, CB_F32, C) || !(eps >= 0.0f) ||
        !isfinite(eps) || (act != CB_ACT_NONE && act != CB_ACT_GELU && act != CB_ACT_RELU))
        return cbi_fail(b, CB_EARG, "groupnorm");
    if (X.s1 != 0 || Y.s1 != 0) /* channels are adjacent */
        return cbi_fail(b, CB_EARG, "groupnorm: channel stride");
    if ((rc = take(&X, nb, npix, 1, C, 0, &x)) != CB_OK ||
        (rc = take(&Y, nb, npix, 1, C, 1, &y)) != CB_OK)
        return cbi_fail(b, rc, "groupnorm: operand");
    if (y.k.dt != x.k.dt && x.k.dt != CB_F32)
        return cbi_fail(b, CB_EDTYPE, "groupnorm: output type");
    if ((overlap(&y, x.lo, x.hi) && !same_place(&x, &y, nb, npix, 1)) || vec_overlap(&y, g, C) ||
        vec_overlap(&y, bias, C))
        return cbi_fail(b, CB_EARG, "groupnorm: output overlaps an input");
    CB_TRY(cbi_enter(b));
    cbi_prof_begin(b, "groupnorm", 8.0 * nb * (double)npix * C,
                   (double)nb * npix * C * (cbi_dtype_size(x.k.dt) + cbi_dtype_size(y.k.dt)));
    rc = cbi_kstatus(b,
                     k_groupnorm(x.k.p, x.k.dt, x.k.ld, x.k.s0, y.k.p, y.k.dt, y.k.ld, y.k.s0,
                                 (const float *)g->ptr, (const float *)bias->ptr, nb, (long)npix,
                                 C, groups, eps, act, (k_stream)b->stream),
                     "groupnorm");
    cbi_prof_end(b);
    return rc;
}
