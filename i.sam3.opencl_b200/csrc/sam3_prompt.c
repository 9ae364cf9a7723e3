/* SPDX-License-Identifier: Unlicense */
/* Operators of the prompt-conditioned path (include/sam3_cuda.h): rotary
 * positions for rows of any layout, cross attention over an encoder's states
 * with their own lengths, group norm. Each checks its arguments in full, then
 * enqueues one kernel on the backend stream; none uses the scratch buffer, so
 * captured graphs and other calls share no memory with them. */
#include <math.h>

#include "operand.h"

/* Turns per position of the pairs of a ladder of rot columns; CB_EARG. */
static int rope_turns(cb_backend *b, int rot, const struct cb_rope_scaling *sc, double *turns)
{
    const double two_pi = 6.283185307179586476925286766559;
    double theta = sc->theta, lo = 0.0, hi = 0.0;
    int j;

    if (!(theta > 1.0) || !isfinite(theta) || !(sc->amplitude > 0.0) || !isfinite((float)sc->amplitude))
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
    return CB_OK;
}

static const struct cb_rope_scaling plain_rope = {10000.0, CB_ROPE_SCALE_NONE, 1.0, 0.0, 0.0, 0.0, 1.0};

static int table_ok(int npos, int rot, int64_t first, cb_mem cs)
{
    return npos > 0 && rot > 0 && rot % 2 == 0 && rot <= K_ROPE_MAX && first >= -((int64_t)1 << 31) &&
           first <= ((int64_t)1 << 31) - npos && vec_ok(cs, CB_F32, (int64_t)npos * rot) &&
           (uintptr_t)cs->ptr % 8 == 0;
}

static int enqueue_table(cb_backend *b, int npos, int rot, int64_t first, const double *turns,
                         double amplitude, cb_mem cs)
{
    int rc;

    CB_TRY(cbi_enter(b));
    cbi_prof_begin(b, "rope_table", (double)npos * rot, 4.0 * npos * rot);
    rc = cbi_kstatus(b,
                     k_rope_table(npos, rot, (long)first, turns, (float)amplitude, (float *)cs->ptr,
                                  (k_stream)b->stream),
                     "rope_table");
    cbi_prof_end(b);
    return rc;
}

int cb_rope_table(cb_backend *b, int npos, int rot, int64_t first,
                  const struct cb_rope_scaling *scaling, cb_mem cs)
{
    const struct cb_rope_scaling *sc = scaling ? scaling : &plain_rope;
    double turns[K_ROPE_MAX / 2];

    if (!b || !table_ok(npos, rot, first, cs))
        return cbi_fail(b, CB_EARG, "rope_table");
    CB_TRY(rope_turns(b, rot, sc, turns));
    return enqueue_table(b, npos, rot, first, turns, sc->amplitude, cs);
}

/* The axis of each pair of the head; the pairs of all axes, 0 when the
 * description is not valid (widths even and positive, with turns no axis
 * behind the first wider than its places). */
static int axes_pairs(const struct cb_rope_axes *ax, uint8_t *axis)
{
    int pairs = 0, count[K_ROPE_AXES] = {0, 0, 0, 0}, a, i, j;

    if (!ax || ax->axes < 1 || ax->axes > K_ROPE_AXES ||
        (ax->order != CB_ROPE_AXES_SECTIONS && ax->order != CB_ROPE_AXES_TURNS))
        return 0;
    for (a = 0; a < ax->axes; a++) {
        if (ax->width[a] <= 0 || ax->width[a] % 2 || ax->width[a] > K_ROPE_MAX)
            return 0;
        pairs += ax->width[a] / 2;
    }
    if (pairs > K_ROPE_MAX / 2)
        return 0;
    if (ax->order == CB_ROPE_AXES_SECTIONS) {
        for (a = 0, j = 0; a < ax->axes; a++)
            for (i = 0; i < ax->width[a] / 2; i++)
                axis[j++] = (uint8_t)a;
        return pairs;
    }
    for (j = 0; j < pairs; j++) {
        a = j % ax->axes;
        axis[j] = (uint8_t)(j / ax->axes < ax->width[a] / 2 ? a : 0);
        count[axis[j]]++;
    }
    for (a = 0; a < ax->axes; a++)
        if (count[a] != ax->width[a] / 2)
            return 0;
    return pairs;
}

int cb_rope_axes_table(cb_backend *b, int npos, const struct cb_rope_axes *axes, int64_t first,
                       const struct cb_rope_scaling *scaling, cb_mem cs)
{
    const struct cb_rope_scaling *sc = scaling ? scaling : &plain_rope;
    double turns[K_ROPE_MAX / 2], own[K_ROPE_AXES][K_ROPE_MAX / 2];
    uint8_t axis[K_ROPE_MAX / 2];
    int at[K_ROPE_AXES] = {0, 0, 0, 0}, pairs, a, j;

    if (!b || (pairs = axes_pairs(axes, axis)) == 0 || !table_ok(npos, 2 * pairs, first, cs))
        return cbi_fail(b, CB_EARG, "rope_axes_table");
    for (a = 0; a < axes->axes; a++)
        CB_TRY(rope_turns(b, axes->width[a], sc, own[a]));
    for (j = 0; j < pairs; j++)
        turns[j] = own[axis[j]][at[axis[j]]++];
    return enqueue_table(b, npos, 2 * pairs, first, turns, sc->amplitude, cs);
}

/* The part of the rotations that does not depend on where positions come
 * from: operands, then the kernel. ax NULL: one axis. */
static int rotate(cb_backend *b, int nb, int N, int heads, int hd, int rot, int layout,
                  const struct cb_opnd *X, const struct cb_opnd *Y, cb_mem cs, int npos, cb_mem pos,
                  int pos0, const struct k_rope_axes *ax, const char *what)
{
    struct rows x, y;
    const int64_t npid = (int64_t)nb * N * (ax ? ax->axes : 1);
    int rc;

    if ((rc = take(X, nb, N, heads, hd, T_FLOAT, 0, &x)) != CB_OK ||
        (rc = take(Y, nb, N, heads, hd, T_FLOAT, 1, &y)) != CB_OK)
        return cbi_fail(b, rc, "rope_rotate: operand");
    if (y.k.dt != x.k.dt && x.k.dt != CB_F32)
        return cbi_fail(b, CB_EDTYPE, "rope_rotate: output type");
    if ((overlap(&y, x.lo, x.hi) && !same_place(&x, &y, nb, N, heads)) ||
        vec_overlap(&y, cs, (int64_t)npos * rot) || vec_overlap(&y, pos, npid))
        return cbi_fail(b, CB_EARG, "rope_rotate: output overlaps an input");
    CB_TRY(cbi_enter(b));
    cbi_prof_begin(b, what, 3.0 * nb * N * heads * rot,
                   (double)nb * N * heads * hd *
                       (cbi_dtype_size(x.k.dt) + cbi_dtype_size(y.k.dt)));
    rc = cbi_kstatus(b,
                     k_rope_rotate(&x.k, &y.k, nb, N, heads, hd, rot, layout,
                                   pos ? (const int *)pos->ptr : NULL, pos0, npos,
                                   (const float *)cs->ptr, ax, (k_stream)b->stream),
                     what);
    cbi_prof_end(b);
    return rc;
}

static int rotate_shape_ok(int nb, int N, int heads, int hd, int rot, int layout, cb_mem cs, int npos)
{
    return nb > 0 && N > 0 && N <= MAX_ROWS && (int64_t)nb * N <= INT32_MAX && heads > 0 && hd > 0 &&
           hd <= (1 << 16) && heads <= (1 << 14) && rot > 0 && rot % 2 == 0 && rot <= hd && npos > 0 &&
           (layout == CB_ROPE_PAIRS || layout == CB_ROPE_HALVES) &&
           vec_ok(cs, CB_F32, (int64_t)npos * rot) && (uintptr_t)cs->ptr % 8 == 0;
}

int cb_rope_rotate(cb_backend *b, int nb, int N, int heads, int hd, int rot, int layout,
                   struct cb_opnd X, struct cb_opnd Y, cb_mem cs, int npos, cb_mem pos, int pos0)
{
    if (!b || !rotate_shape_ok(nb, N, heads, hd, rot, layout, cs, npos))
        return cbi_fail(b, CB_EARG, "rope_rotate");
    if (pos ? (pos0 != 0 || !vec_ok(pos, CB_I32, (int64_t)nb * N))
            : (pos0 < 0 || (int64_t)pos0 + N > npos))
        return cbi_fail(b, CB_EARG, "rope_rotate: positions");
    return rotate(b, nb, N, heads, hd, rot, layout, &X, &Y, cs, npos, pos, pos0, NULL, "rope_rotate");
}

int cb_rope_rotate_axes(cb_backend *b, int nb, int N, int heads, int hd, int rot, int layout,
                        const struct cb_rope_axes *axes, struct cb_opnd X, struct cb_opnd Y,
                        cb_mem cs, int npos, cb_mem pos, const int *grid)
{
    struct k_rope_axes ax = {0};
    int a;

    if (!b || !rotate_shape_ok(nb, N, heads, hd, rot, layout, cs, npos) || rot > K_ROPE_MAX ||
        axes_pairs(axes, ax.axis) * 2 != rot)
        return cbi_fail(b, CB_EARG, "rope_rotate_axes");
    ax.axes = axes->axes;
    ax.sections = axes->order == CB_ROPE_AXES_SECTIONS;
    if (pos ? (grid || !vec_ok(pos, CB_I32, (int64_t)nb * N * ax.axes)) : !grid)
        return cbi_fail(b, CB_EARG, "rope_rotate_axes: positions");
    if (grid) {
        int64_t cells = 1;

        for (a = 0; a < ax.axes; a++) {
            if (grid[a] <= 0 || (cells *= grid[a]) > INT32_MAX)
                return cbi_fail(b, CB_EARG, "rope_rotate_axes: grid");
            ax.grid[a] = grid[a];
        }
        if (N > cells)
            return cbi_fail(b, CB_EARG, "rope_rotate_axes: grid");
    }
    return rotate(b, nb, N, heads, hd, rot, layout, &X, &Y, cs, npos, pos, 0, &ax, "rope_rotate_axes");
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
    if ((rc = take(&Q, nb, Nq, heads, hd, T_FLOAT, 0, &q)) != CB_OK ||
        (rc = take(&K, nb, Nk, kvheads, hd, T_FLOAT, 0, &k)) != CB_OK ||
        (rc = take(&V, nb, Nk, kvheads, hd, T_FLOAT, 0, &v)) != CB_OK ||
        (rc = take(&O, nb, Nq, heads, hd, T_FLOAT, 1, &o)) != CB_OK)
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
    if ((rc = take(&X, nb, npix, 1, C, T_FLOAT, 0, &x)) != CB_OK ||
        (rc = take(&Y, nb, npix, 1, C, T_FLOAT, 1, &y)) != CB_OK)
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
