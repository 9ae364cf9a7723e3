/* SPDX-License-Identifier: Unlicense */
/* Checks of the strided operands (cb_bmat) of the prompt-path and block
 * operators. */
#ifndef SAM3_OPERAND_H
#define SAM3_OPERAND_H

#include "backend_internal.h"

#define MAX_ROWS (1 << 30) /* rows of one sequence */

/* Elements an operand of counts n (strides st) and hd adjacent columns spans;
 * -1 when a stride is negative or the span passes 2^62. */
static inline int64_t span(const int64_t *n, const int64_t *st, int k, int64_t hd)
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
static inline int distinct(const int64_t *n, const int64_t *st, int k, int64_t hd)
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

/* Sets of element types. */
#define T_(dt) (1u << (dt))
#define T_FLOAT (T_(CB_F32) | T_(CB_BF16) | T_(CB_F16))

/* Checks [nb, rows, heads, hd] of one of the types at o and fills r; CB_EARG /
 * CB_EDTYPE. */
static inline int take(const struct cb_opnd *o, int64_t nb, int64_t rows, int64_t heads, int64_t hd,
                       unsigned types, int output, struct rows *r)
{
    const int64_t n[3] = {nb, rows, heads}, st[3] = {o->s0, o->ld, o->s1};
    int64_t sp, es;

    if (!o->buf || !o->buf->ptr)
        return CB_EARG;
    if (!(types & T_(o->buf->dtype)))
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

static inline int overlap(const struct rows *a, const char *lo, const char *hi)
{
    return a->lo < hi && lo < a->hi;
}

/* Same type, address and layout (of the dimensions that have a second step). */
static inline int same_place(const struct rows *a, const struct rows *b, int64_t nb, int64_t n,
                      int64_t heads)
{
    return a->k.p == b->k.p && a->k.dt == b->k.dt && (nb == 1 || a->k.s0 == b->k.s0) &&
           (n == 1 || a->k.ld == b->k.ld) && (heads == 1 || a->k.s1 == b->k.s1);
}

/* A vector of n elements of type dt (4-byte types on a 4-byte boundary). */
static inline int vec_ok(cb_mem m, int dt, int64_t n)
{
    const uint64_t es = cbi_dtype_size(dt);

    return m && m->ptr && m->dtype == dt && n >= 0 && (uint64_t)n <= (uint64_t)m->bytes / es &&
           (uintptr_t)m->ptr % es == 0;
}

static inline int vec_overlap(const struct rows *a, cb_mem m, int64_t n)
{
    return m && overlap(a, (const char *)m->ptr,
                        (const char *)m->ptr + n * (int64_t)cbi_dtype_size(m->dtype));
}

#endif
