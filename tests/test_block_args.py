"""Refusals of the operators around attention in a block (cb_quantize_e4m3,
cb_gemm_e4m3, cb_norm_residual, cb_rope_axes_table, cb_rope_rotate_axes), checked
without a device: arguments are validated before anything touches CUDA, so a
zeroed handle stands in for the backend, wrapped addresses for its buffers. Each
case changes one argument of a call that passes validation (which then fails for
want of a device)."""
import ctypes as C

import pytest

CB_EARG, CB_ECUDA, CB_EDTYPE = 3, 4, 6


@pytest.fixture(scope="module")
def fake(sb):
    torch = pytest.importorskip("torch")
    if torch.cuda.is_available():
        pytest.skip("stand-in addresses must never reach a device")
    buf = C.create_string_buffer(1 << 16)
    be = sb.Backend.__new__(sb.Backend)
    be.h = C.c_void_p(C.addressof(buf))
    be._buf = buf
    yield be
    be.h = C.c_void_p(None)


def size(sb, dt):
    return {sb.F32: 4, sb.I32: 4, sb.BF16: 2, sb.F16: 2}.get(dt, 1)


def mem(sb, be, addr, n, dt):
    """n elements of type dt at addr."""
    m = C.c_void_p()
    assert sb.lib().cb_wrap(be.h, C.c_void_p(addr), n * size(sb, dt), dt, C.byref(m)) == 0
    return sb.Mem(be, m.value)


def status(fn, *a, **k):
    import sys
    try:
        fn(*a, **k)
    except sys.modules["sam3_b200"].CBError as e:
        return e.status
    return 0


A, B, D, E, F, G, H, I, J, K_ = (i << 32 for i in range(1, 11))


def test_element_types(sb, fake):
    for dt in (sb.E4M3, sb.E8M0):
        m = mem(sb, fake, A, 5, dt)
        assert m.nbytes == 5 and m.dtype == dt
    bad = C.c_void_p()
    assert sb.lib().cb_wrap(fake.h, C.c_void_p(A), 4, 7, C.byref(bad)) == CB_EARG


def test_quantize_refusals(sb, fake):
    def call(nb=2, N=5, K=200, brows=1, dx=sb.BF16, dq=sb.E4M3, ds=sb.E8M0, x=A, q=B, s=D, xs=(200, 1000, 0), qs=(208, 1040, 0),
             ss=(2, 10, 0), nx=2000, nq=2072, ns=20, off=0):
        def op(p, n, d, st, o=0):
            return sb.Backend.bmat(mem(sb, fake, p, n, d), o, *st)
        return status(fake.quantize_e4m3, nb, N, K, brows, op(x, nx, dx, xs, off), op(q, nq, dq, qs), op(s, ns, ds, ss))
    assert call() == CB_ECUDA and call(ds=sb.F32) == CB_ECUDA and call(dx=sb.F32) == CB_ECUDA and call(dx=sb.F16) == CB_ECUDA
    assert call(brows=128, ns=4, ss=(2, 2, 0)) == CB_ECUDA and call(xs=(0, 0, 0)) == CB_ECUDA
    for bad in (dict(nb=0), dict(N=0), dict(K=0), dict(brows=0), dict(brows=64), dict(brows=2), dict(xs=(200, 1000, 1)),
                dict(qs=(208, 1040, 8)), dict(ss=(2, 10, 1)), dict(nx=1999), dict(nq=2071), dict(ns=19), dict(off=1), dict(off=-1),
                dict(qs=(199, 1040, 0)), dict(qs=(208, 0, 0)), dict(ss=(1, 10, 0)), dict(ss=(0, 0, 0)), dict(x=0), dict(q=0), dict(s=0),
                dict(x=A + 1), dict(q=A), dict(s=A + 16), dict(q=D), dict(N=(1 << 30) + 1), dict(K=(1 << 30) + 1), dict(xs=(-200, 1000, 0)),
                dict(s=D + 2, ds=sb.F32)):
        assert call(**bad) == CB_EARG, bad
    for bad in (dict(dx=sb.E4M3), dict(dx=sb.I32), dict(dq=sb.U8), dict(dq=sb.BF16), dict(ds=sb.U8), dict(ds=sb.BF16)):
        assert call(**bad) == CB_EDTYPE, bad


def test_gemm_refusals(sb, fake):
    def call(M=5, N=130, K=200, da=sb.E4M3, db=sb.E4M3, dsa=sb.E8M0, dsb=sb.F32, dc=sb.BF16, dsc=None, a=A, w=B, sa=D, sbp=E, c=F, sc=G,
             bias=None, nbias=130, bdt=sb.F32, lda=208, ldb=208, ldsa=2, ldsb=2, ldc=130, ldsc=2, na=1032, nw=27032, nsa=10, nsb=4, nc=650,
             nsc=10, act=0, aoff=0, boff=0, s0=0, s1=0, cs0=0):
        def op(p, n, d, ld, o=0, s0=0, s1=0):
            return sb.Backend.bmat(mem(sb, fake, p, n, d), o, ld, s0, s1)
        SC = None if dsc is None else op(sc, nsc, dsc, ldsc)
        bb = None if bias is None else mem(sb, fake, bias, nbias, bdt)
        return status(fake.gemm_e4m3, M, N, K, op(a, na, da, lda, aoff, s0, s1), op(sa, nsa, dsa, ldsa), op(w, nw, db, ldb, boff),
                      op(sbp, nsb, dsb, ldsb), op(c, nc, dc, ldc, 0, cs0), SC, bb, act)
    assert call() == CB_ECUDA and call(dsa=sb.F32, dsb=sb.E8M0) == CB_ECUDA and call(bias=H) == CB_ECUDA and call(act=2) == CB_ECUDA
    assert call(dc=sb.E4M3, dsc=sb.E8M0) == CB_ECUDA and call(dc=sb.E4M3, dsc=sb.F32) == CB_ECUDA and call(dc=sb.F32) == CB_ECUDA
    assert call(s0=16, cs0=650) == CB_ECUDA
    assert call(dc=sb.F16, ldc=131, nc=654) == CB_ECUDA and call(M=1, lda=7) == CB_ECUDA  # one row's pitch is of no account
    for bad in (dict(M=0), dict(N=0), dict(K=0), dict(act=3), dict(act=-1), dict(s1=16), dict(lda=200), dict(lda=192),
                dict(ldb=207), dict(ldb=0), dict(lda=0), dict(a=A + 8), dict(w=B + 1), dict(aoff=8), dict(boff=4), dict(na=1031), dict(nw=27031),
                dict(nsa=9), dict(nsb=3), dict(nc=649), dict(ldc=129), dict(dc=sb.E4M3), dict(dsc=sb.E8M0), dict(dc=sb.E4M3, dsc=sb.E8M0, nsc=9),
                dict(dc=sb.E4M3, dsc=sb.E8M0, ldsc=1), dict(bias=H, nbias=129), dict(bias=H, bdt=sb.BF16), dict(bias=H + 2), dict(bias=F),
                dict(c=A), dict(c=B + 64), dict(c=D), dict(c=E), dict(dc=sb.E4M3, dsc=sb.E8M0, sc=F + 5), dict(dc=sb.E4M3, dsc=sb.E8M0, sc=A),
                dict(dc=sb.E4M3, dsc=sb.E8M0, sc=D), dict(a=0), dict(w=0), dict(c=0), dict(sa=0), dict(sbp=0), dict(M=(1 << 30) + 1),
                dict(K=(1 << 30) + 1)):
        assert call(**bad) == CB_EARG, bad
    for bad in (dict(da=sb.U8), dict(da=sb.BF16), dict(db=sb.E8M0), dict(dsa=sb.BF16), dict(dsb=sb.U8), dict(dc=sb.I32), dict(dc=sb.E8M0),
                dict(dc=sb.E4M3, dsc=sb.BF16)):
        assert call(**bad) == CB_EDTYPE, bad


def test_norm_refusals(sb, fake):
    Z = (200, 1000, 0)

    def call(nb=2, N=5, Cn=200, x=A, h=B, r=D, y=E, s=F, g=G, ls=H, ga=I, mo=J, dx=sb.BF16, dh=sb.BF16, dr=sb.BF16, dy=sb.BF16, ds=sb.E8M0,
             dga=sb.F32, dmo=sb.F32, dls=sb.F32, xs=Z, hs=Z, rs=Z, ys=Z, ss=(2, 10, 0), gas=(0, 200, 0), mos=(0, 400, 0), nx=2000, nh=2000,
             nr=2000, ny=2000, ns=20, ng=200, nls=200, nga=400, nmo=800, post=1, pre=2, eps=1e-5, alpha=1.0, no=(), gdt=sb.F32):
        def op(name, p, n, d, st, o=0):
            return None if name in no else sb.Backend.bmat(mem(sb, fake, p, n, d), o, *st)
        gm = mem(sb, fake, g, ng, gdt)
        return status(fake.norm_residual, nb, N, Cn, op("x", x, nx, dx, xs), op("h", h, nh, dh, hs),
                      None if "post" in no else sb.Norm(post, eps, gm, gm), alpha, None if "ls" in no else mem(sb, fake, ls, nls, dls),
                      op("ga", ga, nga, dga, gas), op("r", r, nr, dr, rs), None if "pre" in no else sb.Norm(pre, eps, gm, None),
                      op("mo", mo, nmo, dmo, mos), op("mo", mo, nmo, dmo, mos, 200), op("y", y, ny, dy, ys),
                      op("s", s, ns, ds, ss) if dy == sb.E4M3 and "s" not in no else None)
    nh = ("h", "post", "ls", "ga")
    ny = ("y", "pre", "mo", "s")
    assert call() == CB_ECUDA and call(dy=sb.E4M3) == CB_ECUDA and call(dy=sb.E4M3, ds=sb.F32) == CB_ECUDA and call(no=nh) == CB_ECUDA
    assert call(no=ny) == CB_ECUDA and call(no=("post", "ls", "ga", "pre", "mo")) == CB_ECUDA and call(no=("r",)) == CB_ECUDA
    assert call(r=A) == CB_ECUDA and call(r=B) == CB_ECUDA and call(r=A, y=B) == CB_ECUDA and call(y=A, no=("r",)) == CB_ECUDA  # in place
    assert call(dx=sb.F32, dr=sb.F32) == CB_ECUDA and call(dx=sb.F32, dr=sb.F32, dh=sb.F16, dy=sb.F16) == CB_ECUDA
    assert call(gas=Z, nga=2000) == CB_ECUDA and call(gas=(0, 0, 0)) == CB_ECUDA and call(xs=(200, 0, 0)) == CB_ECUDA
    assert call(post=0, no=()) == CB_EARG  # weights without a norm
    for bad in (dict(nb=0), dict(N=0), dict(Cn=0), dict(no=("r",) + ny), dict(no=("h",)), dict(no=("h", "post", "ls")), dict(no=("h", "ls", "ga")),
                dict(no=nh, alpha=2.0), dict(no=("y",)), dict(no=("y", "pre")), dict(no=("y", "mo")), dict(dy=sb.E4M3, no=("s",)),
                dict(alpha=float("nan")), dict(alpha=float("inf")), dict(eps=-1.0), dict(eps=float("nan")), dict(post=3), dict(pre=-1),
                dict(ng=199), dict(gdt=sb.BF16), dict(g=G + 2), dict(nls=199), dict(dls=sb.BF16), dict(nga=399), dict(nmo=799),
                dict(xs=(200, 1000, 1)), dict(ys=(200, 1000, 1)), dict(nx=1999), dict(nh=1999), dict(nr=1999), dict(ny=1999),
                dict(dy=sb.E4M3, ns=19), dict(rs=(199, 1000, 0)), dict(ys=(200, 0, 0)), dict(dy=sb.E4M3, ss=(1, 10, 0)), dict(x=0), dict(h=0),
                dict(r=0), dict(y=0), dict(r=A + 16), dict(y=D), dict(y=D + 3998), dict(r=A, rs=(208, 1040, 0), nr=2080), dict(r=B, y=B),
                dict(r=I), dict(y=J), dict(y=H), dict(y=G), dict(dy=sb.E4M3, s=A), dict(dy=sb.E4M3, s=E), dict(dy=sb.E4M3, s=G),
                dict(dx=sb.F32, dr=sb.F32, dh=sb.BF16, r=B), dict(N=(1 << 30) + 1), dict(Cn=(1 << 30) + 1), dict(ga=I + 2)):
        assert call(**bad) == CB_EARG, bad
    for bad in (dict(dx=sb.E4M3), dict(dh=sb.F16), dict(dh=sb.F32), dict(dr=sb.F32), dict(dr=sb.F16), dict(dy=sb.F32), dict(dy=sb.F16),
                dict(dga=sb.I32), dict(dmo=sb.E4M3), dict(dy=sb.E4M3, ds=sb.BF16)):
        assert call(**bad) == CB_EDTYPE, bad


def test_rope_axes_refusals(sb, fake):
    def table(npos=64, widths=(8, 4, 4), order=0, first=0, n=64 * 16, dt=sb.F32, addr=A, **sc):
        kw = dict(theta=10000.0, kind=0, factor=2.0, orig_len=2048.0)
        kw.update(sc)
        return status(fake.rope_axes_table, npos, sb.RopeAxes(widths, order), first, sb.RopeScaling(**kw), mem(sb, fake, addr, n, dt))
    assert table() == CB_ECUDA and table(order=1) == CB_ECUDA and table(widths=(16,)) == CB_ECUDA and table(kind=3) == CB_ECUDA
    assert table(widths=(4, 4, 4, 4)) == CB_ECUDA and table(first=-31) == CB_ECUDA
    for bad in (dict(widths=()), dict(widths=(8, 3, 5)), dict(widths=(8, 0, 8)), dict(widths=(8, -4, 4)), dict(order=2), dict(npos=0),
                dict(n=64 * 16 - 1), dict(dt=sb.BF16), dict(addr=A + 4), dict(theta=1.0), dict(kind=4), dict(widths=(2, 8), order=1, n=640),
                dict(widths=(256, 2), n=64 * 258), dict(widths=(2, 2, 4), order=1, n=512), dict(first=2 ** 31)):
        assert table(**bad) == CB_EARG, bad
    five = sb.RopeAxes((2, 2, 2, 2))
    five.axes = 5
    assert status(fake.rope_axes_table, 64, five, 0, None, mem(sb, fake, A, 640, sb.F32)) == CB_EARG

    def call(nb=2, N=6, heads=3, hd=16, rot=12, layout=0, widths=(4, 4, 4), order=0, x=A, y=B, cs=D, ncs=7 * 12, npos=7, pos=None, npid=36,
             pdt=None, grid=(1, 2, 3), dx=sb.BF16, dy=sb.BF16, n=576):
        X = sb.Backend.bmat(mem(sb, fake, x, n, dx), 0, 48, 288, 16)
        Y = sb.Backend.bmat(mem(sb, fake, y, 576, dy), 0, 48, 288, 16)
        P = None if pos is None else mem(sb, fake, pos, npid, sb.I32 if pdt is None else pdt)
        return status(fake.rope_rotate_axes, nb, N, heads, hd, rot, layout, sb.RopeAxes(widths, order), X, Y, mem(sb, fake, cs, ncs, sb.F32),
                      npos, P, grid)
    assert call() == CB_ECUDA and call(pos=E, grid=None) == CB_ECUDA and call(x=B) == CB_ECUDA and call(grid=(5, 5, 5)) == CB_ECUDA
    assert call(widths=(12,), grid=(6,)) == CB_ECUDA and call(order=1, layout=1) == CB_ECUDA and call(dx=sb.F32) == CB_ECUDA
    for bad in (dict(pos=E), dict(grid=None), dict(pos=E, grid=None, npid=35), dict(pos=E, grid=None, pdt=sb.F32), dict(grid=(1, 1, 3)),
                dict(grid=(0, 2, 3)), dict(grid=(1, -2, -3)), dict(grid=(1 << 20, 1 << 20, 1)), dict(widths=(4, 4)), dict(widths=(4, 4, 6)),
                dict(rot=10), dict(ncs=83), dict(npos=8), dict(n=575), dict(y=D), dict(pos=B, grid=None), dict(x=B + 32), dict(N=0),
                dict(layout=2), dict(order=2), dict(hd=10), dict(cs=D + 4)):
        assert call(**bad) == CB_EARG, bad
    for bad in (dict(dx=sb.U8), dict(dy=sb.F16), dict(dx=sb.E4M3)):
        assert call(**bad) == CB_EDTYPE, bad


def test_no_backend(sb):
    L = sb.lib()
    z = sb.Opnd()
    n = None
    assert L.cb_quantize_e4m3(n, 1, 1, 1, 1, z, z, z) == CB_EARG
    assert L.cb_gemm_e4m3(n, 1, 1, 1, z, z, z, z, z, n, n, 0) == CB_EARG
    assert L.cb_norm_residual(n, 1, 1, 1, z, n, n, 1.0, n, n, n, n, n, n, n, n) == CB_EARG
    assert L.cb_rope_axes_table(n, 1, n, 0, n, n) == CB_EARG
    assert L.cb_rope_rotate_axes(n, 1, 1, 1, 2, 2, 0, n, z, z, n, 1, n, n) == CB_EARG
