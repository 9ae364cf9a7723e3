"""Refusals of the prompt-path operators (cb_rope_table, cb_rope_rotate,
cb_cross_attend, cb_groupnorm), checked without a device: arguments are
validated before anything touches CUDA, so a zeroed handle stands in for the
backend, wrapped addresses for its buffers. Each case changes one argument of a
call that passes validation (which then fails for want of a device)."""
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


def mem(sb, be, addr, nbytes, dt):
    m = C.c_void_p()
    assert sb.lib().cb_wrap(be.h, C.c_void_p(addr), nbytes, dt, C.byref(m)) == 0
    return sb.Mem(be, m.value)


def status(fn, *a, **k):
    import sys
    try:
        fn(*a, **k)
    except sys.modules["sam3_b200"].CBError as e:
        return e.status
    return 0


A, B, D, E, F, G = (i << 32 for i in range(1, 7))


def test_rope_table_refusals(sb, fake):
    def call(npos=64, rot=32, first=0, n=64 * 32 * 4, dt=sb.F32, addr=A, null=False, **sc):
        kw = dict(theta=10000.0, kind=0, factor=2.0, orig_len=2048.0)
        kw.update(sc)
        return status(fake.rope_table, npos, rot, first, None if null else sb.RopeScaling(**kw),
                      mem(sb, fake, addr, n, dt))
    inf, nan = float("inf"), float("nan")
    assert call() == CB_ECUDA and call(null=True) == CB_ECUDA and call(kind=3) == CB_ECUDA
    assert call(first=2 ** 31 - 64) == CB_ECUDA and call(first=-2 ** 31) == CB_ECUDA
    for bad in (dict(npos=0), dict(npos=-1), dict(rot=0), dict(rot=31), dict(rot=258), dict(n=64 * 32 * 4 - 4),
                dict(npos=65), dict(dt=sb.BF16), dict(addr=A + 4), dict(theta=1.0), dict(theta=nan), dict(theta=inf),
                dict(amplitude=0.0), dict(amplitude=nan), dict(amplitude=-1.0), dict(kind=4), dict(kind=-1),
                dict(kind=1, factor=0.5), dict(kind=2, factor=nan), dict(kind=3, factor=inf),
                dict(kind=3, orig_len=0.0), dict(kind=3, turns_slow=0.0), dict(kind=3, turns_fast=1.0),
                dict(kind=3, orig_len=nan), dict(first=2 ** 31), dict(first=-2 ** 31 - 1)):
        assert call(**bad) == CB_EARG, bad


def test_rope_rotate_refusals(sb, fake):
    def call(nb=2, N=5, heads=3, hd=16, rot=8, layout=0, dx=sb.BF16, dy=sb.BF16, x=A, y=B, xo=0, ld=48, s0=240, s1=16,
             ldy=48, s0y=240, s1y=16, nx=480, ny=480, npos=7, cs=D, ncs=7 * 8, pos=None, npid=10, pdt=None, pos0=0):
        es = {sb.F32: 4, sb.BF16: 2, sb.F16: 2, sb.U8: 1, sb.I32: 4}
        X = sb.Backend.bmat(mem(sb, fake, x, nx * es[dx], dx), xo, ld, s0, s1)
        Y = sb.Backend.bmat(mem(sb, fake, y, ny * es[dy], dy), 0, ldy, s0y, s1y)
        P = None if pos is None else mem(sb, fake, pos, npid * 4, sb.I32 if pdt is None else pdt)
        return status(fake.rope_rotate, nb, N, heads, hd, rot, layout, X, Y, mem(sb, fake, cs, ncs * 4, sb.F32), npos,
                      P, pos0)
    assert call() == CB_ECUDA and call(layout=1) == CB_ECUDA and call(pos=E) == CB_ECUDA and call(pos0=2) == CB_ECUDA
    assert call(x=B) == CB_ECUDA  # in place
    assert call(dx=sb.F32) == CB_ECUDA and call(s0=0) == CB_ECUDA  # converted; one input for every sequence
    assert call(s1y=80, ldy=16, s0y=240) == CB_ECUDA  # head-major output
    for bad in (dict(nb=0), dict(N=0), dict(heads=0), dict(hd=0), dict(rot=0), dict(rot=7), dict(rot=18), dict(layout=2),
                dict(npos=0), dict(npos=4), dict(npos=8), dict(ncs=55), dict(cs=D + 4), dict(pos0=-1), dict(pos0=3),
                dict(pos=E, npid=9), dict(pos=E, pos0=1), dict(pos=E, pdt=sb.F32), dict(pos=E + 2),
                dict(nx=479), dict(ny=479), dict(xo=1), dict(xo=-1), dict(ld=-48), dict(s0=-1), dict(s1=-1), dict(x=A + 1),
                dict(s1y=8), dict(ldy=32), dict(s0y=0), dict(s0y=239), dict(x=0), dict(y=0),
                dict(x=B + 32, nx=480), dict(x=B, s1=8), dict(x=B, dx=sb.F32, nx=480), dict(y=D), dict(y=E, pos=E),
                dict(N=(1 << 30) + 1), dict(s0=1 << 62)):
        assert call(**bad) == CB_EARG, bad
    for bad in (dict(dx=sb.U8), dict(dy=sb.I32), dict(dy=sb.F32), dict(dx=sb.F16)):
        assert call(**bad) == CB_EDTYPE, bad


def test_cross_attend_refusals(sb, fake):
    def call(nb=2, Nq=3, Nk=7, heads=4, kv=2, hd=16, dq=sb.BF16, dk=sb.BF16, dv=sb.BF16, do=sb.BF16, q=A, k=B, v=D, o=E,
             nq=384, nk=448, nv=448, no=384, qs=(64, 192, 16), ks=(32, 224, 16), vs=(32, 224, 16), os_=(64, 192, 16),
             klen=None, nl=2, ldt=None, kmask=None, nm=14, mdt=None, scale=0.25):
        es = {sb.F32: 4, sb.BF16: 2, sb.F16: 2, sb.U8: 1, sb.I32: 4}

        def op(p, n, d, st):
            return sb.Backend.bmat(mem(sb, fake, p, n * es[d], d), 0, *st)
        L = None if klen is None else mem(sb, fake, klen, nl * 4, sb.I32 if ldt is None else ldt)
        M = None if kmask is None else mem(sb, fake, kmask, nm, sb.U8 if mdt is None else mdt)
        return status(fake.cross_attend, nb, Nq, Nk, heads, kv, hd, op(q, nq, dq, qs), op(k, nk, dk, ks),
                      op(v, nv, dv, vs), op(o, no, do, os_), L, M, scale)
    assert call() == CB_ECUDA and call(klen=F, kmask=G) == CB_ECUDA and call(v=B) == CB_ECUDA
    assert call(ks=(32, 0, 16), vs=(32, 0, 16)) == CB_ECUDA  # one encoder for every sequence
    for bad in (dict(nb=0), dict(Nq=0), dict(Nk=0), dict(heads=0), dict(kv=0), dict(kv=3), dict(hd=0), dict(hd=12),
                dict(hd=136), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
                dict(scale=3e38),
                dict(klen=F, nl=1), dict(klen=F, ldt=sb.F32), dict(klen=F + 2), dict(kmask=G, nm=13),
                dict(kmask=G, mdt=sb.I32), dict(nq=383), dict(nk=447), dict(nv=447), dict(no=383),
                dict(os_=(64, 0, 16)), dict(os_=(64, 192, 8)), dict(os_=(48, 192, 16)), dict(ks=(-32, 224, 16)),
                dict(o=A), dict(o=B), dict(o=D + 64), dict(q=0), dict(o=F, klen=F), dict(o=G, kmask=G),
                dict(Nk=(1 << 30) + 1), dict(Nq=(1 << 30) + 1)):
        assert call(**bad) == CB_EARG, bad
    for bad in (dict(dk=sb.F16), dict(dv=sb.F16), dict(do=sb.F16), dict(dq=sb.U8), dict(dq=sb.I32)):
        assert call(**bad) == CB_EDTYPE, bad


def test_groupnorm_refusals(sb, fake):
    def call(nb=2, npix=9, Cn=12, groups=4, dx=sb.BF16, dy=sb.BF16, x=A, y=B, nx=216, ny=216, xs=(12, 108, 0),
             ys=(12, 108, 0), g=D, ng=12, b=E, nbias=12, gd=sb.F32, eps=1e-5, act=0):
        es = {sb.F32: 4, sb.BF16: 2, sb.F16: 2, sb.U8: 1}
        X = sb.Backend.bmat(mem(sb, fake, x, nx * es[dx], dx), 0, *xs)
        Y = sb.Backend.bmat(mem(sb, fake, y, ny * es[dy], dy), 0, *ys)
        return status(fake.groupnorm, nb, npix, Cn, groups, X, Y, mem(sb, fake, g, ng * 4, gd),
                      mem(sb, fake, b, nbias * 4, sb.F32), eps, act)
    assert call() == CB_ECUDA and call(x=B) == CB_ECUDA and call(act=1) == CB_ECUDA and call(act=2) == CB_ECUDA
    assert call(dx=sb.F32) == CB_ECUDA and call(xs=(12, 0, 0)) == CB_ECUDA and call(eps=0.0) == CB_ECUDA
    for bad in (dict(nb=0), dict(npix=0), dict(npix=(1 << 40) + 1), dict(Cn=0), dict(groups=0), dict(groups=5),
                dict(groups=13), dict(nx=215), dict(ny=215), dict(ng=11), dict(nbias=11), dict(gd=sb.BF16), dict(g=D + 2),
                dict(eps=-1.0), dict(eps=float("nan")), dict(act=3), dict(act=-1), dict(xs=(12, 108, 1)),
                dict(ys=(11, 108, 0)), dict(ys=(12, 0, 0)), dict(x=B + 24), dict(x=B, xs=(12, 0, 0)), dict(y=D), dict(y=E),
                dict(x=0), dict(x=B, dx=sb.F32)):
        assert call(**bad) == CB_EARG, bad
    for bad in (dict(dx=sb.U8), dict(dy=sb.F32), dict(dx=sb.F16)):
        assert call(**bad) == CB_EDTYPE, bad


def test_no_backend(sb):
    L = sb.lib()
    z = sb.Opnd()
    assert L.cb_rope_table(None, 1, 2, 0, None, None) == CB_EARG
    assert L.cb_rope_rotate(None, 1, 1, 1, 2, 2, 0, z, z, None, 1, None, 0) == CB_EARG
    assert L.cb_cross_attend(None, 1, 1, 1, 1, 1, 8, z, z, z, z, None, None, 1.0) == CB_EARG
    assert L.cb_groupnorm(None, 1, 1, 1, 1, z, z, None, None, 1e-5, 0) == CB_EARG
