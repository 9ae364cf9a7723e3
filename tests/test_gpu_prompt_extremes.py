"""GPU tests of the prompt-path operators, and of cb_attention, at the ends of what their arguments may hold: scores that
rise late or are huge, weights and values far below or above the others, the largest clusters, NaN payloads, the tail
of GELU. Against plain implementations in 64 bits; tolerances as derived in test_gpu_prompt_ops.py, with what a test
adds to them derived beside it.
"""
import math

import pytest

torch = pytest.importorskip("torch")
from test_gpu_prompt_ops import (DT, attend_ref, attend_tol, be, check_attend, check_norm, gen, op, randn, u)  # noqa: E402,F401

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ f16 weights far below the largest
@pytest.mark.parametrize("nats", [12.0, 18.0, 20.0])
@pytest.mark.parametrize("Nq,Nk,h,hd", [(100, 60, 2, 32), (1, 3000, 4, 64), (40, 3000, 1, 32), (300, 600, 4, 64),
                                        (300, 5184, 4, 64), (200, 600, 2, 128)])
def test_cross_attend_f16_sink(be, Nq, Nk, h, hd, nats):
    """A key far above the others whose values are zero: what is left is the others' share. Their weights are rounded by
    half a step of the type or by 2^-34 of the largest weight (1), so that adds 2^-34 sum |v|."""
    g = gen(Nk + hd)
    scale = hd ** -0.5
    q, k = randn(g, 1, Nq, h, hd), 0.5 * randn(g, 1, Nk, h, hd)
    q[..., 0], k[..., 0] = 8.0, 0.0
    k[:, 7] = 0.0
    k[:, 7, :, 0] = nats / (8.0 * scale)
    v = 300.0 * (1.0 + torch.rand(1, Nk, h, hd, device="cuda", generator=g))
    v[:, 7] = 0.0
    q, k, v = (t.half() for t in (q, k, v))
    o = torch.full_like(q, 5.0)
    be.cross_attend(1, Nq, Nk, h, h, hd, *(op(be, t, 0, h * hd, 0, hd) for t in (q, k, v, o)))
    be.sync()
    want, A, big = attend_ref(q.double(), k.double(), v.double(), torch.ones(1, Nk, dtype=torch.bool, device="cuda"), scale)
    tol = attend_tol(torch.float16, want, A, big, hd, Nk) + 2.0 ** -34 * v.double().abs().sum(1, keepdim=True)
    err = (o.double() - want).abs()
    assert (err <= tol).all(), (float((err / tol).max()), float((err / want.abs()).max()))


# ------------------------------------------------------------------ scores far above those of the first keys
def late_key(g, dt, nb, Nq, Nk, h, hd, at, gap, scale):
    """Scores of about 0 with a deviation of half a nat, key `at` at `gap` powers of two above for every row."""
    q, k = randn(g, nb, Nq, h, hd), 0.5 * randn(g, nb, Nk, h, hd)
    q[..., 0], k[..., 0] = 16.0, 0.0
    k[:, at] = 0.0
    k[:, at, :, 0] = gap * math.log(2.0) / (16.0 * scale)
    return q.to(dt), k.to(dt), (randn(g, nb, Nk, h, hd) + 0.5).to(dt)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("nb,Nq,Nk,h,hd,tile,first", [
    (2, 300, 480, 2, 64, 96, 3),     # whole tiles of 96 keys
    (2, 200, 448, 2, 128, 64, 4),    # of 64 keys
    (1, 1, 448, 64, 128, 64, 4),     # one live row of a tile
    (1, 1, 320, 64, 80, 64, 2),
    (1, 300, 1152, 20, 64, 96, 4),   # keys shared by a cluster, the late key in a CTA's second tile
    (2, 40, 60, 2, 32, 60, 0),       # few keys
    (1, 70, 200, 3, 32, 64, 2),      # 64-row tiles, few rows
    (1, 1, 300, 4, 64, 64, 1),
])
@pytest.mark.parametrize("masked", [False, True])
def test_cross_attend_late_score(be, nb, Nq, Nk, h, hd, tile, first, masked, dt):
    """One key's score 20 to 500 powers of two above all before it, at each kind of column of a tile."""
    g = gen(hd + Nk)
    kmask = None
    if masked:  # a hidden key in the first tile, so that later tiles are whole
        kmask = torch.zeros(nb, Nk, dtype=torch.uint8, device="cuda")
        kmask[:, 5] = 1
    for gap in (20, 100, 130, 150, 200, 260, 300, 400, 500):
        for col in (16, 28, 29, 31):
            q, k, v = late_key(g, DT[dt], nb, Nq, Nk, h, hd, first * tile + col, gap, hd ** -0.5)
            check_attend(be, q, k, v, None, kmask)


@pytest.mark.parametrize("gap", [20, 100, 130, 150, 200, 260, 300, 400, 500])
@pytest.mark.parametrize("col", [0, 12, 13, 15])
def test_attention_late_score(be, sb, gap, col):
    """cb_attention on 16-bit rows, as above. Its output is 32-bit: u(bf16) only of the weights."""
    nb, N, h, hd = 2, 576, 16, 64
    E = h * hd
    q, k, v = late_key(gen(gap + col), torch.bfloat16, nb, N, N, h, hd, 3 * 96 + 16 + col, gap, 0.125)
    qkv = torch.cat([t.reshape(nb * N, E) for t in (q, k, v)], 1).contiguous()
    o = torch.empty(nb * N, E, device="cuda")
    be.attention(be.wrap(qkv), nb, N, E, h, hd, None, 0, 0.125, sb.ATTN_TC, be.wrap(o))
    be.sync()
    want, A, big = attend_ref(q.double(), k.double(), v.double(), torch.ones(nb, N, dtype=torch.bool, device="cuda"), 0.125)
    # its exponentials are within 7.5e-5 (2^-13.7) of the weight, not 2^-20
    tol = attend_tol(torch.bfloat16, want, A, big, hd, N) + 2.0 ** -13 * A
    assert ((o.view(nb, N, h, hd).double() - want).abs() <= tol).all()


# ------------------------------------------------------------------ scores of any size
FORMS = [(2, 40, 60, 2, 32),      # few keys
         (1, 1, 300, 4, 64),      # one row, the keys dealt to four warps
         (1, 1, 5000, 2, 128),    # and to a cluster
         (1, 70, 200, 3, 32),     # 64-row tiles
         (1, 40, 3000, 1, 32),    # shared by a cluster
         (2, 300, 480, 2, 64),    # tcgen05
         (2, 200, 448, 2, 128),
         (1, 300, 1152, 20, 64)]  # tcgen05, keys shared by a cluster


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("nb,Nq,Nk,h,hd", FORMS)
def test_cross_attend_huge_scores(be, nb, Nq, Nk, h, hd, dt):
    """Whole-number scores times scales up to 1e38: the largest score has all the weight, so a row is that key's value up
    to the value's own rounding (16 bits: none but the type's; 32 bits: its two parts, 2^-21, and the sum's 2^-22)."""
    g = gen(Nk + hd)
    t = DT[dt]
    q = torch.zeros(nb, Nq, h, hd, device="cuda")
    q[..., 0] = 2.0 ** torch.randint(0, 3, (nb, Nq, h), device="cuda", generator=g) * \
        (1 - 2 * torch.randint(0, 2, (nb, Nq, h), device="cuda", generator=g))
    k = randn(g, nb, Nk, h, hd)
    k[..., 0] = torch.randint(-50, 51, (nb, Nk, h), device="cuda", generator=g).float()
    v = (randn(g, nb, Nk, h, hd) + 0.5).to(t)
    for most, least in ((Nk - 1, 3), (3, Nk // 2), (Nk // 2 + 5, Nk - 3)):
        ki = k.clone()
        ki[:, most, :, 0], ki[:, least, :, 0] = 113.0, -107.0
        want = torch.where((q[..., :1] > 0), v[:, most][:, None].float(), v[:, least][:, None].float())
        for scale in (100.0, 1e6, 1e8, 1e10, 1e20, 1e30, 1e38):
            o = torch.full_like(v[:, :1].expand(nb, Nq, h, hd), 5.0).contiguous()
            qd, kd = q.to(t), ki.to(t)
            be.cross_attend(nb, Nq, Nk, h, h, hd, *(op(be, x, 0, h * hd, x.shape[1] * h * hd, hd) for x in (qd, kd, v, o)),
                            None, None, scale)
            be.sync()
            tol = (2.0 ** -20 if dt == "f32" else u(t)) * want.abs()
            assert ((o.float() - want).abs() <= tol).all(), (scale, most)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("nb,Nq,Nk,h,hd", FORMS)
@pytest.mark.parametrize("common", [2.0 ** 11, 2.0 ** 14, 2.0 ** 15])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_cross_attend_large_common_score(be, nb, Nq, Nk, h, hd, common, sign, dt):
    """All scores near one large number, which must drop out. They are sums of whole numbers, exact in 32 bits; the
    offset may be rounded twice at 2^-24 of up to 2^12 powers of two (2^-12 in a weight's exponent, ln 2 of it in the
    weight), larger ones are not formed before the difference is taken."""
    g = gen(Nk + hd + int(common))
    t = DT[dt]
    q, k = torch.zeros(nb, Nq, h, hd, device="cuda"), torch.zeros(nb, Nk, h, hd, device="cuda")
    q[..., 0], q[..., 1] = 64.0, 1.0
    k[..., 0] = sign * common / 64.0
    k[..., 1] = torch.randint(0, 21, (nb, Nk, h), device="cuda", generator=g).float()
    v = randn(g, nb, Nk, h, hd)
    for scale in (0.25, 1.0, 64.0):
        qd, kd, vd = q.to(t), k.to(t), v.to(t)
        o = torch.full_like(qd, 5.0)
        be.cross_attend(nb, Nq, Nk, h, h, hd, *(op(be, x, 0, h * hd, x.shape[1] * h * hd, hd) for x in (qd, kd, vd, o)),
                        None, None, scale)
        be.sync()
        see = torch.ones(nb, Nk, dtype=torch.bool, device="cuda")
        want, A, _ = attend_ref(qd.double(), kd.double(), vd.double(), see, scale)
        # the differences alone: at most 20 scale each, rounded
        tol = attend_tol(t, want, A, 20.0 * scale, hd, Nk)
        top = min(2.0 ** 12, (common + 20.0) * scale * 1.4427)
        tol = tol + 4 * 2.0 ** -24 * top * A + (2.0 ** -34 * vd.double().abs().sum(1, keepdim=True) if dt == "f16" else 0.0)
        err = (o.double() - want).abs()
        assert (err <= tol).all(), (scale, float((err / tol).max()))


# ------------------------------------------------------------------ 32-bit values of any size
F32_FORMS = [(2, 1, 40, 3, 32), (1, 3, 300, 4, 64), (1, 1, 5000, 2, 128), (2, 90, 60, 2, 32), (1, 600, 700, 4, 40),
             (1, 70, 3000, 2, 128), (1, 40, 3000, 1, 24)]


def check_f32_values(be, q, k, v, klen=None, kmask=None):
    """As check_attend, without its allowance for small numbers: what is allowed is half a step of the smallest ones for
    the result and as much for each of the two products that bring it to its size."""
    nb, Nq, h, hd = q.shape
    Nk, kv = k.shape[1], k.shape[2]
    o = torch.full_like(q, 5.0)
    be.cross_attend(nb, Nq, Nk, h, kv, hd, *(op(be, x, 0, x.stride(1), x.stride(0), x.stride(2)) for x in (q, k, v, o)),
                    be.wrap(klen) if klen is not None else None, be.wrap(kmask) if kmask is not None else None)
    be.sync()
    see = torch.ones(nb, Nk, dtype=torch.bool, device="cuda")
    if klen is not None:
        see &= torch.arange(Nk, device="cuda") < klen[:, None]
    if kmask is not None:
        see &= kmask == 0
    want, A, big = attend_ref(q.double(), k.double(), v.double(), see, hd ** -0.5)
    w = 2 * (hd + 16) * 2.0 ** -23 * big + 2.0 ** -20 + (Nk + 16) * 2.0 ** -23
    tol = (u(torch.float32) * want.abs() + w * (1 + u(torch.float32)) * A) * 1.01 + 1.5 * 2.0 ** -149
    err = (o.double() - want).abs()
    assert (err <= tol).all(), (float((err / tol).max()), float(err.max()))


@pytest.mark.parametrize("nb,Nq,Nk,h,hd", F32_FORMS)
@pytest.mark.parametrize("ex", [-147, -140, -130, -122, -115, -105, -90, -75, -20, 90, 115, 123])
def test_cross_attend_f32_value_sizes(be, nb, Nq, Nk, h, hd, ex):
    """Values of any size keep their bits, with weights spread over many keys and with nearly all of it on one."""
    g = gen(Nk + hd)
    q, k = randn(g, nb, Nq, h, hd), randn(g, nb, Nk, h, hd)
    v = (randn(g, nb, Nk, h, hd).double() * 2.0 ** ex).float()
    assert v.isfinite().all() and v.abs().max() > 0
    check_f32_values(be, q, k, v)
    k[:, Nk // 2] += 4.0 * q[:, 0].mean(1, keepdim=True)
    check_f32_values(be, q, k, v)


@pytest.mark.parametrize("nb,Nq,Nk,h,hd", F32_FORMS)
@pytest.mark.parametrize("low,high", [(-140, -120), (-120, 0), (-120, 124), (0, 126), (-30, 60)])
def test_cross_attend_f32_values_of_two_sizes(be, nb, Nq, Nk, h, hd, low, high):
    """One half of the keys with small values, the other with large ones, either half hidden in some sequences (lengths
    and masks): what is hidden decides nothing, and small values beside larger ones keep what the larger ones leave."""
    nb = 4
    g = gen(Nk + hd + high)
    q, k = randn(g, nb, Nq, h, hd), randn(g, nb, Nk, h, hd)
    ex = torch.where(torch.arange(Nk, device="cuda") < Nk // 2, float(low), float(high)).double()
    sign = torch.where(randn(g, nb, Nk, h, hd) > 0, 1.0, -1.0)
    v = (sign * (1.0 + torch.rand(nb, Nk, h, hd, device="cuda", generator=g).double()) * 2.0 ** ex[:, None, None]).float()
    klen = torch.tensor([Nk, Nk // 2, Nk, 0], device="cuda", dtype=torch.int32)
    kmask = torch.zeros(nb, Nk, dtype=torch.uint8, device="cuda")
    kmask[2, Nk // 2:] = 1
    check_f32_values(be, q, k, v, klen, kmask)


def test_cross_attend_f32_values_that_cancel(be):
    """Sums of nothing, or next to it, of values of ordinary size."""
    g = gen(3)
    q, k, v = randn(g, 1, 40, 2, 32), randn(g, 1, 80, 2, 32), randn(g, 1, 80, 2, 32)
    k[:, 1::2], v[:, 1::2] = k[:, 0::2], -v[:, 0::2]
    check_f32_values(be, q, k, v)
    check_f32_values(be, q, k, v * 2.0 ** 100)
    check_f32_values(be, q, k, torch.zeros_like(v))


@pytest.mark.parametrize("nb,Nq,Nk,h,hd", F32_FORMS)
def test_cross_attend_f32_not_a_number(be, nb, Nq, Nk, h, hd):
    """A visible key that is not a number makes every row NaN, an infinite value its column, whatever the other values'
    sizes; other columns stay what they were."""
    g = gen(5)
    q, k = randn(g, nb, Nq, h, hd).abs() + 0.25, randn(g, nb, Nk, h, hd)
    for ex in (0, -120, 122):
        v = (randn(g, nb, Nk, h, hd).double() * 2.0 ** ex).float()

        def run(k, v):
            o = torch.full_like(q, 5.0)
            be.cross_attend(nb, Nq, Nk, h, h, hd, *(op(be, x, 0, h * hd, x.shape[1] * h * hd, hd) for x in (q, k, v, o)))
            be.sync()
            return o
        for j in (0, Nk // 2, Nk - 1):
            kn = k.clone()
            kn[:, j, :, 3] = math.nan
            assert run(kn, v).isnan().all()
            vn = v.clone()
            vn[:, j, :, 5] = math.inf
            o, want = run(k, vn), run(k, v)
            rest = torch.arange(hd, device="cuda") != 5
            assert (~o[..., 5].isfinite()).all()
            # the same sums, perhaps of values times another power of two
            lim = 2.0 ** -18 * v[..., rest].abs().amax((1, 3))[:, None, :, None]
            assert ((o - want)[..., rest].abs() <= lim).all()


@pytest.mark.parametrize("nb,Nq,Nk,h,hd", FORMS)
@pytest.mark.parametrize("size", ["large", "small"])
def test_cross_attend_bf16_value_sizes(be, nb, Nq, Nk, h, hd, size):
    """bf16 values up to 2^127 / Nk and down to the smallest normal ones, with scores that rise by up to 12 powers of two
    after the first keys. Allowed besides: half a step of the type's smallest numbers (2^-134), and half a step
    of 32 bits' (2^-150) for each of Nk products with weights of 2^-13 of the plain ones, so 2^-137 each."""
    g = gen(Nk + hd)
    q, k, v = late_key(g, torch.bfloat16, nb, Nq, Nk, h, hd, Nk * 2 // 3, 12.0, hd ** -0.5)
    top = 2.0 ** (126 - math.ceil(math.log2(Nk)))
    ex = top if size == "large" else 2.0 ** -126
    v = ((1.0 + torch.rand(nb, Nk, h, hd, device="cuda", generator=g).double()) * ex *
         torch.where(randn(g, nb, Nk, h, hd) > 0, 1.0, -1.0)).bfloat16()
    o = torch.full_like(q, 5.0)
    be.cross_attend(nb, Nq, Nk, h, h, hd, *(op(be, x, 0, h * hd, x.shape[1] * h * hd, hd) for x in (q, k, v, o)))
    be.sync()
    want, A, big = attend_ref(q.double(), k.double(), v.double(), torch.ones(nb, Nk, dtype=torch.bool, device="cuda"),
                              hd ** -0.5)
    e = (hd + 16) * 2.0 ** -23 * big
    w = u(torch.bfloat16) + 2 * e + 2.0 ** -13 + (Nk + 16) * 2.0 ** -23
    tol = (u(torch.bfloat16) * want.abs() + w * (1 + u(torch.bfloat16)) * A) * 1.01 + 2.0 ** -134 + Nk * 2.0 ** -137
    err = (o.double() - want).abs()
    assert (err <= tol).all(), (float((err / tol).max()), float(err.max()))


# ------------------------------------------------------------------ the largest clusters
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("Nq,Nk,h,kv,hd", [(10, 5000, 8, 1, 64), (20, 6000, 5, 1, 32), (15, 4500, 8, 1, 128),
                                           (100, 9000, 1, 1, 128), (1, 9000, 1, 1, 32), (300, 9000, 1, 1, 64)])
def test_cross_attend_sixteen_ctas(be, Nq, Nk, h, kv, hd, dt):
    """Tiles of 64 rows (and others) whose keys 16 CTAs (tcgen05: 8) share, with lengths that leave some of them none."""
    g = gen(Nk)
    q, k, v = (randn(g, 1, n, hh, hd).to(DT[dt]) for n, hh in ((Nq, h), (Nk, kv), (Nk, kv)))
    for n in (Nk, 3 * Nk // 4 + 1, 70, 1, 0):
        check_attend(be, q, k, v, torch.tensor([n], device="cuda", dtype=torch.int32))


# ------------------------------------------------------------------ rotation: what is copied
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("off,hd,rot", [(0, 64, 32), (1, 48, 10), (0, 80, 64)])
def test_rope_rotate_copies_bits(be, sb, dt, halves, off, hd, rot):
    """Columns behind the rotated ones and rows without a position keep every bit: NaN payloads, signalling NaN, -0,
    subnormals, in place and not."""
    nb, N, h = 2, 33, 3
    g = gen(hd)
    it = torch.int32 if dt == "f32" else torch.int16
    info = torch.iinfo(it)
    bits = torch.randint(info.min, info.max, (nb * N * h * hd + off,), device="cuda", generator=g, dtype=torch.int64).to(it)
    nan = {"bf16": 0x7f81, "f16": 0x7c05, "f32": 0x7f800123}[dt]
    bits[::5] = nan
    bits[1::7] = nan - 2 ** 16 + 2 ** 15 if dt != "f32" else nan - 2 ** 31
    x = bits.view(DT[dt])
    pos = torch.where(torch.arange(nb * N, device="cuda") % 3 == 0, -1, 2).int()
    cs = randn(g, 4, rot // 2, 2)
    for place in (False, True):
        y = x.clone() if place else torch.zeros_like(x)
        src = y if place else x
        be.rope_rotate(nb, N, h, hd, rot, int(halves), op(be, src, off, h * hd, N * h * hd, hd),
                       op(be, y, off, h * hd, N * h * hd, hd), be.wrap(cs), 4, be.wrap(pos))
        be.sync()
        got, want = (t[off:].view(it).view(nb * N, h, hd) for t in (y, x))
        assert torch.equal(got[pos < 0], want[pos < 0])
        assert torch.equal(got[..., rot:], want[..., rot:])


# ------------------------------------------------------------------ group norm: the tail of GELU
@pytest.mark.parametrize("tx,ty", [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16")])
def test_groupnorm_gelu_tail(be, tx, ty):
    """GELU over -13 to 7 (gamma 0, so that z = beta exactly) is off by the output's rounding and
    16 bits: |z| h, h = erfc(|z| / sqrt 2) / 2, off by the fit's 3.7e-6 of h, about 20 roundings of 2^-23 for t, the
      polynomial and the products, and three of the exponent z^2 log2(e) / 2: (3.7e-6 + (z^2 + 20) 2^-23) |z| h, and the last
      sum's 2^-24;
    32 bits: 0.5 z (1 + erf): erf off by 2 units and the sum rounded, 2.5 * 2^-24 |z| / 2, and three more roundings."""
    Cn = 4096
    z = torch.linspace(-13.0, 7.0, Cn, device="cuda")
    x = randn(gen(1), 1, 40, Cn).to(DT[tx])
    y = torch.empty(1, 40, Cn, device="cuda", dtype=DT[ty])
    gamma = torch.zeros(Cn, device="cuda")
    be.groupnorm(1, 40, Cn, 32, op(be, x, 0, Cn), op(be, y, 0, Cn), be.wrap(gamma), be.wrap(z), 1e-5, 1)
    be.sync()
    d = z.double()
    want = 0.5 * d * torch.special.erfc(d * -math.sqrt(0.5))
    h = 0.5 * torch.special.erfc(d.abs() * math.sqrt(0.5))
    if ty == "f32":
        own = 1.25 * 2.0 ** -24 * d.abs() + 3 * 2.0 ** -24 * want.abs()
    else:
        own = (3.7e-6 + (d * d + 20.0) * 2.0 ** -23) * d.abs() * h + 2.0 ** -24 * want.abs()
    least = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}[ty]
    tol = u(DT[ty]) * want.abs() + own * (1 + u(DT[ty])) + least
    err = (y[0].double() - want).abs()
    assert (err <= tol).all(), (float((err / tol).max()), float(z[(err / tol).amax(0).argmax()]))


# ------------------------------------------------------------------ group norm: means whose squares pass 32 bits
@pytest.mark.parametrize("nb,n,Cn,G,dt,ex", [(2, 3000, 32, 4, "f32", 57), (1, 3, 32, 4, "f32", 57), (1, 900, 60, 6, "f32", 55),
                                             (1, 20000, 64, 8, "f32", 52), (1, 40, 2051, 1, "f32", 57),
                                             (2, 500, 64, 8, "bf16", 60), (1, 2, 48, 4, "bf16", 62)])
def test_groupnorm_means_of_any_size(be, nb, n, Cn, G, dt, ex):
    """A mean near 2^67 (its square is 2^134) with deviations whose squares and their sums are finite."""
    if dt == "f32":
        x = (randn(gen(n), nb, n, Cn) + 1000.0) * 2.0 ** ex
    else:
        x = ((randn(gen(n), nb, n, Cn) + 16.0) * 2.0 ** ex).bfloat16()
    check_norm(be, x, torch.empty_like(x), G, 0, steps=n // 16)


@pytest.mark.parametrize("N", [576, 130])
def test_attention_not_a_number(be, sb, N):
    """cb_attention: a key that is not a number makes every row of its head NaN at each kind of column of a tile, and no
    row of another head or sequence."""
    nb, h, hd = 2, 16, 64
    E = h * hd
    x = randn(gen(N), nb, N, 3, h, hd).bfloat16()
    for j in (0, 12, 13, 14, 15, 100, N - 1):
        y = x.clone()
        y[1, j, 1, 3, 7] = math.nan
        o = torch.zeros(nb * N, E, device="cuda")
        be.attention(be.wrap(y.view(nb * N, 3 * E)), nb, N, E, h, hd, None, 0, 0.125, sb.ATTN_TC, be.wrap(o))
        be.sync()
        bad = o.view(nb, N, h, hd).isnan()
        assert bad[1, :, 3].all() and int(bad.sum()) == N * hd
