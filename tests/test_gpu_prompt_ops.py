"""GPU tests of the prompt-path operators (cb_rope_table, cb_rope_rotate,
cb_cross_attend, cb_groupnorm) against plain implementations in 64 bits on the
same (already rounded) inputs.

Tolerances. u(T) is half a step of T relative to the value (2^-8 bf16, 2^-11
f16, 2^-24 f32); every result is rounded to T once: u |y|.
  rotation: two products and a sum in 32 bits, 4 * 2^-24 (|x0| + |x1|) |cs|;
  table: the remainder's rounding turns an angle by at most pi/4 * 2^-24, the
    32-bit sine and cosine are within 2 ulp, the amplitude and its product
    round once each: 8 * 2^-24 amplitude; the 64-bit turns are off by two
    roundings of 2^-53, |p| w 2^-52 in all;
  group norm: mean and M2 are merged over at most `steps` partial results of at
    most 32 values in 32 bits and over 512 threads and 16 CTAs, so with n =
    64 + steps each is off by less than n 2^-24 of max |x| / of itself;
    y = act(z), z = (x - mean) rstd g + b: n 2^-24 (rstd max|x| |g| + |z - b| +
    |b|), times 1.13 (the steepest slope of GELU);
  attention: a 32-bit score of hd products is off by e = (hd + 16) 2^-23 scale
    sum |q k| (2^-23: the matrix unit may truncate), which moves a weight by a
    factor of at most 1 + 2 e; exponentials add 2^-20; 16-bit weights are
    rounded: u(T) each; sums over keys add (keys + 16) 2^-23. All of it scales
    with A = sum_j p_j |v_j|.
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def u(dt):
    return torch.finfo(dt).eps / 2


@pytest.fixture()
def be(sb):
    """A backend whose calls run on torch's default stream."""
    b = sb.Backend(torch.cuda.current_device())
    b.set_stream(1)
    yield b
    b.sync()
    b.close()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def op(be, t, off=0, ld=0, s0=0, s1=0):
    return be.bmat(be.wrap(t), off, ld, s0, s1)


# ------------------------------------------------------------------ rotary
def frequencies(rot, sc):
    L = np.longdouble
    j = np.arange(rot // 2).astype(L)
    theta = L(sc.theta)
    if sc.kind == 2 and rot > 2:
        theta = theta * L(sc.factor) ** (L(rot) / L(rot - 2))
    w = theta ** (-2 * j / rot)
    if sc.kind == 1:
        w = w / L(sc.factor)
    if sc.kind == 3:
        def at(n):
            return rot * math.log(sc.orig_len / (2 * math.pi * n)) / (2 * math.log(sc.theta))
        lo, hi = max(math.floor(at(sc.turns_fast)), 0), min(math.ceil(at(sc.turns_slow)), rot - 1)
        r = np.clip((j - lo) / max(hi - lo, 1e-3), 0, 1)
        w = w * (1 - r) + w / L(sc.factor) * r
    return w


@pytest.mark.parametrize("npos,rot,first,sc", [
    (1, 2, 0, {}),
    (5184, 64, 0, {}),
    (77, 256, 0, dict(kind=1, factor=3.0)),
    (129, 2, 5, dict(kind=2, factor=4.0)),
    (1000, 50, 1000000, dict(kind=2, factor=8.0, theta=500000.0)),
    (4097, 128, 60000, dict(kind=3, factor=16.0, orig_len=8192.0, theta=500000.0, amplitude=1.277)),
    (300, 96, 2 ** 31 - 300, {}),
    (300, 96, -(2 ** 31), dict(amplitude=0.5)),
])
def test_rope_table(be, sb, npos, rot, first, sc):
    sc = sb.RopeScaling(**sc)
    cs = torch.full((npos * rot + 8,), 7.0, device="cuda")
    be.rope_table(npos, rot, first, sc, be.wrap(cs))
    w = frequencies(rot, sc)
    p = np.arange(first, first + npos).astype(np.longdouble)
    a = p[:, None] * w[None]
    want = np.stack([np.cos(a), np.sin(a)], -1) * sc.amplitude
    tol = sc.amplitude * (8 * 2.0 ** -24 + np.abs(a)[..., None] * 2.0 ** -52)
    got = cs.cpu().numpy().astype(np.float64)
    assert (got[npos * rot:] == 7.0).all()
    err = np.abs(got[:npos * rot].reshape(npos, rot // 2, 2) - want)
    assert (err <= tol).all(), float((err / tol).max())


def rotate_ref(x, cs, pos, rot, halves, npos):
    """x [nb, N, h, hd] f64, cs [npos, rot/2, 2] f64, pos [nb, N]: (y, bound of the 32-bit arithmetic)."""
    keep = (pos >= 0) & (pos < npos)
    t = cs[pos.clamp(0, npos - 1).long()][:, :, None]
    c, s = t[..., 0], t[..., 1]
    i0 = torch.arange(rot // 2, device="cuda") * (1 if halves else 2)
    i1 = i0 + (rot // 2 if halves else 1)
    a, b = x[..., i0], x[..., i1]
    y, e = x.clone(), torch.zeros_like(x)
    k = keep[:, :, None, None]
    y[..., i0] = torch.where(k, a * c - b * s, a)
    y[..., i1] = torch.where(k, a * s + b * c, b)
    m = 4 * 2.0 ** -24 * (a.abs() + b.abs()) * torch.maximum(c.abs(), s.abs())
    e[..., i0] = torch.where(k, m, 0.0)
    e[..., i1] = torch.where(k, m, 0.0)
    return y, e


@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("nb,N,h,hd,rot,tx,ty,mode", [
    (1, 1, 1, 2, 2, "f32", "f32", "rows"),
    (3, 1, 20, 64, 64, "bf16", "bf16", "pos"),
    (2, 130, 6, 64, 64, "bf16", "bf16", "rows"),
    (2, 33, 3, 80, 32, "f32", "f32", "pos"),
    (2, 33, 3, 80, 32, "f16", "f16", "pos"),
    (1, 65, 5, 72, 34, "bf16", "bf16", "pos"),     # no whole vectors
    (2, 9, 4, 128, 128, "f32", "bf16", "rows"),
    (2, 9, 4, 96, 48, "f32", "f16", "pos"),
    (1, 3000, 33, 128, 128, "f16", "f16", "rows"),  # several heads per thread
])
def test_rope_rotate(be, sb, nb, N, h, hd, rot, tx, ty, mode, halves):
    g = gen(100 + N + h)
    npos = N + 5
    pad, tail = 8, 16
    ld = h * hd + pad
    x = randn(g, nb, N, ld).to(DT[tx])
    y = torch.full((nb * N * h * hd + tail,), 3.0, device="cuda", dtype=DT[ty])
    ang = torch.rand(npos, rot // 2, device="cuda", generator=g, dtype=torch.float64) * 6.3
    cs = torch.stack([ang.cos(), ang.sin()], -1).float()
    pos = None
    pos0 = 3
    if mode == "pos":
        pos0 = 0
        pos = torch.randint(-2, npos + 2, (nb, N), device="cuda", generator=g, dtype=torch.int32)
    be.rope_rotate(nb, N, h, hd, rot, sb.ROPE_HALVES if halves else sb.ROPE_PAIRS,
                   op(be, x, 0, ld, N * ld, hd), op(be, y, 0, h * hd, N * h * hd, hd), be.wrap(cs), npos,
                   be.wrap(pos) if pos is not None else None, pos0)
    at = pos if pos is not None else (torch.arange(N, device="cuda") + pos0).expand(nb, N)
    want, e = rotate_ref(x[..., :h * hd].reshape(nb, N, h, hd).double(), cs.double(), at, rot, halves, npos)
    got = y[:nb * N * h * hd].view(nb, N, h, hd).double()
    tol = u(DT[ty]) * want.abs() + e * (1 + u(DT[ty])) + 2.0 ** -24 * 2 * (ty == "f16")  # f16 subnormals
    assert ((got - want).abs() <= tol).all()
    assert (y[nb * N * h * hd:] == 3.0).all()


@pytest.mark.parametrize("off,ldpad,dt", [(1, 0, "bf16"), (3, 1, "f32"), (8, 8, "bf16"), (0, 2, "f16")])
@pytest.mark.parametrize("halves", [False, True])
def test_rope_rotate_in_place_heads_first_and_odd_strides(be, sb, off, ldpad, dt, halves):
    """[nb, h, N, hd] order, starts and strides off the vectors' alignment, in place; the rest of the buffer stays."""
    nb, N, h, hd, rot = 2, 37, 3, 48, 32
    ld = hd + ldpad
    g = gen(7)
    buf = randn(g, off + nb * h * N * ld).to(DT[dt])
    before = buf.clone()
    cs = randn(g, N, rot // 2, 2)
    o = op(be, buf, off, ld, h * N * ld, N * ld)
    be.rope_rotate(nb, N, h, hd, rot, int(halves), o, o, be.wrap(cs), N)
    x = before[off:].view(nb, h, N, ld)[..., :hd].permute(0, 2, 1, 3)
    want, e = rotate_ref(x.double(), cs.double(), torch.arange(N, device="cuda").expand(nb, N), rot, halves, N)
    got = buf[off:].view(nb, h, N, ld)
    tol = u(DT[dt]) * want.abs() + 1.01 * e + 2.0 ** -24 * 2 * (dt == "f16")
    assert ((got[..., :hd].permute(0, 2, 1, 3).double() - want).abs() <= tol).all()
    assert torch.equal(got[..., hd:], before[off:].view(nb, h, N, ld)[..., hd:])
    assert torch.equal(buf[:off], before[:off])


def test_rope_rotate_matches_rope_apply_and_undoes_itself(be, sb):
    """The pair layout is cb_rope_apply's on the same table; turning by the negated angles gives the rows back."""
    N, E, hd = 50, 128, 64
    g = gen(3)
    qkv = randn(g, N, 3 * E)
    cs = torch.empty(N, hd // 2, 2, device="cuda")
    be.rope_table(N, hd, 0, None, be.wrap(cs))
    out = torch.empty(N, 2 * E, device="cuda")
    be.rope_rotate(1, N, 2 * E // hd, hd, hd, sb.ROPE_PAIRS, op(be, qkv, 0, 3 * E, 0, hd), op(be, out, 0, 2 * E, 0, hd),
                   be.wrap(cs), N)
    ref = qkv.clone()
    be.rope_apply(be.wrap(ref), N, E, hd, N, be.wrap(cs))
    assert (out - ref[:, :2 * E]).abs().max() <= 8 * 2.0 ** -24 * qkv.abs().max()
    back = cs.clone()
    back[..., 1] *= -1
    o = op(be, out, 0, 2 * E, 0, hd)
    be.rope_rotate(1, N, 2 * E // hd, hd, hd, sb.ROPE_PAIRS, o, o, be.wrap(back), N)
    assert (out - qkv[:, :2 * E]).abs().max() <= 24 * 2.0 ** -24 * qkv.abs().max()


# ------------------------------------------------------------------ cross attention
def attend_ref(q, k, v, see, scale):
    """q [nb, Nq, h, hd], k, v [nb, Nk, kv, hd], see [nb, Nk], all f64: (o, A, largest scale sum |q k|)."""
    g = q.shape[2] // k.shape[2]
    k = torch.where(see[:, :, None, None], k, 0.0).repeat_interleave(g, 2)
    v = torch.where(see[:, :, None, None], v, 0.0).repeat_interleave(g, 2)
    s = torch.einsum("bqhd,bkhd->bhqk", q, k) * scale
    big = float(torch.einsum("bqhd,bkhd->bhqk", q.abs(), k.abs()).max()) * scale if s.numel() else 0.0
    s = s.masked_fill(~see[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m.isinf(), 0.0, m))
    t = p.sum(-1, keepdim=True)
    p = torch.where(t > 0, p / t, 0.0)
    return torch.einsum("bhqk,bkhd->bqhd", p, v), torch.einsum("bhqk,bkhd->bqhd", p, v.abs()), big


def attend_tol(dt, o, A, big, hd, Nk):
    e = (hd + 16) * 2.0 ** -23 * big
    w = (0.0 if dt == torch.float32 else u(dt)) + 2 * e + 2.0 ** -20 + (Nk + 16) * 2.0 ** -23
    return (u(dt) * o.abs() + w * (1 + u(dt)) * A) * 1.01 + 1e-30 + (2.0 ** -24 if dt == torch.float16 else 0.0)


def check_attend(be, q, k, v, klen=None, kmask=None, scale=None, o=None, args=None):
    nb, Nq, h, hd = q.shape
    Nk, kv = k.shape[1], k.shape[2]
    scale = hd ** -0.5 if scale is None else scale
    if o is None:
        o = torch.full((nb, Nq, h, hd), 5.0, device="cuda", dtype=q.dtype)
    def d(t):
        return op(be, t, 0, t.stride(1), t.stride(0), t.stride(2))
    a = args or [d(q), d(k), d(v), d(o)]
    be.cross_attend(nb, Nq, Nk, h, kv, hd, *a, be.wrap(klen) if klen is not None else None,
                    be.wrap(kmask) if kmask is not None else None, scale)
    be.sync()
    see = torch.ones(nb, Nk, dtype=torch.bool, device="cuda")
    if klen is not None:
        see &= torch.arange(Nk, device="cuda") < klen[:, None]
    if kmask is not None:
        see &= kmask == 0
    want, A, big = attend_ref(q.double(), k.double(), v.double(), see, scale)
    tol = attend_tol(q.dtype, want, A, big, hd, Nk)
    err = (o.double() - want).abs()
    assert (err <= tol).all(), (float((err / tol).max()), float(err.max()))
    none = ~see.any(1)
    assert (o[none] == 0).all()
    return o


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("nb,Nq,Nk,h,kv,hd", [
    (1, 1, 1, 1, 1, 8),
    (2, 1, 63, 4, 1, 64),
    (3, 1, 1500, 16, 4, 64),      # single tokens, shared key heads, keys split over CTAs
    (1, 1, 5000, 2, 2, 128),      # 16 CTAs share the keys of one row
    (2, 5, 64, 6, 2, 32),         # 15 rows of a key head
    (1, 17, 65, 3, 1, 40),        # rows of one query in two tiles
    (2, 200, 33, 8, 8, 32),
    (1, 201, 1300, 8, 8, 32),
    (2, 130, 257, 4, 2, 64),
    (1, 300, 700, 5, 5, 80),
    (1, 129, 640, 2, 1, 128),
    (1, 64, 128, 1, 1, 16),
    (2, 700, 900, 4, 4, 64),
    (1, 513, 1025, 4, 2, 128),
])
def test_cross_attend(be, nb, Nq, Nk, h, kv, hd, dt):
    g = gen(Nq * 7 + Nk)
    check_attend(be, randn(g, nb, Nq, h, hd).to(DT[dt]), randn(g, nb, Nk, kv, hd).to(DT[dt]),
                 (randn(g, nb, Nk, kv, hd) + 0.5).to(DT[dt]))


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("Nq,Nk,h,kv,hd", [(1, 300, 4, 1, 64), (70, 39, 8, 8, 32), (3, 1700, 8, 2, 128), (300, 600, 4, 4, 64),
                                           (260, 500, 2, 2, 128), (400, 1000, 4, 4, 32)])
@pytest.mark.parametrize("with_len,with_mask", [(True, False), (False, True), (True, True)])
def test_cross_attend_lengths_and_masks(be, Nq, Nk, h, kv, hd, dt, with_len, with_mask):
    """Lengths of zero, one, past Nk and below zero, masks that leave a sequence empty or one key, a masked tile in
    front; what masked and absent rows hold (NaN, infinities, the type's lowest value) must not show."""
    nb = 6
    g = gen(Nk + hd)
    q, k, v = (randn(g, nb, n, hh, hd).to(DT[dt]) for n, hh in ((Nq, h), (Nk, kv), (Nk, kv)))
    see = torch.ones(nb, Nk, dtype=torch.bool, device="cuda")
    klen = kmask = None
    if with_len:
        klen = torch.tensor([0, 1, Nk, Nk + 100, -5, Nk // 2 + 1], device="cuda", dtype=torch.int32)
        see &= torch.arange(Nk, device="cuda") < klen[:, None]
    if with_mask:
        kmask = (torch.rand(nb, Nk, device="cuda", generator=g) < 0.4).to(torch.uint8) * 255
        kmask[2] = 1
        kmask[3] = 2
        kmask[3, Nk - 1] = 0
        kmask[5, :min(Nk // 2, 130)] = 1
        see &= kmask == 0
    bad = torch.tensor([math.nan, math.inf, -math.inf, float(torch.finfo(DT[dt]).min)], device="cuda")
    fill = bad[torch.randint(0, 4, (nb, Nk, kv, hd), device="cuda", generator=g)].to(DT[dt])
    hide = ~see[:, :, None, None]
    k2, v2 = torch.where(hide, fill, k), torch.where(hide, fill, v)
    o = torch.full((nb, Nq, h, hd), 5.0, device="cuda", dtype=DT[dt])
    check_attend(be, q, torch.where(hide, 0.0, k), torch.where(hide, 0.0, v), klen, kmask, None, o)
    o2 = torch.empty_like(o)
    def d(t):
        return op(be, t, 0, t.stride(1), t.stride(0), t.stride(2))
    be.cross_attend(nb, Nq, Nk, h, kv, hd, d(q), d(k2), d(v2), d(o2), be.wrap(klen) if klen is not None else None,
                    be.wrap(kmask) if kmask is not None else None)
    be.sync()
    assert torch.equal(o, o2)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("masked", [False, True])
def test_cross_attend_hidden_keys_many_times(be, hd, masked):
    """Short sequences of other lengths after one another in each CTA's rings: what lies behind their ends (the
    type's largest values) must never be taken for values, however loads and products interleave."""
    nb, Nq, Nk, h = 40, 300, 500, 4
    g = gen(77)
    dt = torch.float16
    q, k, v = (randn(g, nb, n, h, hd).to(dt) for n in (Nq, Nk, Nk))
    klen = torch.randint(1, Nk + 1, (nb,), device="cuda", generator=g, dtype=torch.int32)
    see = torch.arange(Nk, device="cuda") < klen[:, None]
    kmask = None
    if masked:
        kmask = (torch.rand(nb, Nk, device="cuda", generator=g) < 0.3).to(torch.uint8)
        see &= kmask == 0
    v[~see] = math.inf
    k[~see] = math.nan
    first = None
    def d(t):
        return op(be, t, 0, t.stride(1), t.stride(0), t.stride(2))
    for _ in range(25):
        o = torch.full_like(q, 3.0)
        be.cross_attend(nb, Nq, Nk, h, h, hd, d(q), d(k), d(v), d(o), be.wrap(klen),
                        be.wrap(kmask) if masked else None)
        be.sync()
        first = o if first is None else first
        assert torch.equal(o, first)
    assert first.isfinite().all()
    want, A, big = attend_ref(q.double(), torch.where(see[:, :, None, None], k, 0).double(),
                              torch.where(see[:, :, None, None], v, 0).double(), see, hd ** -0.5)
    assert ((first.double() - want).abs() <= attend_tol(dt, want, A, big, hd, Nk)).all()


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("Nq,Nk,hd,shift", [(4, 200, 64, 0), (150, 300, 32, 1), (150, 300, 32, 2), (200, 700, 64, 4),
                                            (200, 700, 128, 8)])
def test_cross_attend_layouts(be, Nq, Nk, hd, shift, dt):
    """k | v in one row, heads before rows, starts and strides off the vectors' alignment; around O nothing changes."""
    nb, h = 2, 4
    g = gen(shift + 31)
    ld = 2 * h * hd + shift
    kv = randn(g, nb * Nk * ld + 16).to(DT[dt])
    at = kv[shift:shift + nb * Nk * ld].view(nb, Nk, ld)
    k, v = at[..., :h * hd].unflatten(2, (h, hd)), at[..., h * hd:2 * h * hd].unflatten(2, (h, hd))
    qs = (Nq + 1) * hd + shift
    qb = randn(g, nb * h * qs + 16).to(DT[dt])
    q = torch.as_strided(qb, (nb, Nq, h, hd), (h * qs, hd, qs, 1), shift)
    lo = h * hd + shift
    ob = torch.full((nb * Nq * lo + 16,), 9.0, device="cuda", dtype=DT[dt])
    o = torch.as_strided(ob, (nb, Nq, h, hd), (Nq * lo, lo, hd, 1), shift)
    mkv, mq, mo = be.wrap(kv), be.wrap(qb), be.wrap(ob)
    check_attend(be, q, k, v, o=o, args=[
        be.bmat(mq, shift, hd, h * qs, qs), be.bmat(mkv, shift, ld, Nk * ld, hd),
        be.bmat(mkv, shift + h * hd, ld, Nk * ld, hd), be.bmat(mo, shift, lo, Nq * lo, hd)])
    rest = torch.ones_like(ob, dtype=torch.bool)
    torch.as_strided(rest, o.shape, o.stride(), shift).fill_(False)
    assert (ob[rest] == 9.0).all()


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_cross_attend_one_encoder_for_all_and_large_scores(be, dt):
    """Keys and values of stride 0 over sequences; scores that jump late so that running maxima are raised."""
    nb, Nq, Nk, h, hd = 3, 140, 520, 2, 64
    g = gen(5)
    q = randn(g, nb, Nq, h, hd).to(DT[dt])
    k = randn(g, Nk, h, hd)
    k *= torch.linspace(0.2, 5.0, Nk, device="cuda")[:, None, None]
    k, v = k.to(DT[dt]), randn(g, Nk, h, hd).to(DT[dt])
    check_attend(be, q, k.expand(nb, Nk, h, hd), v.expand(nb, Nk, h, hd))
    q1 = q[:, :1].contiguous()
    check_attend(be, q1, k.expand(nb, Nk, h, hd), v.expand(nb, Nk, h, hd), scale=1.0)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("Nq,Nk,hd", [(2, 150, 64), (50, 40, 32), (300, 450, 64), (200, 300, 128)])
def test_cross_attend_nan_and_infinities_of_visible_keys(be, Nq, Nk, hd, dt):
    """A key that is seen and not a number makes every row NaN wherever it lies, one whose scores are -inf for all
    queries counts nothing, an infinite value shows in its column."""
    h = 2
    g = gen(9)
    q = randn(g, 1, Nq, h, hd).abs().to(DT[dt]) + 0.25
    k, v = (randn(g, 1, Nk, h, hd).to(DT[dt]) for _ in range(2))
    def d(t):
        return op(be, t, 0, t.stride(1), t.stride(0), t.stride(2))
    def run(k, v):
        o = torch.empty_like(q)
        be.cross_attend(1, Nq, Nk, h, h, hd, d(q), d(k), d(v), d(o))
        be.sync()
        return o
    for j in (0, 13, 14, 31, Nk - 1):
        kn = k.clone()
        kn[0, j, :, 3] = math.nan
        assert run(kn, v).isnan().all()
        if dt != "f32":  # 32-bit operands are split into parts: finite values only
            kn = k.clone()
            kn[0, j, :, 3] = math.inf
            assert run(kn, v).isnan().all()
            kn[0, j, :, 3] = -math.inf  # q is positive
            keep = torch.arange(Nk, device="cuda") != j
            klen = torch.tensor([Nk], device="cuda", dtype=torch.int32)
            mask = (~keep).to(torch.uint8)
            o = torch.empty_like(q)
            be.cross_attend(1, Nq, Nk, h, h, hd, d(q), d(k), d(v), d(o), be.wrap(klen), be.wrap(mask))
            be.sync()
            assert ((run(kn, v) - o).abs() <= 4 * u(DT[dt]) * v.abs().max()).all()
            vn = v.clone()
            vn[0, j, :, 5] = math.inf
            o = run(k, vn)
            assert (o[..., 5] == math.inf).all() and o[..., :5].isfinite().all()


def test_cross_attend_largest_numbers(be):
    """Values next to the largest of 32 bits come through (an operand is split into parts that must not overflow)."""
    g = gen(15)
    q, k = randn(g, 1, 40, 1, 32), randn(g, 1, 90, 1, 32)
    big = torch.finfo(torch.float32).max
    v = torch.where(randn(g, 1, 90, 1, 32) > 0, big, -big)
    v[..., :8] = big
    o = torch.empty_like(q)
    be.cross_attend(1, 40, 90, 1, 1, 32, op(be, q, 0, 32), op(be, k, 0, 32), op(be, v, 0, 32), op(be, o, 0, 32))
    be.sync()
    assert not o.isnan().any() and (o[..., 8:].abs() < math.inf).all()
    # an average of equal numbers is that number up to the errors of the weights' sum, infinite where these exceed it
    assert ((o[..., :8] == math.inf) | ((o[..., :8] / big - 1).abs() <= (32 + 16 + 90 + 16) * 2.0 ** -23)).all()


@pytest.mark.parametrize("Nk", [16, 39, 64, 200, 300])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_cross_attend_infinite_query(be, Nk, dt):
    """A query of infinities: zeros where every visible score is -inf, NaN where one is +inf, other rows as always."""
    g = gen(16)
    hd = 32
    q, k, v = (randn(g, 1, n, 1, hd).to(dt) for n in (70, Nk, Nk))
    k[:, :, :, 0] = k[:, :, :, 0].abs() + 0.5
    out = []
    for low, high in ((0.0, 0.0), (-math.inf, math.inf)):
        qi = q.clone()
        qi[0, 3, 0, 0], qi[0, 20, 0, 0], qi[0, 69, 0, 0] = low, high, low
        kmask = torch.zeros(1, Nk, dtype=torch.uint8, device="cuda")
        kmask[0, 5] = 1
        o = torch.empty_like(q)
        be.cross_attend(1, 70, Nk, 1, 1, hd, op(be, qi, 0, hd), op(be, k, 0, hd), op(be, v, 0, hd),
                        op(be, o, 0, hd), None, be.wrap(kmask))
        be.sync()
        out.append(o[0, :, 0])
    assert (out[1][[3, 69]] == 0).all() and out[1][20].isnan().all()
    rest = [r for r in range(70) if r not in (3, 20, 69)]
    if Nk <= 200:
        assert torch.equal(out[0][rest], out[1][rest])
    else:
        # The tcgen05 form takes a tile again for 32 rows at once, so a neighbour's weights are evaluated twice, each
        # time rounded to the type (u = eps / 2) and off by the exponential's 2^-12 at most: weights w, w' of sum 1
        # with |w - w'| <= (2 u + 2 * 2^-12) w in numerator and, unrounded, 2 * 2^-12 w in the sum, then both
        # results rounded: |o - o'| <= (2 u + 4 * 2^-12 + 2 u) max |v|.
        u = torch.finfo(dt).eps / 2
        lim = (4 * u + 2.0 ** -10) * v.float().abs().max()
        assert ((out[0][rest].float() - out[1][rest].float()).abs() <= lim).all()


def test_rope_table_of_every_position(be):
    """As many positions as the call takes."""
    npos = 2 ** 31 - 8
    buf = torch.empty(npos, 2, device="cuda")
    be.rope_table(npos, 2, 8, None, be.wrap(buf))
    be.sync()
    for at in (0, npos // 2, npos - 300):
        p = torch.arange(at + 8, at + 308, dtype=torch.float64, device="cuda")
        want = torch.stack([p.cos(), p.sin()], -1)
        # the angle in turns off by half a step of 64 bits for the frequency and as much for the product, each
        # 2^-53 of up to 2^31 / (2 pi) turns, so 2^-52 2^31 in the angle; the rest rounds in 32 bits: the
        # remainder's angle (pi / 4, three roundings), the polynomial's five steps
        assert (buf[at:at + 300].double() - want).abs().max() <= 2.0 ** -21 + 8 * 2.0 ** -24
    del buf
    torch.cuda.empty_cache()


def test_operands_far_into_a_buffer(be, sb):
    """Offsets past 2^31 elements."""
    far = 2 ** 31 + 64
    buf = torch.empty(far + (1 << 20), device="cuda", dtype=torch.bfloat16)
    g = gen(2)
    n = 60 * 128
    tail = buf[far:]
    tail[:4 * n] = randn(g, 4 * n).bfloat16()
    near = tail[:4 * n].clone()
    m, mn = be.wrap(buf), be.wrap(near)
    out = torch.empty(2, n, device="cuda", dtype=torch.bfloat16)
    mo = be.wrap(out)
    cs = torch.empty(60, 32, 2, device="cuda")
    be.rope_table(60, 64, 0, None, be.wrap(cs))
    for i, (b, o) in enumerate(((m, far), (mn, 0))):
        be.rope_rotate(1, 60, 2, 64, 64, 0, be.bmat(b, o, 128, 0, 64), be.bmat(mo, i * n, 128, 0, 64), be.wrap(cs), 60)
    be.sync()
    assert torch.equal(out[0], out[1])
    for i, (b, o) in enumerate(((m, far), (mn, 0))):
        be.cross_attend(1, 60, 60, 2, 2, 64, *(be.bmat(b, o + j * n, 128, 0, 64) for j in range(3)),
                        be.bmat(mo, i * n, 128, 0, 64))
    be.sync()
    assert torch.equal(out[0], out[1])
    gamma, beta = torch.ones(128, device="cuda"), torch.zeros(128, device="cuda")
    for i, (b, o) in enumerate(((m, far), (mn, 0))):
        be.groupnorm(1, 60, 128, 8, be.bmat(b, o, 128), be.bmat(mo, i * n, 128), be.wrap(gamma), be.wrap(beta))
    be.sync()
    assert torch.equal(out[0], out[1])
    # results written there, rows 2^29 elements apart
    ld = 2 ** 29
    x = randn(g, 4, 64).bfloat16()
    be.groupnorm(1, 4, 64, 8, op(be, x, 0, 64), be.bmat(m, 0, ld), be.wrap(gamma), be.wrap(beta))
    be.groupnorm(1, 4, 64, 8, op(be, x, 0, 64), be.bmat(mo, 0, 64), be.wrap(gamma), be.wrap(beta))
    be.sync()
    assert all(torch.equal(buf[i * ld:i * ld + 64], out.view(-1)[i * 64:i * 64 + 64]) for i in range(4))
    q = randn(g, 1, 100, 1, 64).bfloat16()
    for i in range(4):
        buf[i * ld:i * ld + 128] = randn(g, 128).bfloat16()
    k = torch.stack([buf[i * ld:i * ld + 64] for i in range(4)]).view(1, 4, 1, 64)
    v = torch.stack([buf[i * ld + 64:i * ld + 128] for i in range(4)]).view(1, 4, 1, 64)
    o = torch.empty_like(q)
    check_attend(be, q, k, v, o=o, args=[op(be, q, 0, 64), be.bmat(m, 0, ld), be.bmat(m, 64, ld), op(be, o, 0, 64)])


# ------------------------------------------------------------------ group norm
def norm_ref(x, G, gamma, beta, eps, act):
    nb, n, Cn = x.shape
    r = x.view(nb, n, G, Cn // G)
    mean = r.mean((1, 3), keepdim=True)
    rstd = 1.0 / torch.sqrt(((r - mean) ** 2).mean((1, 3), keepdim=True) + eps)
    z0 = ((r - mean) * rstd).view(nb, n, Cn) * gamma
    z = z0 + beta
    y = {0: z, 1: z * torch.special.ndtr(z), 2: z.clamp_min(0)}[act]
    e = (rstd * r.abs().amax((1, 3), keepdim=True)).expand_as(r).reshape(nb, n, Cn) * gamma.abs() + z0.abs() + beta.abs()
    return y, e


def check_norm(be, x, y, G, act, eps=1e-5, steps=0, xs=None, ys=None, seed=1):
    nb, n, Cn = x.shape
    g = gen(seed)
    gamma, beta = 1 + 0.3 * randn(g, Cn), 0.3 * randn(g, Cn)
    be.groupnorm(nb, n, Cn, G, xs or op(be, x, 0, Cn, n * Cn), ys or op(be, y, 0, Cn, n * Cn), be.wrap(gamma),
                 be.wrap(beta), eps, act)
    be.sync()
    want, e = norm_ref(x.double(), G, gamma.double(), beta.double(), eps, act)
    tol = u(y.dtype) * want.abs() + 1.13 * (64 + steps) * 2.0 ** -24 * e * (1 + u(y.dtype)) + 1e-30
    if y.dtype == torch.float16:
        tol = tol + 2.0 ** -24
    err = (y.double() - want).abs()
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("act", [0, 1, 2])
@pytest.mark.parametrize("nb,n,Cn,G,tx,ty", [
    (1, 1, 1, 1, "f32", "f32"),
    (2, 1, 64, 8, "bf16", "bf16"),
    (1, 576, 64, 8, "f32", "f32"),
    (3, 4697, 320, 32, "f16", "f16"),      # ten channels a group
    (2, 5184, 256, 8, "bf16", "bf16"),
    (2, 20736, 256, 32, "f32", "bf16"),
    (1, 333, 96, 96, "f16", "f16"),        # one channel a group
    (2, 130, 93, 31, "f32", "f16"),        # odd widths
    (1, 200, 2051, 1, "f32", "f32"),       # a group wider than a block's row, no vectors
    (1, 70, 6000, 2, "bf16", "bf16"),
    (9, 100, 48, 4, "bf16", "bf16"),
])
def test_groupnorm(be, nb, n, Cn, G, tx, ty, act):
    g = gen(n + Cn)
    x = (randn(g, nb, n, Cn) * 2 + randn(g, Cn)).to(DT[tx])
    check_norm(be, x, torch.empty(nb, n, Cn, device="cuda", dtype=DT[ty]), G, act, steps=n // 16)


def test_groupnorm_large_map(be):
    """More pixels than the CTAs of a cluster keep in shared memory."""
    x = (randn(gen(8), 1, 288 * 288, 64) + 3).bfloat16()
    check_norm(be, x, torch.empty_like(x), 8, 2, steps=1000)
    x = randn(gen(9), 1, 288 * 288, 32)
    check_norm(be, x, torch.empty_like(x), 1, 1, steps=1000)


def test_groupnorm_mean_far_from_zero(be):
    """A mean of 1000 deviations: E[x^2] - E[x]^2 in 32 bits would lose the variance."""
    x = randn(gen(4), 2, 3000, 32) + 1000.0
    check_norm(be, x, torch.empty_like(x), 4, 0, steps=200)


@pytest.mark.parametrize("off,pad,dt", [(0, 8, "bf16"), (1, 3, "bf16"), (2, 2, "f32"), (4, 4, "f16")])
def test_groupnorm_strides_and_in_place(be, off, pad, dt):
    nb, n, Cn, G = 2, 500, 64, 8
    ld, gap = Cn + pad, 24
    s0 = n * ld + gap
    buf = randn(gen(6), off + nb * s0).to(DT[dt])
    before = buf.clone()
    m = be.wrap(buf)
    o = be.bmat(m, off, ld, s0)
    view = torch.as_strided(buf, (nb, n, Cn), (s0, ld, 1), off)
    x = torch.as_strided(before, (nb, n, Cn), (s0, ld, 1), off).contiguous()
    gamma, beta = torch.ones(Cn, device="cuda"), torch.zeros(Cn, device="cuda")
    be.groupnorm(nb, n, Cn, G, o, o, be.wrap(gamma), be.wrap(beta), 1e-5, 0)
    be.sync()
    want, e = norm_ref(x.double(), G, gamma.double(), beta.double(), 1e-5, 0)
    tol = u(DT[dt]) * want.abs() + 128 * 2.0 ** -24 * e + 2.0 ** -24 * (dt == "f16")
    assert ((view.double() - want).abs() <= tol).all()
    rest = torch.ones_like(buf, dtype=torch.bool)
    torch.as_strided(rest, view.shape, view.stride(), off).fill_(False)
    assert torch.equal(buf[rest], before[rest])


def test_groupnorm_constant_group_and_nan(be):
    x = torch.full((1, 50, 16), 2.0, device="cuda")
    x[0, 3, 9] = math.nan
    y = torch.empty_like(x)
    gamma, beta = torch.ones(16, device="cuda"), torch.full((16,), 0.25, device="cuda")
    be.groupnorm(1, 50, 16, 2, op(be, x, 0, 16, 800), op(be, y, 0, 16, 800), be.wrap(gamma), be.wrap(beta), 0.0, 0)
    be.sync()
    # eps 0 and no variance: 0 * inf, as the formula has it; a NaN stays within its group
    assert y[..., :8].isnan().all() and y[..., 8:].isnan().all()
    be.groupnorm(1, 50, 16, 2, op(be, x, 0, 16, 800), op(be, y, 0, 16, 800), be.wrap(gamma), be.wrap(beta), 1e-5, 2)
    be.sync()
    assert (y[..., :8] == 0.25).all() and y[..., 8:].isnan().all()


# ------------------------------------------------------------------ together
def chain(be, sb, x):
    """Rotate queries and keys, attend, normalise the resulting map."""
    nb, N, Nk, h, hd = x["nb"], x["N"], x["Nk"], x["h"], x["hd"]
    w = h * hd
    q, kv = be.wrap(x["q"]), be.wrap(x["kv"])
    rq, rk, o, y = (be.wrap(x[k]) for k in ("rq", "rk", "o", "y"))
    cs = be.wrap(x["cs"])
    be.rope_table(x["npos"], hd, 0, None, cs)
    be.rope_rotate(nb, N, h, hd, hd, sb.ROPE_PAIRS, be.bmat(q, 0, w, N * w, hd), be.bmat(rq, 0, w, N * w, hd), cs, x["npos"])
    be.rope_rotate(nb, Nk, h, hd, hd, sb.ROPE_PAIRS, be.bmat(kv, 0, 2 * w, Nk * 2 * w, hd),
                   be.bmat(rk, 0, w, Nk * w, hd), cs, x["npos"], be.wrap(x["pos"]))
    be.cross_attend(nb, N, Nk, h, h, hd, be.bmat(rq, 0, w, N * w, hd), be.bmat(rk, 0, w, Nk * w, hd),
                    be.bmat(kv, w, 2 * w, Nk * 2 * w, hd), be.bmat(o, 0, w, N * w, hd), be.wrap(x["klen"]),
                    be.wrap(x["kmask"]))
    be.groupnorm(nb, N, w, 8, be.bmat(o, 0, w, N * w), be.bmat(y, 0, w, N * w), be.wrap(x["gamma"]), be.wrap(x["beta"]),
                 1e-5, sb.ACT_RELU)


def chain_inputs(seed, dt, nb=2, N=576, Nk=45, h=8, hd=32):
    g = gen(seed)
    w = h * hd
    e = dict(device="cuda", dtype=dt)
    klen = torch.tensor([Nk, Nk - 7], device="cuda", dtype=torch.int32)[:nb]
    return dict(nb=nb, N=N, Nk=Nk, h=h, hd=hd, npos=1024, q=randn(g, nb, N, w).to(dt), kv=(randn(g, nb, Nk, 2 * w)).to(dt),
                rq=torch.empty(nb, N, w, **e), rk=torch.empty(nb, Nk, w, **e), o=torch.empty(nb, N, w, **e),
                y=torch.empty(nb, N, w, **e), cs=torch.empty(1024, hd // 2, 2, device="cuda"), klen=klen,
                pos=torch.randint(-1, 1024, (nb, Nk), device="cuda", generator=g, dtype=torch.int32),
                kmask=(torch.rand(nb, Nk, device="cuda", generator=g) < 0.2).to(torch.uint8),
                gamma=1 + 0.1 * randn(g, w), beta=0.1 * randn(g, w))


def chain_ref(x):
    nb, N, Nk, h, hd = x["nb"], x["N"], x["Nk"], x["h"], x["hd"]
    w = h * hd
    a = torch.arange(x["npos"], device="cuda", dtype=torch.float64)[:, None] * \
        10000.0 ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
    cs = torch.stack([a.cos(), a.sin()], -1)
    q, _ = rotate_ref(x["q"].double().view(nb, N, h, hd), cs, torch.arange(N, device="cuda").expand(nb, N), hd, False, x["npos"])
    k, _ = rotate_ref(x["kv"][..., :w].double().reshape(nb, Nk, h, hd), cs, x["pos"], hd, False, x["npos"])
    see = (torch.arange(Nk, device="cuda") < x["klen"][:, None]) & (x["kmask"] == 0)
    o, A, _ = attend_ref(q, k, x["kv"][..., w:].double().reshape(nb, Nk, h, hd), see, hd ** -0.5)
    y, e = norm_ref(o.reshape(nb, N, w), 8, x["gamma"].double(), x["beta"].double(), 1e-5, 2)
    return o.reshape(nb, N, w), A.reshape(nb, N, w), y, e


def test_together(be, sb):
    """In 32 bits: rotated rows are off by 2^-21, scores of 32 products by less than 2^-14, so the attended map by less
    than 2^-13 A; the norm scales that by rstd |gamma| (bounded through e / max |o|) and adds its own error."""
    x = chain_inputs(1, torch.float32)
    chain(be, sb, x)
    be.sync()
    o, A, y, e = chain_ref(x)
    assert ((x["o"].double() - o).abs() <= 2.0 ** -13 * A).all()
    tol = 4 * 2.0 ** -13 * float(A.max()) / float(o.abs().max()) * e + 128 * 2.0 ** -24 * e
    assert ((x["y"].double() - y).abs() <= tol).all()
    # far below that in the mean: the bound is the worst case of every rounding at once
    assert float((x["y"].double() - y).norm() / y.norm()) <= 2e-5


def test_together_captured_and_replayed(sb):
    """Two graphs captured on streams of their own replay at the same time, again on new inputs, beside an eager call."""
    dt = torch.bfloat16
    xs = [chain_inputs(s, dt) for s in (11, 12)]
    wants, graphs, streams, bes = [], [], [], []
    for x in xs:
        b = sb.Backend(torch.cuda.current_device())
        b.set_stream(1)
        chain(b, sb, x)
        b.sync()
        wants.append(x["y"].clone())
        s = torch.cuda.Stream()
        b.set_stream(s.cuda_stream)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            chain(b, sb, x)
        graphs.append(g)
        streams.append(s)
        bes.append(b)
    torch.cuda.synchronize()
    for x in xs:
        x["y"].zero_()
    eager = chain_inputs(13, dt)
    b3 = sb.Backend(torch.cuda.current_device())
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        chain(b3, sb, eager)  # on the backend's own stream
    torch.cuda.synchronize()
    for x, w in zip(xs, wants):
        assert torch.equal(x["y"], w)
    first = eager["y"].clone()
    xs[0]["q"].copy_(eager["q"])
    for k in ("kv", "klen", "pos", "kmask", "gamma", "beta"):
        xs[0][k].copy_(eager[k])
    torch.cuda.synchronize()
    with torch.cuda.stream(streams[0]):
        graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(xs[0]["y"], first)
    for b in bes + [b3]:
        b.sync()
        b.close()


def test_first_call_of_a_process_may_be_captured():
    """Nothing that a call sets up once is refused during a capture."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    code = """
import sys, torch
sys.path.insert(0, %r)
import conftest
sb = conftest.load_product()
import test_gpu_prompt_ops as T
x = T.chain_inputs(5, torch.bfloat16, N=300, Nk=700)
b = sb.Backend(0)
s = torch.cuda.Stream()
b.set_stream(s.cuda_stream)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=s):
    T.chain(b, sb, x)
g.replay()
torch.cuda.synchronize()
y = x["y"].clone()
b.set_stream(1)
T.chain(b, sb, x)
b.sync()
assert torch.equal(x["y"], y) and y.float().abs().sum() > 0
""" % here
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_profile_names(be, sb):
    be.profile(True)
    chain(be, sb, chain_inputs(3, torch.bfloat16))
    table = be.profile_table()
    be.profile(False)
    assert {n: table[n]["calls"] for n in ("rope_table", "rope_rotate", "cross_attend", "groupnorm")} == \
        {"rope_table": 1, "rope_rotate": 2, "cross_attend": 1, "groupnorm": 1}
    assert all(table[n]["ms"] > 0 and table[n]["bytes"] > 0 for n in table)


def test_same_result_each_time(be, sb):
    """No result depends on the order CTAs run in."""
    x = chain_inputs(21, torch.bfloat16, nb=1, N=1, Nk=3000, h=8, hd=64)
    x["klen"] = torch.tensor([2900], device="cuda", dtype=torch.int32)
    chain(be, sb, x)
    be.sync()
    want = x["o"].clone(), x["y"].clone()
    for _ in range(20):
        chain(be, sb, x)
    be.sync()
    assert torch.equal(x["o"], want[0]) and torch.equal(x["y"], want[1])
