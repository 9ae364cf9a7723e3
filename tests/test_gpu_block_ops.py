"""GPU tests of the operators around attention in a block (cb_quantize_e4m3,
cb_gemm_e4m3, cb_norm_residual, cb_rope_axes_table, cb_rope_rotate_axes) against
plain implementations in 64 bits on the same (already rounded) inputs.

Tolerances. u(T) is half a step of T relative to the value (2^-24 f32, 2^-8 bf16,
2^-11 f16, 2^-4 E4M3); every result is rounded to T once: u |y|, and below the
smallest normal number half the smallest step.
  quantiser: exact arithmetic, compared bit for bit;
  product: a block's 128 products are exact in 32 bits; their sum, which the
    matrix unit may truncate at each addition, is off by at most 128 * 2^-23 of
    A = sum |sa a sb b|, the scales' product by 2^-24, its product with the sum
    and the addition to the row's total by 2^-24 of at most A for each of the kb
    blocks: (128 * 2^-23 + (kb + 4) 2^-24) A; the bias adds 2^-24 |z|; GELU's
    slope is at most 1.13 and it is off by 4.2e-6 (32-bit results: 4 * 2^-24) of |z|;
  norm: sums of C values in chains of at most k = max(32, C / 1024) + 40, so a
    mean is off by k 2^-24 mean |v| and a sum of squares by k 2^-24 of itself; see
    norm_ref;
  rotation: two products and a sum in 32 bits, 4 * 2^-24 (|x0| + |x1|) |cs|.
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "e4m3": E4M3, "e8m0": E8M0}
f64 = torch.float64
INF, NAN = float("inf"), float("nan")


def u(dt):
    return torch.finfo(dt).eps / 2


def least(dt):
    """Half the smallest step of the type."""
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2


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


def op(be, t, ld=0, s0=0, s1=0, off=0):
    return be.bmat(be.wrap(t), off, ld, s0, s1)


def ceil(a, b):
    return -(-a // b)


# ------------------------------------------------------------------ quantiser
def quant_ref(x, brows):
    """x [rows, K] f64: (q f64 as E4M3 values, exponents int64 [blocks])."""
    n, k = x.shape
    e = torch.empty(ceil(n, brows), ceil(k, 128), dtype=torch.int64, device=x.device)
    q = torch.empty_like(x)
    fin = torch.where(torch.isfinite(x), x.abs(), 0.0)
    for j in range(e.shape[1]):
        c = slice(128 * j, 128 * j + 128)
        a = fin[:, c].amax(1)
        a = torch.nn.functional.pad(a, (0, -n % brows)).view(-1, brows).amax(1)
        # 448 * 2^e >= a, e the smallest such integer from -126 on
        m, ex = torch.frexp(a / 448.0)
        ee = torch.where(m == 0.5, ex - 1, ex).long()
        ee = torch.where(a > 0, ee, -126).clamp_min(-126)
        e[:, j] = ee
        s = torch.pow(torch.tensor(2.0, dtype=f64, device=x.device), ee.to(f64)).repeat_interleave(brows)[:n, None]
        q[:, c] = (x[:, c] / s).float().to(E4M3).to(f64)
    return q, e


def scale_bytes(s):
    return s.view(torch.uint8).long() - 127 if s.dtype == E8M0 else torch.frexp(s)[1].long() - 1


def same(a, b):
    """Equal, NaN at the same places."""
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))


@pytest.mark.parametrize("nb,N,K,brows,dt,ds,pad,xoff", [
    (1, 1, 1, 1, "f32", "e8m0", 0, 0),
    (1, 1, 128, 128, "bf16", "e8m0", 0, 0),
    (2, 3, 127, 1, "bf16", "e8m0", 1, 0),
    (3, 33, 129, 1, "f16", "f32", 7, 3),
    (2, 17, 1024, 1, "bf16", "e8m0", 8, 8),
    (1, 5, 136, 1, "f32", "e8m0", 8, 4),        # a block of one vector
    (2, 300, 520, 128, "f32", "e8m0", 0, 0),
    (2, 129, 257, 128, "bf16", "f32", 5, 1),
    (1, 1000, 4096, 1, "f16", "e8m0", 0, 0),
    (9, 128, 128, 128, "f16", "e8m0", 64, 16),
])
def test_quantize(be, sb, nb, N, K, brows, dt, ds, pad, xoff):
    g = gen(N * 7 + K)
    ld, kb, nr = K + pad, ceil(K, 128), ceil(N, brows)
    x = torch.zeros(xoff + nb * N * ld, device="cuda", dtype=DT[dt])
    xv = x[xoff:].view(nb, N, ld)
    v = randn(g, nb, N, K) * torch.exp2(torch.randint(-20, 14, (nb, N, 1), device="cuda", generator=g).float())
    xv[..., :K] = v.to(DT[dt])
    xv[..., K:] = 30000.0                        # behind the rows: not a part of any block
    if K >= 8:
        xv[0, 0, 3], xv[0, 0, 5], xv[0, 0, 7] = INF, -INF, NAN
        xv[-1, -1, :K] = 0.0
    q = torch.full((nb, N, K + 8), 0.75, device="cuda").to(E4M3)
    s = torch.zeros(nb, nr, kb + 1, device="cuda", dtype=torch.float32).to(DT[ds])
    be.quantize_e4m3(nb, N, K, brows, op(be, x, ld, N * ld, 0, xoff), op(be, q, K + 8, N * (K + 8)), op(be, s, kb + 1, nr * (kb + 1)))
    for b in range(nb):
        want, e = quant_ref(xv[b, :, :K].to(f64), brows)
        assert torch.equal(scale_bytes(s[b, :, :kb].contiguous()), e)
        assert same(q[b, :, :K].to(f64), want)
    assert (q[..., K:].float() == 0.75).all()


def test_quantize_borders(be, sb):
    """Largest magnitudes at and next to 448 * 2^e, the ends of the 32-bit range, halfway values."""
    rows = []
    for e in (-140, -126, -20, 0, 5, 119):
        for m in (447.99997, 448.0, 448.00003, 224.0, 1.0, 449.0, 864.0):
            if m * 2.0 ** e > 3.4e38:
                continue
            top = np.float32(m * 2.0 ** e)
            row = np.zeros(128, np.float32)
            row[0] = -top
            row[1:] = (np.arange(127, dtype=np.float64) * 0.0625 * float(top) / 448.0 * 33).astype(np.float32) % top if top > 0 else 0
            rows.append(row)
    rows.append(np.full(128, np.float32(3.4028235e38)))
    rows.append(np.full(128, np.float32(1e-45)))
    x = torch.tensor(np.stack(rows), device="cuda")
    n = x.shape[0]
    q, s = torch.empty(n, 128, device="cuda", dtype=E4M3), torch.empty(n, 1, device="cuda", dtype=E8M0)
    be.quantize_e4m3(1, n, 128, 1, op(be, x, 128), op(be, q, 128), op(be, s, 1))
    want, e = quant_ref(x.to(f64), 1)
    assert torch.equal(scale_bytes(s), e)
    assert same(q.to(f64), want)


# ------------------------------------------------------------------ product
def make_operand(g, rows, K, brows, ds, spread=0.5):
    """(padded E4M3 rows [rows, ld], scales, f64 values of the blocks' parts [rows, K], f64 scale per element)."""
    x = randn(g, rows, K) * torch.exp(spread * randn(g, K))
    q, e = quant_ref(x.to(f64), brows)
    if ds == "e8m0":
        s = (e + 127).to(torch.uint8).view(E8M0)
        sv = torch.exp2(e.to(f64))
    else:  # any numbers
        s = (torch.exp2(e.float()) * (0.5 + torch.rand(e.shape, device="cuda", generator=g))).contiguous()
        sv = s.to(f64)
    store = torch.full((rows, ceil(K, 16) * 16), 0x7f, dtype=torch.uint8, device="cuda")  # NaN behind the rows
    store[:, :K] = q.float().to(E4M3).view(torch.uint8)
    per = sv.repeat_interleave(brows, 0)[:rows].repeat_interleave(128, 1)[:, :K]
    return store.view(E4M3), s, q * per


def gelu64(z):
    return z * torch.special.ndtr(z)


def product_ref(a, b, bias, act, out):
    """z = act(a b^T + bias) and the bound of its 32-bit form before rounding to the output's type."""
    K = a.shape[1]
    z, big = a @ b.t(), a.abs() @ b.abs().t()
    tol = (128 * 2.0 ** -23 + (ceil(K, 128) + 4) * 2.0 ** -24) * big
    if bias is not None:
        z = z + bias.to(f64)
        tol = tol + 2.0 ** -24 * (z.abs() + big)
    if act == "gelu":
        tol = 1.13 * tol + (4 * 2.0 ** -24 if out == "f32" else 4.2e-6) * z.abs()
        z = gelu64(z)
    elif act == "relu":
        z = z.clamp_min(0.0)
    return z, tol


def check_rounded(got, z, tol, dt):
    err = (got.to(f64) - z).abs()
    lim = tol * (1 + u(dt)) + u(dt) * z.abs() + least(dt)
    assert (err <= lim).all(), float((err / lim).max())


def check_quantised(q, s, z, tol):
    """E4M3 rows and their scales against z known to within tol."""
    n, N = z.shape
    for j in range(ceil(N, 128)):
        c = slice(128 * j, 128 * j + 128)
        zc, tc = z[:, c], tol[:, c]
        hi, lo = (zc.abs() + tc).amax(1), (zc.abs() - tc).clamp_min(0).amax(1)
        sv = torch.exp2(scale_bytes(s[:, j].contiguous()).to(f64))
        assert (lo <= 448 * sv).all()
        assert ((hi > 224 * sv) | (sv == 2.0 ** -126)).all()
        err = (q[:, c].to(f64) * sv[:, None] - zc).abs()
        lim = tc * (1 + 2.0 ** -4) + 2.0 ** -4 * zc.abs() + 2.0 ** -10 * sv[:, None]
        assert (err <= lim).all(), float((err / lim).max())


def run_gemm(be, sb, M, N, K, dsa, dsb, out, act, use_bias, seed=0, ldc=None, off=0, dsc="e8m0"):
    g = gen(seed + M * 3 + N * 5 + K)
    a, sa, av = make_operand(g, M, K, 1, dsa)
    b, s_b, bv = make_operand(g, N, K, 128, dsb, 0.0)
    bias = randn(g, N) if use_bias else None
    ldc = N if ldc is None else ldc
    kb = ceil(K, 128)
    c = torch.full((off + M * ldc,), 3.0, device="cuda").to(DT[out])
    sc = torch.zeros(M, ceil(N, 128), device="cuda").to(DT[dsc]) if out == "e4m3" else None
    be.gemm_e4m3(M, N, K, op(be, a, a.shape[1]), op(be, sa, kb), op(be, b, b.shape[1]), op(be, s_b, kb), op(be, c, ldc, 0, 0, off),
                 None if sc is None else op(be, sc, ceil(N, 128)), None if bias is None else be.wrap(bias),
                 {"none": 0, "gelu": 1, "relu": 2}[act])
    z, tol = product_ref(av, bv, bias, act, out)
    got = c[off:].view(M, ldc)
    if out == "e4m3":
        check_quantised(got[:, :N], sc, z, tol)
    else:
        check_rounded(got[:, :N], z, tol, DT[out])
    assert (c[:off].float() == 3.0).all() and (got[:, N:].float() == 3.0).all()
    return c


@pytest.mark.parametrize("M,N,K,dsa,dsb,out,act,use_bias", [
    (1, 1, 1, "e8m0", "e8m0", "f32", "none", False),
    (1, 128, 128, "e8m0", "e8m0", "bf16", "none", False),
    (1, 4096, 1024, "e8m0", "f32", "bf16", "none", True),
    (8, 1024, 4096, "e8m0", "e8m0", "f16", "gelu", True),
    (3, 200, 100, "f32", "f32", "f32", "relu", True),
    (16, 257, 588, "e8m0", "e8m0", "bf16", "none", True),
    (17, 136, 1032, "f32", "e8m0", "f32", "gelu", True),
    (33, 1000, 300, "e8m0", "f32", "f16", "relu", False),
    (64, 64, 2048, "e8m0", "e8m0", "f32", "none", False),
    (5, 300, 700, "e8m0", "e8m0", "e4m3", "gelu", True),
    (128, 128, 128, "e8m0", "e8m0", "f32", "none", False),
    (129, 129, 129, "e8m0", "e8m0", "f32", "none", True),
    (200, 1000, 1176, "e8m0", "f32", "bf16", "gelu", True),
    (603, 520, 588, "f32", "f32", "f32", "none", True),
    (777, 1023, 1040, "e8m0", "e8m0", "e4m3", "gelu", True),
    (5184, 1024, 588, "e8m0", "e8m0", "f32", "none", True),
    (5184, 256, 256, "e8m0", "f32", "e4m3", "none", False),
    (5184, 2048, 256, "e8m0", "f32", "f16", "relu", True),
    (5185, 1111, 640, "e8m0", "e8m0", "bf16", "gelu", True),
    (2500, 4096, 1024, "e8m0", "e8m0", "e4m3", "gelu", True),
    (20000, 300, 4096, "e8m0", "e8m0", "bf16", "none", False),
    (250, 100, 1000, "f32", "f32", "f16", "gelu", True),     # few rows, in groups of 32
    (77, 2000, 33, "f32", "e8m0", "f32", "none", True),
    (250, 1500, 4096, "f32", "f32", "bf16", "none", True),   # the groups take k-blocks in turn
    (300, 1500, 700, "f32", "f32", "e4m3", "gelu", True),
    (20000, 140, 128, "f32", "f32", "f32", "none", True),
    (9000, 700, 1030, "e8m0", "f32", "e4m3", "relu", False),
    (128, 128, 1, "f32", "f32", "e4m3", "none", False),
])
def test_gemm(be, sb, M, N, K, dsa, dsb, out, act, use_bias):
    run_gemm(be, sb, M, N, K, dsa, dsb, out, act, use_bias)


@pytest.mark.parametrize("M", [4, 300])
@pytest.mark.parametrize("out,ldc,off", [("bf16", 331, 1), ("f16", 336, 8), ("f32", 333, 3), ("e4m3", 321, 5), ("e4m3", 336, 16)])
def test_gemm_any_result_layout(be, sb, M, out, ldc, off):
    run_gemm(be, sb, M, 320, 256, "e8m0", "e8m0", out, "none", True, ldc=ldc, off=off, dsc="f32")


# ------------------------------------------------------------------ norm
def norm64(v, dv, kind, g, b, eps, k):
    """The norm of v (known to within dv) in 64 bits and the bound of its 32-bit form."""
    if kind == 0:
        return v, dv
    C = v.shape[-1]
    e = 2.0 ** -24
    mean = v.mean(-1, keepdim=True) if kind == 1 else torch.zeros_like(v[..., :1])
    d = v - mean
    var = (d * d).mean(-1, keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    # the mean's own error; it enters each difference, and the variance by its square
    em = ((k * e * v.abs().mean(-1, keepdim=True) + dv.mean(-1, keepdim=True)) if kind == 1 else torch.zeros_like(var))
    rms = torch.sqrt(((dv + e * d.abs() + em) ** 2).mean(-1, keepdim=True))
    rel = (k + 8) * e + 1.01 * r * rms + (r * em) ** 2
    z = d * r
    dz = z.abs() * rel + r * (dv + em + e * d.abs()) * (1 + rel) + 2 * e * z.abs()
    gg = torch.ones(C, dtype=f64, device=v.device) if g is None else g.to(f64)
    y = z * gg + (0 if b is None else b.to(f64))
    return y, dz * gg.abs() + 2 * e * (z * gg).abs() + e * y.abs()


def norm_ref(x, h, post, alpha, ls, gate, pre, scale, shift, k):
    """x, h f64 [nb, N, C]; post, pre (kind, g, b, eps): r, y and their bounds."""
    e = 2.0 ** -24
    r, dr = x, torch.zeros_like(x)
    if h is not None:
        hh, dh = norm64(h, torch.zeros_like(h), *post, k)
        f = torch.full_like(x[..., :1], alpha)
        for t in (ls, gate):
            if t is not None:
                f = f * t.to(f64)
        r = x + f * hh
        dr = f.abs() * dh + 4 * e * (f * hh).abs() + e * r.abs()
    y, dy = norm64(r, dr, *pre, k)
    if scale is not None:
        s = 1 + scale.to(f64)
        dy = dy * s.abs() + 2 * e * (y.abs() + (y * s).abs())
        y = y * s
    if shift is not None:
        y = y + shift.to(f64)
        dy = dy + e * (y.abs() + shift.to(f64).abs())
    return r, dr, y, dy


CASES = [
    # nb, N, C, x, h, y, post, pre, gate, ls, mod, bias, alpha, pad
    (1, 1, 1, "f32", "f32", "f32", 0, 2, "none", False, False, False, 1.0, 0),
    (8, 1, 1024, "bf16", "bf16", "bf16", 0, 2, "none", False, False, False, 1.0, 0),
    (2, 5, 1024, "bf16", "bf16", "bf16", 0, 1, "sample", True, True, True, 1.0, 0),
    (3, 7, 1000, "f32", "f32", "e4m3", 2, 2, "none", False, False, False, 1.0, 0),
    (2, 9, 127, "f16", "f16", "f16", 1, 1, "row", True, True, True, 0.5, 1),
    (2, 3, 250, "f32", "bf16", "bf16", 1, 2, "sample", False, True, False, -1.25, 3),
    (1, 300, 512, "bf16", "bf16", "e4m3", 2, 1, "row", False, False, True, 1.0, 8),
    (5, 2, 264, "f16", "f16", "e4m3", 0, 1, "none", False, True, True, 1.0, 0),
    (2, 11, 2048, "f32", "f16", "f16", 1, 1, "row", True, False, True, 1.0, 0),
    (1, 6, 4096, "bf16", "bf16", "bf16", 2, 2, "sample", True, True, False, 1.0, 0),
    (2, 2, 4104, "f32", "f32", "e4m3", 1, 1, "none", True, True, True, 1.0, 0),
    (1, 3, 8192, "bf16", "bf16", "e4m3", 2, 2, "none", False, False, False, 1.0, 0),
    (1, 3, 8200, "f32", "f32", "f32", 1, 1, "row", True, True, True, 1.0, 0),
    (2, 2, 20001, "bf16", "bf16", "e4m3", 1, 2, "sample", True, True, True, 1.0, 7),
    (2, 700, 1024, "bf16", "bf16", "bf16", 0, 1, "sample", True, True, True, 1.0, 0),
    (3, 1801, 1000, "f32", "f32", "e4m3", 2, 2, "none", False, False, False, 1.0, 0),
    (2, 5184, 256, "bf16", "bf16", "e4m3", 1, 2, "sample", True, True, False, 1.0, 0),
    (1, 13, 64, "bf16", "bf16", "e4m3", 1, 1, "row", True, True, True, 1.0, 8),        # parts of a warp
    (3, 5001, 40, "f16", "f16", "e4m3", 1, 2, "sample", True, True, True, 1.0, 0),
    (7, 1003, 128, "f32", "bf16", "f16", 2, 1, "row", False, True, True, 1.0, 0),
    (2, 3003, 96, "bf16", "bf16", "bf16", 0, 1, "sample", True, True, True, 1.0, 8),
    (2, 3003, 77, "bf16", "bf16", "e4m3", 1, 1, "sample", True, True, True, 1.0, 0),   # rows that are not aligned
    (1, 3100, 333, "f32", "f16", "e4m3", 1, 2, "row", True, False, True, 1.0, 1),
    (2, 700, 1021, "f16", "f16", "e4m3", 2, 1, "sample", True, True, True, 1.0, 2),
    (1, 1300, 2047, "f32", "f32", "e4m3", 1, 1, "none", True, True, True, 1.0, 0),
    (2, 400, 5001, "bf16", "bf16", "bf16", 1, 1, "sample", True, True, True, 1.0, 0),
    (1, 20000, 1024, "bf16", "bf16", "e4m3", 2, 2, "row", True, False, False, 1.0, 0),
    (3, 300, 8192, "f16", "f16", "f16", 1, 1, "sample", True, True, True, 1.0, 0),
]


def run_norm(be, sb, nb, N, C, xt, ht, yt, post, pre, gate, ls, mod, bias, alpha, pad, seed=0, place="apart", offset=0.0):
    g = gen(seed + N + C)
    ld = C + pad

    def rows(dt, scale=1.0, mean=0.0):
        t = torch.full((nb, N, ld), 5.0, device="cuda")
        t[..., :C] = randn(g, nb, N, C) * scale + mean
        return t.to(DT[dt])

    def vec():
        return 1 + 0.3 * randn(g, C), (0.3 * randn(g, C) if bias else None)

    def opr(t):
        return op(be, t, ld, N * ld)
    x, h = rows(xt, 1.5, 0.2 + offset), rows(ht, 0.7, 0.1)
    x0, h0 = x.clone(), h.clone()
    params = {"post": vec() if post else (None, None), "pre": vec() if pre else (None, None)}
    lsv = 0.3 * randn(g, C) if ls else None
    m = 0.5 * randn(g, nb, 3 * C)
    gt = None
    go = None
    if gate == "sample":
        gt, go = m[:, None, :C], op(be, m, 0, 3 * C)
    elif gate == "row":
        gr = rows(ht, 0.5)
        gt, go = gr[..., :C].to(f64), opr(gr)
    sc, sh = (m[:, None, C : 2 * C], m[:, None, 2 * C :]) if mod else (None, None)
    r = x if place == "R=X" else (h if place == "R=H" else torch.full((nb, N, ld), 5.0, device="cuda").to(DT[xt]))
    y = x if place == "Y=X" else (h if place == "Y=H" else torch.full((nb, N, ld), 5.0, device="cuda").to(DT[yt]))
    s = torch.zeros(nb, N, ceil(C, 128), device="cuda").to(E8M0) if yt == "e4m3" else None

    def norm(kind, name, eps):
        w, b = params[name]
        return None if kind == 0 else sb.Norm(kind, eps, be.wrap(w), None if b is None else be.wrap(b))
    be.norm_residual(nb, N, C, opr(x), opr(h), norm(post, "post", 1e-5), alpha, None if lsv is None else be.wrap(lsv), go, opr(r),
                     norm(pre, "pre", 1e-3), op(be, m, 0, 3 * C, 0, C) if mod else None, op(be, m, 0, 3 * C, 0, 2 * C) if mod else None,
                     opr(y), None if s is None else op(be, s, ceil(C, 128), N * ceil(C, 128)))
    k = max(32, C / 1024) + 40
    rr, dr, yy, dy = norm_ref(x0[..., :C].to(f64), h0[..., :C].to(f64), (post, *params["post"], 1e-5), alpha, lsv, gt,
                              (pre, *params["pre"], 1e-3), sc, sh, k)
    check_rounded(r[..., :C], rr, dr, DT[xt])
    if yt == "e4m3":
        check_quantised(y[..., :C].reshape(nb * N, C), s.view(nb * N, -1), yy.view(nb * N, C), dy.view(nb * N, C))
    else:
        check_rounded(y[..., :C], yy, dy, DT[yt])
    if pad:
        for t in (r, y):
            assert (t[..., C:].float() == 5.0).all()
    return r, y


@pytest.mark.parametrize("case", CASES)
def test_norm_residual(be, sb, case):
    run_norm(be, sb, *case)


@pytest.mark.parametrize("place", ["R=X", "R=H", "Y=X", "Y=H"])
@pytest.mark.parametrize("C", [96, 1024, 3000, 9000])
def test_norm_residual_in_place(be, sb, place, C):
    run_norm(be, sb, 2, 5, C, "bf16", "bf16", "bf16", 1, 1, "sample", True, True, True, 1.0, 0, place=place)


# ------------------------------------------------------------------ rotary positions with several axes
def axis_of(widths, order):
    pairs = [w // 2 for w in widths]
    if order == 0:
        return [a for a, n in enumerate(pairs) for _ in range(n)]
    k = len(pairs)
    return [j % k if j // k < pairs[j % k] else 0 for j in range(sum(pairs))]


@pytest.mark.parametrize("widths,order", [((64,), 0), ((16, 24, 24), 0), ((24, 20, 20), 1), ((2, 2), 0), ((6, 2, 2, 2), 1), ((128, 64, 64), 0)])
def test_rope_axes_table(be, sb, widths, order):
    rot, npos, first = sum(widths), 301, -7
    cs = torch.full((npos * rot + 4,), 7.0, device="cuda")
    sc = sb.RopeScaling(theta=500000.0, kind=1, factor=2.0, amplitude=1.5)
    be.rope_axes_table(npos, sb.RopeAxes(widths, order), first, sc, be.wrap(cs))
    p = np.arange(first, first + npos).astype(np.longdouble)
    seen = [0] * len(widths)
    for j, a in enumerate(axis_of(widths, order)):
        w = np.longdouble(500000.0) ** (np.longdouble(-2 * seen[a]) / widths[a]) / 2
        seen[a] += 1
        want = np.stack([np.cos(p * w), np.sin(p * w)], -1) * 1.5
        got = cs[:npos * rot].view(npos, rot // 2, 2)[:, j].cpu().numpy().astype(np.float64)
        tol = 1.5 * (8 * 2.0 ** -24 + np.abs(p * w)[:, None] * 2.0 ** -52)
        assert (np.abs(got - want) <= tol).all()
    assert (cs[npos * rot:] == 7.0).all()


@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("nb,N,h,hd,widths,order,tx,ty,grid", [
    (1, 1, 1, 2, (2,), 0, "f32", "f32", None),
    (8, 1, 20, 64, (16, 24, 24), 0, "bf16", "bf16", None),
    (2, 60, 6, 64, (16, 24, 24), 0, "bf16", "bf16", (3, 4, 5)),
    (2, 33, 3, 80, (24, 18, 18), 1, "f32", "f32", None),
    (2, 31, 3, 80, (24, 18, 18), 1, "f16", "f16", (2, 4, 4)),
    (1, 65, 5, 72, (10, 6), 0, "bf16", "bf16", None),
    (3, 9, 4, 128, (32, 32, 32, 32), 1, "f32", "bf16", (1, 3, 1, 3)),
    (2, 9, 4, 96, (64, 32), 0, "f32", "f16", (3, 3)),
    (1, 3000, 33, 128, (44, 42, 42), 0, "f16", "f16", (10, 20, 15)),
    (2, 50, 3, 256, (128, 64, 64), 0, "bf16", "bf16", (2, 5, 5)),
])
def test_rope_rotate_axes(be, sb, nb, N, h, hd, widths, order, tx, ty, grid, halves):
    g = gen(N + h + hd)
    rot, npos, pad, tail, axes = sum(widths), 17, 8, 16, len(widths)
    ld = h * hd + pad
    x = randn(g, nb, N, ld).to(DT[tx])
    x[0, 0, 0] = INF
    y = torch.full((nb * N * h * hd + tail,), 3.0, device="cuda", dtype=DT[ty])
    ang = torch.rand(npos, rot // 2, device="cuda", generator=g, dtype=f64) * 6.3
    cs = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()
    if grid is None:
        pos = torch.randint(-2, npos + 2, (nb, N, axes), device="cuda", generator=g, dtype=torch.int32)
        pos[0, 0] = -1                             # the row with an infinity is left as it is
    else:
        n = torch.arange(N, device="cuda")
        p = [n // math.prod(grid[a + 1:]) % grid[a] for a in range(axes)]
        pos = torch.stack(p, -1)[None].expand(nb, N, axes)
        x[0, 0, 0] = 1.0
    be.rope_rotate_axes(nb, N, h, hd, rot, int(halves), sb.RopeAxes(widths, order), op(be, x, ld, N * ld, hd), op(be, y, h * hd, N * h * hd, hd),
                        be.wrap(cs), npos, None if grid else be.wrap(pos), grid)
    xv = x[..., :h * hd].reshape(nb, N, h, hd).to(f64)
    want, lim = xv.clone(), torch.zeros_like(xv)
    for j, a in enumerate(axis_of(widths, order)):
        at = pos[..., a].long()
        keep = ((at >= 0) & (at < npos))[..., None]
        t = cs[at.clamp(0, npos - 1), j].to(f64)
        c, s = t[..., 0][..., None], t[..., 1][..., None]
        i0, i1 = (j, rot // 2 + j) if halves else (2 * j, 2 * j + 1)
        p, q = xv[..., i0], xv[..., i1]
        want[..., i0] = torch.where(keep, p * c - q * s, p)
        want[..., i1] = torch.where(keep, p * s + q * c, q)
        m = torch.where(keep, 4 * 2.0 ** -24 * (p.abs() + q.abs()) * torch.maximum(c.abs(), s.abs()), 0.0)
        lim[..., i0] = lim[..., i1] = m
    got = y[:nb * N * h * hd].view(nb, N, h, hd).to(f64)
    fin = torch.isfinite(want)
    assert torch.equal(got[~fin], want[~fin])
    err = (got - want).abs()[fin]
    bound = (lim + (0.0 if tx == ty else 1.0) * u(DT[ty]) * want.abs() + u(DT[ty]) * want.abs() + least(DT[ty]))[fin]
    assert (err <= bound).all(), float((err / bound).max())
    assert (y[nb * N * h * hd:] == 3.0).all()
