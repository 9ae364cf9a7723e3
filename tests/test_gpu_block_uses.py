"""GPU tests of the operators around attention in a block as they are used: a block
of their calls in a row, captured and replayed, on several streams and from several
threads; values that are not finite, scales at the ends of their range, operands
far into a buffer, results that do not depend on the run. Tolerances as in
test_gpu_block_ops.py."""
import math
import os

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
from test_gpu_block_ops import (E4M3, E8M0, DT, INF, NAN, be, ceil, check_quantised, check_rounded, f64, gelu64, gen,  # noqa: E402,F401
                                make_operand, norm_ref, op, product_ref, quant_ref, randn, same, scale_bytes)


# ------------------------------------------------------------------ a block
def block_inputs(seed, nb=2, grid=(2, 8, 15), E=256, heads=4, mlp=512, dsb="e8m0"):
    g = gen(seed)
    N = math.prod(grid)
    x = dict(nb=nb, N=N, E=E, heads=heads, mlp=mlp, grid=grid, rows=nb * N)
    new = lambda *s, dt=torch.bfloat16: torch.zeros(*s, device="cuda").to(dt)  # noqa: E731
    x["x"] = randn(g, nb, N, E).to(torch.bfloat16)
    x["mod"] = 0.3 * randn(g, nb, 6 * E)                      # shift, scale, gate of both halves
    x["ls"] = 0.5 + 0.1 * randn(g, E)
    x["g1"], x["g2"], x["gp"] = (1 + 0.1 * randn(g, E) for _ in range(3))
    for name, n, k in (("wqkv", 3 * E, E), ("wo", E, E), ("w1", mlp, E), ("w2", E, mlp)):
        w, s, v = make_operand(g, n, k, 128, dsb if name != "w2" else "f32", 0.0)
        x[name], x[name + "s"], x[name + "v"] = w, s, v
        x[name + "b"] = 0.1 * randn(g, n)
    ang = torch.arange(64, device="cuda", dtype=f64)[:, None] * 10000.0 ** (-torch.arange(32, device="cuda", dtype=f64) / 32)
    x["cs"] = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()
    r = x["rows"]
    x["q1"], x["s1"] = new(r, E, dt=E4M3), new(r, ceil(E, 128), dt=E8M0)
    x["qkv"], x["qk"], x["att"] = new(r, 3 * E), new(r, 2 * E), new(r, E)
    x["qa"], x["sa"] = new(r, E, dt=E4M3), new(r, ceil(E, 128), dt=E8M0)
    x["po"], x["r1"] = new(r, E), new(nb, N, E)
    x["q2"], x["s2"] = new(r, E, dt=E4M3), new(r, ceil(E, 128), dt=E8M0)
    x["qh"], x["sh"] = new(r, mlp, dt=E4M3), new(r, ceil(mlp, 128), dt=E8M0)
    x["mo"], x["r2"] = new(r, E), new(nb, N, E)
    return x


def run_block(b, sb, x):
    nb, N, E, h, mlp, r = (x[k] for k in ("nb", "N", "E", "heads", "mlp", "rows"))
    kE, kM = ceil(E, 128), ceil(mlp, 128)

    def rows(t, w, wd=None):
        return op(b, t, wd or w, N * (wd or w))

    def mod(i):
        return op(b, x["mod"], 0, 6 * E, 0, i * E)

    def mat(name, w):
        return op(b, x[name], w)
    rms = lambda name: sb.Norm(sb.NORM_RMS, 1e-6, b.wrap(x[name]))  # noqa: E731
    b.norm_residual(nb, N, E, rows(x["x"], E), pre=rms("g1"), scale=mod(1), shift=mod(0), Y=rows(x["q1"], E), S=rows(x["s1"], kE))
    b.gemm_e4m3(r, 3 * E, E, mat("q1", E), mat("s1", kE), mat("wqkv", E), mat("wqkvs", kE), mat("qkv", 3 * E), None, b.wrap(x["wqkvb"]))
    hd = E // h
    b.rope_rotate_axes(x["nb"], N, 2 * h, hd, hd, sb.ROPE_HALVES, sb.RopeAxes((16, 24, 24)), op(b, x["qkv"], 3 * E, N * 3 * E, hd),
                       op(b, x["qk"], 2 * E, N * 2 * E, hd), b.wrap(x["cs"]), 64, None, x["grid"])
    b.cross_attend(nb, N, N, h, h, hd, op(b, x["qk"], 2 * E, N * 2 * E, hd), op(b, x["qk"], 2 * E, N * 2 * E, hd, E),
                   op(b, x["qkv"], 3 * E, N * 3 * E, hd, 2 * E), op(b, x["att"], E, N * E, hd))
    b.quantize_e4m3(1, r, E, 1, mat("att", E), mat("qa", E), mat("sa", kE))
    b.gemm_e4m3(r, E, E, mat("qa", E), mat("sa", kE), mat("wo", E), mat("wos", kE), mat("po", E), None, b.wrap(x["wob"]))
    b.norm_residual(nb, N, E, rows(x["x"], E), rows(x["po"], E), rms("gp"), 1.0, b.wrap(x["ls"]), mod(2), rows(x["r1"], E), rms("g2"),
                    mod(4), mod(3), rows(x["q2"], E), rows(x["s2"], kE))
    b.gemm_e4m3(r, mlp, E, mat("q2", E), mat("s2", kE), mat("w1", E), mat("w1s", kE), mat("qh", mlp), mat("sh", kM), b.wrap(x["w1b"]),
                sb.ACT_GELU)
    b.gemm_e4m3(r, E, mlp, mat("qh", mlp), mat("sh", kM), mat("w2", mlp), mat("w2s", kM), mat("mo", E), None, b.wrap(x["w2b"]))
    b.norm_residual(nb, N, E, rows(x["r1"], E), rows(x["mo"], E), None, 1.0, None, mod(5), rows(x["r2"], E))


OUTS = ("q1", "s1", "qkv", "qk", "att", "qa", "sa", "po", "r1", "q2", "s2", "qh", "sh", "mo", "r2")


def bits(x):
    return [x[k].view(torch.uint8).clone() for k in OUTS]


def values(q, s, K):
    return q.to(f64) * torch.exp2(scale_bytes(s).to(f64)).repeat_interleave(128, 1)[:, :K]


@pytest.mark.parametrize("kw", [dict(), dict(nb=1, grid=(1, 1, 1)), dict(nb=3, grid=(3, 19, 23)), dict(dsb="f32", grid=(2, 9, 9))])
def test_block(be, sb, kw):
    """Every step against 64 bits on what the step before left."""
    x = block_inputs(3, **kw)
    run_block(be, sb, x)
    be.sync()
    nb, N, E, h, mlp, r = (x[k] for k in ("nb", "N", "E", "heads", "mlp", "rows"))
    m = x["mod"].to(f64).view(nb, 1, 6, E)
    k = 72
    xs = x["x"].to(f64)
    _, _, y, dy = norm_ref(xs, None, None, 1.0, None, None, (2, x["g1"], None, 1e-6), m[:, :, 1], m[:, :, 0], k)
    check_quantised(x["q1"], x["s1"], y.view(r, E), dy.view(r, E))
    z, tol = product_ref(values(x["q1"], x["s1"], E), x["wqkvv"], x["wqkvb"], "none", "bf16")
    check_rounded(x["qkv"], z, tol, torch.bfloat16)
    hd = E // h
    n = torch.arange(N, device="cuda")
    gr = x["grid"]
    pos = torch.stack([n // (gr[1] * gr[2]), n // gr[2] % gr[1], n % gr[2]], -1)
    axis = torch.tensor([0] * 8 + [1] * 12 + [2] * 12, device="cuda")
    t = x["cs"].to(f64)[pos[:, axis], torch.arange(hd // 2, device="cuda")]
    qk = x["qkv"].to(f64).view(nb, N, 3 * h, hd)[:, :, :2 * h]
    c, s = t[..., 0][None, :, None], t[..., 1][None, :, None]
    a, b = qk[..., :hd // 2], qk[..., hd // 2:]
    want = torch.cat([a * c - b * s, a * s + b * c], -1).view(r, 2 * E)
    big = torch.cat([a.abs() + b.abs()] * 2, -1).reshape(r, 2 * E)
    check_rounded(x["qk"], want, 4 * 2.0 ** -24 * big, torch.bfloat16)
    q, e = quant_ref(x["att"].to(f64), 1)
    assert same(x["qa"].to(f64), q) and torch.equal(scale_bytes(x["sa"]), e)
    z, tol = product_ref(values(x["qa"], x["sa"], E), x["wov"], x["wob"], "none", "bf16")
    check_rounded(x["po"], z, tol, torch.bfloat16)
    rr, dr, y, dy = norm_ref(xs, x["po"].to(f64).view(nb, N, E), (2, x["gp"], None, 1e-6), 1.0, x["ls"], m[:, :, 2], (2, x["g2"], None, 1e-6),
                             m[:, :, 4], m[:, :, 3], k)
    check_rounded(x["r1"], rr, dr, torch.bfloat16)
    check_quantised(x["q2"], x["s2"], y.view(r, E), dy.view(r, E))
    z, tol = product_ref(values(x["q2"], x["s2"], E), x["w1v"], x["w1b"], "gelu", "e4m3")
    check_quantised(x["qh"], x["sh"], z, tol)
    z, tol = product_ref(values(x["qh"], x["sh"], mlp), x["w2v"], x["w2b"], "none", "bf16")
    check_rounded(x["mo"], z, tol, torch.bfloat16)
    rr, dr, _, _ = norm_ref(x["r1"].to(f64), x["mo"].to(f64).view(nb, N, E), (0, None, None, 0.0), 1.0, None, m[:, :, 5], (0, None, None, 0.0),
                            None, None, k)
    check_rounded(x["r2"], rr, dr, torch.bfloat16)


def test_block_captured_and_replayed(sb):
    """Two captured blocks on their own buffers, replayed at the same time, and again after new inputs were copied in."""
    xs = [block_inputs(5), block_inputs(6, grid=(2, 20, 30))]
    graphs, backends = [], []
    for x in xs:
        b = sb.Backend(0)
        s = torch.cuda.Stream()
        b.set_stream(s.cuda_stream)
        run_block(b, sb, x)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            run_block(b, sb, x)
        graphs.append((g, s))
        backends.append(b)
    for seed in (0, 1):
        want = []
        for i, x in enumerate(xs):
            x["x"].copy_(block_inputs(50 + 2 * seed + i, grid=x["grid"])["x"])
            torch.cuda.synchronize()
            run_block(backends[i], sb, x)
            torch.cuda.synchronize()
            want.append(bits(x))
            for k in OUTS:
                x[k].view(torch.uint8).zero_()
        torch.cuda.synchronize()
        for _ in range(5):
            for g, s in graphs:
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for x, w in zip(xs, want):
            assert all(torch.equal(a, b) for a, b in zip(bits(x), w))
    del graphs
    for b in backends:
        b.sync()
        b.close()


def test_first_call_of_a_process_may_be_captured():
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    code = """
import sys, torch
sys.path.insert(0, %r)
import conftest
sb = conftest.load_product()
import test_gpu_block_uses as T
x = T.block_inputs(5, nb=4, grid=(2, 40, 40))
b = sb.Backend(0)
s = torch.cuda.Stream()
b.set_stream(s.cuda_stream)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=s):
    T.run_block(b, sb, x)
g.replay()
torch.cuda.synchronize()
y = T.bits(x)
b.set_stream(1)
T.run_block(b, sb, x)
b.sync()
assert all(torch.equal(p, q) for p, q in zip(y, T.bits(x))) and x["r2"].float().abs().sum() > 0
""" % here
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_threads_of_their_own(sb):
    """Two host threads, a backend each, at once: what each leaves alone, bit for bit."""
    import threading
    xs = [block_inputs(11, grid=(2, 16, 30)), block_inputs(12, nb=1, grid=(1, 25, 33), dsb="f32")]
    want = []
    for x in xs:
        b = sb.Backend(0)
        run_block(b, sb, x)
        b.sync()
        b.close()
        want.append(bits(x))
        for k in OUTS:
            x[k].view(torch.uint8).zero_()
    torch.cuda.synchronize()
    errors = []

    def work(x):
        try:
            b = sb.Backend(0)
            for _ in range(10):
                run_block(b, sb, x)
            b.sync()
            b.close()
        except Exception as e:  # noqa: BLE001
            errors.append(e)
    ts = [threading.Thread(target=work, args=(x,)) for x in xs]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not errors
    for x, w in zip(xs, want):
        assert all(torch.equal(a, b) for a, b in zip(bits(x), w))


def test_same_result_each_time(be, sb):
    for kw in (dict(nb=1, grid=(1, 1, 5)), dict(nb=4, grid=(2, 30, 31))):
        x = block_inputs(21, **kw)
        run_block(be, sb, x)
        be.sync()
        want = bits(x)
        for _ in range(20):
            run_block(be, sb, x)
        be.sync()
        assert all(torch.equal(a, b) for a, b in zip(bits(x), want))


def test_profile_names(be, sb):
    be.profile(True)
    run_block(be, sb, block_inputs(3))
    table = be.profile_table()
    be.profile(False)
    want = {"norm_residual": 3, "gemm_e4m3": 4, "quantize_e4m3": 1, "rope_rotate_axes": 1}
    assert {n: table[n]["calls"] for n in want} == want
    assert all(table[n]["ms"] > 0 and table[n]["bytes"] > 0 for n in want)


# ------------------------------------------------------------------ products at the ends
FORMS = [(5, "e8m0", "e8m0", "bf16"), (5, "f32", "e8m0", "f32"), (300, "e8m0", "e8m0", "bf16"), (300, "e8m0", "e8m0", "e4m3"),
         (5000, "e8m0", "e8m0", "f16"), (300, "f32", "f32", "bf16"), (300, "e8m0", "e8m0", "f32"), (6000, "f32", "f32", "e4m3")]


def product(be, M, N, K, a, sa, b, s_b, out, act=0, bias=None):
    c = torch.zeros(M, N, device="cuda").to(DT[out])
    sc = torch.zeros(M, ceil(N, 128), device="cuda").to(E8M0) if out == "e4m3" else None
    be.gemm_e4m3(M, N, K, op(be, a, a.shape[1]), op(be, sa, sa.shape[1]), op(be, b, b.shape[1]), op(be, s_b, s_b.shape[1]), op(be, c, N),
                 None if sc is None else op(be, sc, ceil(N, 128)), None if bias is None else be.wrap(bias), act)
    return c, sc


@pytest.mark.parametrize("M,dsa,dsb,out", FORMS)
def test_gemm_not_a_number_stays_in_its_row(be, sb, M, dsa, dsb, out):
    """A NaN among A's values or scales shows in its row, one among B's in its column or columns, and nowhere else."""
    N, K = 520, 400
    g = gen(M)
    a, sa, _ = make_operand(g, M, K, 1, dsa)
    b, s_b, _ = make_operand(g, N, K, 128, dsb, 0.0)
    clean, csc = product(be, M, N, K, a, sa, b, s_b, out)

    def poison(t, *at):
        t = t.clone()
        t.view(torch.uint8 if t.element_size() == 1 else torch.int32)[at] = (0xff if t.dtype == E8M0 else 0x7f) if t.element_size() == 1 else 0x7fc00000
        return t
    for which, at, rows, cols in (("a", (3, 130), slice(3, 4), slice(None)), ("sa", (4, 3), slice(4, 5), slice(None)),
                                  ("b", (200, 399), slice(None), slice(200, 201)), ("sb", (4, 0), slice(None), slice(512, 520))):
        t = dict(a=a, sa=sa, b=b, sb=s_b)
        t[which] = poison(t[which], *at)
        got, gsc = product(be, M, N, K, t["a"], t["sa"], t["b"], t["sb"], out)
        bad = torch.zeros(M, N, dtype=torch.bool, device="cuda")
        bad[rows, cols] = True
        assert torch.equal(torch.isnan(got.float()), bad), which
        if out == "e4m3":   # the others' scales may change with what is left of the block
            for j in range(ceil(N, 128)):
                keep = ~bad[:, 128 * j:128 * j + 128].any(1)
                assert torch.equal(got.view(torch.uint8)[keep, 128 * j:128 * j + 128], clean.view(torch.uint8)[keep, 128 * j:128 * j + 128])
        else:
            assert torch.equal(got[~bad], clean[~bad]), which


@pytest.mark.parametrize("M,dsa,dsb,out", FORMS)
def test_gemm_scales_of_any_size(be, sb, M, dsa, dsb, out):
    """Scales from 2^-100 to 2^60 (their products within 32 bits), one of zero and one negative where they are numbers."""
    N, K = 264, 384
    g = gen(M + 1)
    a, sa, _ = make_operand(g, M, K, 1, dsa)
    b, s_b, _ = make_operand(g, N, K, 128, dsb, 0.0)

    def resize(s, lo, hi):
        e = torch.randint(lo, hi, s.shape, device="cuda", generator=g)
        if s.dtype == E8M0:
            return (e + 127).to(torch.uint8).view(E8M0)
        return torch.exp2(e.float()) * (0.5 + torch.rand(s.shape, device="cuda", generator=g))
    big = out == "f16"      # its range is 2^16
    sa, s_b = resize(sa, -6 if big else -100, -3 if big else 60), resize(s_b, -6 if big else -20, -3 if big else 20)
    if dsa == "f32":
        sa[0, 0], sa[1, 1] = 0.0, -sa[1, 1]
    values = lambda q, s, rows, br: q[:, :K].to(f64) * s.to(f64).repeat_interleave(br, 0)[:rows].repeat_interleave(128, 1)[:, :K]  # noqa: E731
    av, bv = values(a, sa, M, 1), values(b, s_b, N, 128)
    z, tol = product_ref(av, bv, None, "none", out)
    got, gsc = product(be, M, N, K, a, sa, b, s_b, out)
    if out == "e4m3":
        check_quantised(got, gsc, z, tol)
    else:
        # (a sum's largest parts decide: below 2^-126 nothing is asked)
        check_rounded(got, z, tol + 2.0 ** -126, DT[out])


@pytest.mark.parametrize("M,dsa,dsb,out", FORMS)
def test_gemm_strided_scales_and_infinite_sums(be, sb, M, dsa, dsb, out):
    N, K = 140, 300
    g = gen(M + 2)
    a, sa, av = make_operand(g, M, K, 1, dsa)
    b, s_b, bv = make_operand(g, N, K, 128, dsb, 0.0)
    kb = ceil(K, 128)

    def wide(s, pad, off):
        t = torch.zeros(off + s.shape[0] * (kb + pad), device="cuda", dtype=s.dtype if s.dtype == torch.float32 else torch.uint8)
        v = t[off:].view(s.shape[0], kb + pad)
        v[:, :kb] = s if s.dtype == torch.float32 else s.view(torch.uint8)
        return t if s.dtype == torch.float32 else t.view(E8M0)
    bias = torch.zeros(N, device="cuda")
    bias[7], bias[9] = INF, -INF
    for pad, off in ((5, 3), (1, 4), (5, 0)):
        c = torch.zeros(M, N, device="cuda").to(DT[out])
        sc = torch.zeros(M, 5, device="cuda").to(E8M0)
        be.gemm_e4m3(M, N, K, op(be, a, a.shape[1]), op(be, wide(sa, pad, off), kb + pad, 0, 0, off), op(be, b, b.shape[1]),
                     op(be, wide(s_b, pad, off), kb + pad, 0, 0, off), op(be, c, N), op(be, sc, 5) if out == "e4m3" else None, be.wrap(bias))
        z, tol = product_ref(av, bv, None, "none", out)
        keep = torch.ones(N, dtype=torch.bool, device="cuda")
        keep[7] = keep[9] = False
        if out == "e4m3":  # NaN, and the block's scale from its finite values
            assert torch.isnan(c.float()[:, ~keep]).all() and not torch.isnan(c.float()[:, keep]).any()
            z, tol, cc = z.clone(), tol.clone(), c.float().clone()
            z[:, ~keep], tol[:, ~keep], cc[:, ~keep] = 0.0, 0.0, 0.0
            check_quantised(cc.to(E4M3), sc[:, :2].contiguous(), z, tol)
        else:
            assert (c[:, 7] == INF).all() and (c[:, 9] == -INF).all()
            check_rounded(c[:, keep], z[:, keep], tol[:, keep], DT[out])


@pytest.mark.parametrize("out", ["bf16", "f16", "e4m3", "f32"])
@pytest.mark.parametrize("M", [4, 400])
def test_gemm_gelu_over_its_range(be, sb, out, M):
    """GELU of sums from -40 to 40, with 32-bit sums known exactly: A picks one column of B."""
    N, K = 256, 128
    x = torch.linspace(-40, 40, M * N, device="cuda").view(M, N)
    a = torch.zeros(M, K, device="cuda").to(E4M3)
    sa, s_b = torch.full((M, 1), 1.0, device="cuda"), torch.full((2, 1), 1.0, device="cuda")
    b = torch.zeros(N, K, device="cuda").to(E4M3)
    for m in (0, M - 1):
        c, sc = product(be, M, N, K, a, sa.to(E8M0), b, s_b.to(E8M0), out, 1, x[m].contiguous())
        z = x[m].to(f64)[None].expand(M, N)
        y = gelu64(z)
        if out == "e4m3":
            check_quantised(c, sc, y, 1.2e-5 * y.abs() + 6e-15)
        else:
            # 16 bits: the polynomial's 1.2e-5 of h, x h as much; 32 bits: 1 + erf rounds to 2^-24
            tol = 1.2e-5 * torch.minimum(y.abs(), z.abs() * torch.special.ndtr(-z.abs())) + 2 * 2.0 ** -24 * z.abs() + 6e-15
            if out == "f32":
                tol = 4 * 2.0 ** -24 * z.abs()
            check_rounded(c, y, tol, DT[out])


# ------------------------------------------------------------------ norms at the ends
@pytest.mark.parametrize("nb,N,C,dt", [(1, 7, 100, "f32"), (2, 9, 1024, "bf16"), (1, 3000, 1024, "bf16"), (1, 1300, 333, "f16"), (2, 5, 9000, "f32")])
def test_norm_rows_of_their_own(be, sb, nb, N, C, dt):
    """A row of zeros, one with a NaN, one with an infinity: the others as without them, zeros where the weight of zeros is taken."""
    g = gen(C)
    x = randn(g, nb, N, C).to(DT[dt])
    h = randn(g, nb, N, C).to(DT[dt])

    def call(x, h, kind):
        r, y = torch.empty_like(x), torch.empty_like(x)
        be.norm_residual(nb, N, C, op(be, x, C, N * C), op(be, h, C, N * C), sb.Norm(kind, 1e-5), 1.0, None, None, op(be, r, C, N * C),
                         sb.Norm(kind, 1e-5), None, None, op(be, y, C, N * C))
        return r, y
    for kind in (sb.NORM_LAYER, sb.NORM_RMS):
        r0, y0 = call(x, h, kind)
        x1, h1 = x.clone(), h.clone()
        x1[0, 1], h1[0, 1] = 0.0, 0.0
        x1[0, 2, C // 2] = NAN
        h1[0, 4, C - 1] = INF
        r1, y1 = call(x1, h1, kind)
        keep = torch.ones(nb, N, dtype=torch.bool, device="cuda")
        keep[0, 1] = keep[0, 2] = keep[0, 4] = False
        assert torch.equal(r0[keep], r1[keep]) and torch.equal(y0[keep], y1[keep])
        assert (r1[0, 1] == 0).all() and (y1[0, 1] == 0).all()
        assert torch.isnan(y1[0, 2]).all() and torch.isnan(r1[0, 2]).sum() == 1
        assert torch.isnan(r1[0, 4, C - 1]) and torch.isnan(y1[0, 4]).all()


def test_norm_mean_far_from_zero(be, sb):
    """Variance 1 around 1000: what E[x^2] - E[x]^2 would lose."""
    from test_gpu_block_ops import run_norm
    for C in (512, 1024, 4096, 9000):
        run_norm(be, sb, 2, 3, C, "f32", "f32", "f32", 1, 1, "none", False, False, True, 1.0, 0, offset=1000.0)


# ------------------------------------------------------------------ far into a buffer
def test_operands_far_into_a_buffer(be, sb):
    """Elements behind 2^31 of their buffers."""
    far = (1 << 31) + 64
    g = gen(9)
    big = torch.zeros(far + 3000, device="cuda", dtype=torch.bfloat16)
    K = 1000
    v = randn(g, 2, K).to(torch.bfloat16)
    big[:K], big[far:far + K] = v[0], v[1]
    q, s = torch.zeros(2, 1008, device="cuda").to(E4M3), torch.zeros(2, 8, device="cuda").to(E8M0)
    be.quantize_e4m3(2, 1, K, 1, op(be, big, K, far), op(be, q, 1008, 1008), op(be, s, 8, 8))
    want, e = quant_ref(v.to(f64), 1)
    assert same(q[:, :K].to(f64), want) and torch.equal(scale_bytes(s), e)
    # the norm reads a row and writes behind it; two rows so far apart in one call
    rr, dr, y, dy = norm_ref(v.to(f64)[:, None], None, None, 1.0, None, None, (2, None, None, 1e-6), None, None, 72)
    r, yy = torch.zeros(2, K, device="cuda", dtype=torch.bfloat16), torch.zeros(2, K, device="cuda", dtype=torch.bfloat16)
    be.norm_residual(2, 1, K, op(be, big, K, far), R=op(be, r, K, K), pre=sb.Norm(sb.NORM_RMS, 1e-6), Y=op(be, yy, K, K))
    assert torch.equal(r, v)
    check_rounded(yy, y[:, 0], dy[:, 0], torch.bfloat16)
    be.norm_residual(1, 1, K, op(be, big, K, K, 0, far), pre=sb.Norm(sb.NORM_RMS, 1e-6), Y=op(be, big, K, K, 0, far + 1000))
    assert torch.equal(big[far + 1000:far + 2000], yy[1]) and torch.equal(big[far:far + K], v[1])
    # rotation
    cs = torch.stack([torch.zeros(8, 32), torch.ones(8, 32)], -1).cuda().contiguous()
    o = torch.zeros(2, 128, device="cuda", dtype=torch.bfloat16)
    pos = torch.full((2, 1, 2), 3, device="cuda", dtype=torch.int32)
    be.rope_rotate_axes(2, 1, 2, 64, 64, sb.ROPE_HALVES, sb.RopeAxes((32, 32)), op(be, big, 128, far, 64), op(be, o, 128, 128, 64), be.wrap(cs), 8,
                        be.wrap(pos))
    w = v[:, :128].view(2, 2, 64)
    assert torch.equal(o.view(2, 2, 64), torch.cat([-w[..., 32:], w[..., :32]], -1))
    del big
    # a product whose result passes 2^31 elements, in rows far apart
    M, N, ld = 70000, 130, 32768
    a, sa, av = make_operand(g, M, 256, 1, "e8m0")
    b, s_b, bv = make_operand(g, N, 256, 128, "e8m0", 0.0)
    for dt in ("bf16", "e4m3"):
        c = torch.zeros(M * ld, device="cuda", dtype=torch.uint8 if dt == "e4m3" else DT[dt])
        c = c.view(E4M3) if dt == "e4m3" else c
        sc = torch.zeros(M, 2, device="cuda").to(E8M0)
        be.gemm_e4m3(M, N, 256, op(be, a, 256), op(be, sa, 2), op(be, b, 256), op(be, s_b, 2), op(be, c, ld),
                     op(be, sc, 2) if dt == "e4m3" else None)
        z, tol = product_ref(av, bv, None, "none", dt)
        got = c.view(M, ld)[:, :N]
        if dt == "e4m3":
            check_quantised(got.contiguous(), sc, z, tol)
        else:
            check_rounded(got, z, tol, DT[dt])
        del c, got
