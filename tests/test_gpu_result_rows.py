"""GPU tests of products whose result is part of a wider matrix: rows that start at
multiples of 16 bytes and end anywhere. What lies behind a row's last column, and behind the last
row, keeps its bits, at every width and in every form of cb_gemm and cb_gemm_e4m3.

Tolerance of cb_gemm on bf16 operands: products are exact in 32 bits, their sum is off by
at most K 2^-23 of sum |a b| (the matrix unit may truncate each addition), bias and residual
add 2^-24 of theirs; the result is rounded once.
"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_block_ops import DT, E8M0, be, ceil, check_quantised, check_rounded, f64, gen, make_operand, op, product_ref, randn  # noqa: E402, F401

WIDTHS = (1, 3, 7, 15, 17, 100, 129, 209, 220, 223, 264)


def surroundings(n, dt, seed):
    """n elements of any bits: NaN, -0 and infinities among them."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    size = torch.empty(0, dtype=dt).element_size()
    return torch.randint(0, 256, (n * size,), device="cuda", generator=g, dtype=torch.uint8).view(dt)


def bits(t):
    return t.contiguous().view(torch.uint8)


class Matrix:
    """M x N at `off` of a buffer with pitch ld, the buffer given to the library up to its last element only."""

    def __init__(self, be, M, N, dt, pad, off, seed=0):
        step = 16 // torch.empty(0, dtype=dt).element_size()
        self.M, self.N, self.off = M, N, off * step
        self.ld = ceil(N, step) * step + pad * step
        self.all = surroundings(self.off + M * self.ld + 64, dt, seed)
        self.rows = self.all[self.off:self.off + M * self.ld].view(M, self.ld)
        self.given = self.all[:self.off + (M - 1) * self.ld + N]
        self.op = op(be, self.given, self.ld, 0, 0, self.off)

    def start(self):
        self.before = bits(self.all)

    def result(self):
        """The result, everything around it checked."""
        now, was = bits(self.all), self.before
        size = self.all.element_size()
        out = torch.ones(self.all.numel(), dtype=torch.bool, device="cuda")
        out[self.off:self.off + self.M * self.ld].view(self.M, self.ld)[:, :self.N] = False
        out = out.repeat_interleave(size)
        assert torch.equal(now[out], was[out])
        return self.rows[:, :self.N]


@pytest.mark.parametrize("pad", [0, 1])
@pytest.mark.parametrize("N", WIDTHS)
@pytest.mark.parametrize("M,dsa,dsb,out", [
    (1, "e8m0", "e8m0", "e4m3"), (3, "e8m0", "f32", "e4m3"), (3, "f32", "e8m0", "f32"), (8, "e8m0", "e8m0", "bf16"),
    (300, "e8m0", "e8m0", "bf16"), (531, "f32", "f32", "bf16"), (531, "e8m0", "e8m0", "f16"), (300, "e8m0", "e8m0", "e4m3"),
    (531, "e8m0", "e8m0", "f32"), (531, "f32", "f32", "e4m3"), (20000, "e8m0", "e8m0", "e4m3"), (20000, "f32", "e8m0", "f32")])
def test_gemm_e4m3_inside_a_matrix(be, sb, M, N, dsa, dsb, out, pad):
    K = 272
    g = gen(M + N)
    a, sa, av = make_operand(g, M, K, 1, dsa)
    b, s_b, bv = make_operand(g, N, K, 128, dsb, 0.0)
    bias = randn(g, N)
    c = Matrix(be, M, N, DT[out], pad, pad)
    sc = torch.zeros(M, ceil(N, 128), device="cuda").to(E8M0) if out == "e4m3" else None
    c.start()
    be.gemm_e4m3(M, N, K, op(be, a, a.shape[1]), op(be, sa, 3), op(be, b, b.shape[1]), op(be, s_b, 3), c.op,
                 None if sc is None else op(be, sc, ceil(N, 128)), be.wrap(bias), 2)
    z, tol = product_ref(av, bv, bias, "relu", out)
    got = c.result()
    if out == "e4m3":
        check_quantised(got, sc, z, tol)
    else:
        check_rounded(got, z, tol, DT[out])


def test_gemm_e4m3_pairs_inside_a_matrix(be, sb):
    """The form of CTA pairs: many rows, a long enough K."""
    for N, out in ((1001, "e4m3"), (1021, "bf16"), (515, "e4m3")):
        M, K = 20000, 1024
        g = gen(N)
        a, sa, av = make_operand(g, M, K, 1, "e8m0")
        b, s_b, bv = make_operand(g, N, K, 128, "e8m0", 0.0)
        c = Matrix(be, M, N, DT[out], 1, 0)
        sc = torch.zeros(M, ceil(N, 128), device="cuda").to(E8M0) if out == "e4m3" else None
        c.start()
        be.gemm_e4m3(M, N, K, op(be, a, K), op(be, sa, 8), op(be, b, K), op(be, s_b, 8), c.op, None if sc is None else op(be, sc, ceil(N, 128)))
        z, tol = product_ref(av, bv, None, "none", out)
        got = c.result()
        if out == "e4m3":
            check_quantised(got, sc, z, tol)
        else:
            check_rounded(got, z, tol, DT[out])


@pytest.mark.parametrize("how", ["bf16", "f32", "in place", "residual"])
@pytest.mark.parametrize("N", WIDTHS)
@pytest.mark.parametrize("M,K", [(1, 64), (300, 64), (20000, 136)])
def test_gemm_inside_a_matrix(be, sb, M, N, K, how):
    run_gemm(be, sb, M, N, K, how)


@pytest.mark.parametrize("how", ["bf16", "in place", "f32"])
def test_gemm_pairs_inside_a_matrix(be, sb, how):
    run_gemm(be, sb, 20000, 1021, 1032, how)


def run_gemm(be, sb, M, N, K, how):
    g = gen(M + N)
    dt = torch.bfloat16 if how == "bf16" else torch.float32
    a, b, bias = randn(g, M, K).bfloat16(), randn(g, N, K).bfloat16(), randn(g, N)
    c = Matrix(be, M, N, dt, 1, 1)
    other = Matrix(be, M, N, dt, 1, 1, 1) if how == "residual" else c
    if how in ("residual", "in place"):
        other.rows[:, :N] = randn(g, M, N)
    c.start()
    was = other.rows[:, :N].to(f64) if how in ("residual", "in place") else 0.0
    d = c.op
    be.gemm(M, N, K, (be.wrap(a), 0, K), (be.wrap(b), 0, K), 1, (be.wrap(c.given), d.off, d.ld), bias=be.wrap(bias),
            R=be.wrap(other.given) if how in ("residual", "in place") else None, roff=d.off)
    be.sync()
    av, bv = a.to(f64), b.to(f64)
    z = av @ bv.t() + bias.to(f64)
    tol = (K * 2.0 ** -23 + 2.0 ** -24) * (av.abs() @ bv.abs().t()) + 2.0 ** -24 * (z.abs() + bias.abs().to(f64))
    z = z + was
    check_rounded(c.result(), z, tol + 2.0 ** -24 * z.abs(), dt)
