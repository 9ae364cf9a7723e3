"""GPU tests that E4M3 results are the quantiser's: cb_norm_residual without norms and cb_gemm_e4m3
with sums known exactly give, bit for bit, what cb_quantize_e4m3 makes of the same values,
infinities, NaN, zeros of either sign, blocks of nothing else and magnitudes over the whole range among
them.
"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_block_ops import DT, E4M3, E8M0, INF, NAN, be, ceil, gen, op, randn  # noqa: E402, F401


def values(g, rows, C, lo=-140, hi=127):
    """fp32 rows: sizes from 2^lo to 2^hi, special values in places and in whole blocks."""
    x = randn(g, rows, C).clamp(-3.9, 3.9) / 4 * torch.exp2(torch.randint(lo, hi + 1, (rows, ceil(C, 128)), device="cuda", generator=g).float()
                                                            ).repeat_interleave(128, 1)[:, :C]
    for v in (INF, -INF, NAN, 0.0, -0.0):
        x = torch.where(torch.rand(rows, C, device="cuda", generator=g) < 0.004, v, x)
    if rows > 5:
        x[1, :128], x[2, :128], x[3, :128], x[4, :128], x[5, :128] = NAN, INF, 0.0, -0.0, 1e-45
    return x.contiguous()


def quantised(be, x, ds):
    rows, C = x.shape
    q, s = torch.zeros(rows, C, device="cuda").to(E4M3), torch.zeros(rows, ceil(C, 128), device="cuda").to(DT[ds])
    be.quantize_e4m3(1, rows, C, 1, op(be, x, C), op(be, q, C), op(be, s, ceil(C, 128)))
    return q, s


def equal(a, b):
    return torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("ds", ["e8m0", "f32"])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,C", [(7, 1), (33, 24), (300, 64), (20001, 64), (300, 77), (300, 128), (11001, 128), (300, 256), (15001, 256), (300, 333),
                                    (8003, 333), (10001, 1024), (300, 1000), (300, 1001), (43001, 1000), (300, 2048), (300, 4096), (17001, 4096),
                                    (300, 5001), (3001, 5001), (64, 8192), (64, 9000), (64, 9001)])
def test_norm_without_norms(be, sb, rows, C, dt, ds):
    g = gen(rows + C)
    x = values(g, rows, C, *((-20, 15) if dt == "f16" else (-140, 127))).to(DT[dt])
    q, s = torch.zeros(rows, C, device="cuda").to(E4M3), torch.zeros(rows, ceil(C, 128), device="cuda").to(DT[ds])
    be.norm_residual(1, rows, C, op(be, x, C), Y=op(be, q, C), S=op(be, s, ceil(C, 128)))
    wq, ws = quantised(be, x, ds)
    assert equal(s, ws)
    assert equal(q, wq)


@pytest.mark.parametrize("dsa,dsb", [("e8m0", "e8m0"), ("f32", "e8m0"), ("f32", "f32")])
@pytest.mark.parametrize("M,N,K,ldc", [(3, 130, 16, 130), (3, 130, 16, 144), (300, 257, 100, 257), (300, 1000, 128, 1008), (5000, 512, 256, 512),
                                       (20000, 640, 1024, 640), (20000, 1000, 640, 1008)])
def test_product_of_known_sums(be, sb, M, N, K, ldc, dsa, dsb):
    """A is zero, so that a result is its bias: one row of values, and a block's scale for every row."""
    g = gen(M + N)
    x = values(g, 1, N)[0].contiguous()
    a, b = torch.zeros(M, ceil(K, 16) * 16, device="cuda").to(E4M3), randn(g, N, ceil(K, 16) * 16).to(E4M3)
    kb = ceil(K, 128)
    sa, s_b = torch.ones(M, kb, device="cuda").to(DT[dsa]), torch.ones(ceil(N, 128), kb, device="cuda").to(DT[dsb])
    for ds in ("e8m0", "f32"):
        c, sc = torch.full((M, ldc), 1.0, device="cuda").to(E4M3), torch.zeros(M, ceil(N, 128), device="cuda").to(DT[ds])
        be.gemm_e4m3(M, N, K, op(be, a, a.shape[1]), op(be, sa, kb), op(be, b, b.shape[1]), op(be, s_b, kb), op(be, c, ldc), op(be, sc, ceil(N, 128)),
                     be.wrap(x))
        # -0 + 0 is 0: the sums are zeros of the positive sign
        wq, ws = quantised(be, (x + 0.0)[None].contiguous(), ds)
        assert equal(sc, ws.expand(M, -1).contiguous())
        assert equal(c[:, :N].contiguous(), wq.expand(M, -1).contiguous())
        assert (c[:, N:].float() == 1.0).all()
