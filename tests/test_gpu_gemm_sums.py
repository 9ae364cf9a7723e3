"""GPU tests of how cb_gemm_e4m3 sums 32-bit results: rounded to nearest from block to block
over more than 1024 columns or with scales given as F32, else by the matrix unit, which
truncates.

Bounds on the rms error against 64 bits, relative to the rms of the results. Rounding a sum of
size s to 32 bits is off by at most 2^-23 / sqrt(12) s (rms); the sum behind block i of kb has
the rms sqrt(i / kb) of the result, so kb roundings that know nothing of one another come to
2^-23 / sqrt(12) sqrt((kb + 1) / 2): 7.3e-8 for 8 blocks, 1.4e-7 for 32. What the matrix unit
cuts off inside a block is at most a quarter of that again. By the matrix unit over 8 blocks: the
documented 7e-8 and half of it more.
"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_block_ops import be, ceil, f64, gen, make_operand, op  # noqa: E402, F401


def products(be, M, N, K):
    """(with E8M0 scales, with the same scales as F32, in 64 bits)"""
    g = gen(M + N + K)
    a, sa, av = make_operand(g, M, K, 1, "e8m0")
    b, s_b, bv = make_operand(g, N, K, 128, "e8m0", 0.0)
    kb, out = ceil(K, 128), []
    for as_f32 in (False, True):
        x, y = (t.float().contiguous() if as_f32 else t for t in (sa, s_b))
        c = torch.empty(M, N, device="cuda")
        be.gemm_e4m3(M, N, K, op(be, a, a.shape[1]), op(be, x, kb), op(be, b, b.shape[1]), op(be, y, kb), op(be, c, N))
        out.append(c)
    return out[0], out[1], av @ bv.t()


def rms(c, z):
    return float((c.to(f64) - z).norm() / z.norm())


@pytest.mark.parametrize("M,N,K", [(2048, 1024, 4096), (20000, 512, 4096), (2048, 1024, 1025), (300, 300, 2048)])
def test_long_sums_are_rounded(be, sb, M, N, K):
    """The same bits with E8M0 scales and with F32 ones."""
    e8m0, f32, z = products(be, M, N, K)
    assert torch.equal(e8m0, f32)
    kb = ceil(K, 128)
    assert rms(e8m0, z) <= 1.25 * 2.0 ** -23 / 12 ** 0.5 * ((kb + 1) / 2) ** 0.5


@pytest.mark.parametrize("M,N,K", [(2048, 1024, 1024), (20000, 512, 1024), (2048, 1024, 588)])
def test_short_sums(be, sb, M, N, K):
    e8m0, f32, z = products(be, M, N, K)
    kb = ceil(K, 128)
    assert rms(f32, z) <= 1.25 * 2.0 ** -23 / 12 ** 0.5 * ((kb + 1) / 2) ** 0.5
    assert rms(e8m0, z) <= 1.05e-7
