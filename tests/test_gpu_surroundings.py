"""GPU tests of what the prompt path's and the blocks' operators leave alone: results that
are parts of a buffer of random bits, given to the library up to their last element, in rows and
heads that do not touch one another. Every other byte of the buffer keeps its value; what the
results are is tested beside each operator.
"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_block_ops import DT, be, ceil, gen, op, randn  # noqa: E402, F401
from test_gpu_result_rows import bits, surroundings  # noqa: E402


class Part:
    """[nb, N, heads, hd] of a buffer: gap0, gap and gap1 elements between sequences, rows and heads, `off` in front."""

    def __init__(self, be, dt, nb, N, heads, hd, gap0, gap, gap1, off, seed=0):
        s1 = hd + gap1 if heads > 1 or gap1 else 0
        ld = (heads * s1 if heads > 1 else hd) + gap
        s0 = N * ld + gap0
        last = off + (nb - 1) * s0 + (N - 1) * ld + (heads - 1) * s1 + hd
        self.all = surroundings(last + 100, DT[dt], seed)
        self.index = (off + torch.arange(nb)[:, None, None, None] * s0 + torch.arange(N)[:, None, None] * ld +
                      torch.arange(heads)[:, None] * s1 + torch.arange(hd)).flatten().cuda()
        self.op = op(be, self.all[:last], ld, s0, s1 if heads > 1 else 0, off)
        self.before = bits(self.all).clone()

    def check(self):
        size = self.all.element_size()
        out = torch.ones(self.all.numel(), dtype=torch.bool, device="cuda")
        out[self.index] = False
        out = out.repeat_interleave(size)
        assert torch.equal(bits(self.all)[out], self.before[out])


def rows(be, g, dt, nb, N, C):
    return op(be, randn(g, nb, N, C).to(DT[dt]), C, N * C)


GAPS = [(0, 0, 0), (3, 5, 1), (16, 8, 8), (0, 16, 0)]  # elements behind sequences and rows, and in front


@pytest.mark.parametrize("gaps", GAPS)
@pytest.mark.parametrize("brows", [1, 128])
@pytest.mark.parametrize("nb,N,K", [(1, 1, 1), (3, 5, 100), (2, 131, 257), (2, 300, 1000), (1, 3000, 1028)])
def test_quantiser(be, nb, N, K, brows, gaps):
    for i, (dt, ds) in enumerate((("bf16", "e8m0"), ("f32", "f32"))):
        g = gen(N + K + i)
        q, s = Part(be, "e4m3", nb, N, 1, K, gaps[0], gaps[1], 0, gaps[2]), Part(be, ds, nb, ceil(N, brows), 1, ceil(K, 128), gaps[0], gaps[1], 0, gaps[2], 1)
        be.quantize_e4m3(nb, N, K, brows, rows(be, g, dt, nb, N, K), q.op, s.op)
        q.check()
        s.check()


@pytest.mark.parametrize("gaps", GAPS)
@pytest.mark.parametrize("nb,N,C", [(1, 1, 1), (3, 5, 100), (2, 301, 64), (2, 33, 257), (3, 2001, 520), (2, 401, 1024), (2, 7, 1030), (2, 9, 4096), (2, 3, 9001)])
def test_norm(be, sb, nb, N, C, gaps):
    for i, (dt, yt) in enumerate((("bf16", "bf16"), ("f32", "e4m3"), ("f32", "f16"))):
        g = gen(N + C + i)
        r, y = Part(be, dt, nb, N, 1, C, gaps[0], gaps[1], 0, gaps[2]), Part(be, yt, nb, N, 1, C, gaps[0], gaps[1], 0, gaps[2], 1)
        s = Part(be, "e8m0", nb, N, 1, ceil(C, 128), gaps[0], gaps[1], 0, gaps[2], 2) if yt == "e4m3" else None
        be.norm_residual(nb, N, C, rows(be, g, dt, nb, N, C), rows(be, g, dt, nb, N, C), R=r.op, pre=sb.Norm(sb.NORM_LAYER), Y=y.op, S=s.op if s else None)
        for part in (r, y, s):
            if part:
                part.check()


@pytest.mark.parametrize("gap0,gap,gap1,off", [(0, 0, 0, 0), (3, 5, 3, 1), (16, 8, 16, 8)])
@pytest.mark.parametrize("halves", [0, 1])
@pytest.mark.parametrize("nb,N,h,hd,rot", [(1, 1, 1, 2, 2), (2, 9, 3, 64, 64), (2, 33, 5, 80, 60), (1, 301, 24, 64, 32)])
def test_rotation(be, sb, nb, N, h, hd, rot, halves, gap0, gap, gap1, off):
    for tx, ty in (("bf16", "bf16"), ("f32", "f32"), ("f32", "f16")):
        g = gen(N + hd)
        x = op(be, randn(g, nb, N, h, hd).to(DT[tx]), h * hd, N * h * hd, hd)
        cs = be.wrap(randn(g, N, rot))
        for axes in (False, True):
            y = Part(be, ty, nb, N, h, hd, gap0, gap, gap1, off)
            if axes:
                be.rope_rotate_axes(nb, N, h, hd, rot, halves, sb.RopeAxes((rot,)), x, y.op, cs, N, None, (N,))
            else:
                be.rope_rotate(nb, N, h, hd, rot, halves, x, y.op, cs, N)
            y.check()


@pytest.mark.parametrize("gap0,gap,gap1,off", [(0, 0, 0, 0), (3, 5, 3, 1), (16, 8, 8, 8)])
@pytest.mark.parametrize("nb,Nq,Nk,h,kv,hd", [(2, 1, 77, 4, 2, 32), (2, 201, 333, 8, 8, 32), (1, 700, 39, 8, 8, 64), (2, 300, 700, 4, 4, 40), (1, 900, 900, 4, 4, 128)])
def test_cross_attention(be, sb, nb, Nq, Nk, h, kv, hd, gap0, gap, gap1, off):
    for dt in ("bf16", "f32"):
        g = gen(Nq + Nk)
        q = op(be, randn(g, nb, Nq, h, hd).to(DT[dt]), h * hd, Nq * h * hd, hd)
        k, v = (op(be, randn(g, nb, Nk, kv, hd).to(DT[dt]), kv * hd, Nk * kv * hd, hd) for _ in range(2))
        o = Part(be, dt, nb, Nq, h, hd, gap0, gap, gap1, off)
        be.cross_attend(nb, Nq, Nk, h, kv, hd, q, k, v, o.op, None, None, hd ** -0.5)
        o.check()


@pytest.mark.parametrize("gaps", GAPS)
@pytest.mark.parametrize("nb,npix,C,groups", [(1, 1, 4, 2), (2, 77, 96, 8), (3, 1000, 256, 32), (1, 5184, 100, 5)])
def test_groupnorm(be, nb, npix, C, groups, gaps):
    for tx, ty in (("bf16", "bf16"), ("f32", "f32"), ("f32", "bf16")):
        g = gen(npix + C)
        y = Part(be, ty, nb, npix, 1, C, gaps[0], gaps[1], 0, gaps[2])
        be.groupnorm(nb, npix, C, groups, rows(be, g, tx, nb, npix, C), y.op, be.wrap(randn(g, C)), be.wrap(randn(g, C)), 1e-5, 1)
        y.check()
