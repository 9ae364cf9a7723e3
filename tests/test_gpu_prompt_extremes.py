"""GPU tests of the prompt-path operators, and of cb_attention, at the ends of what their arguments may hold: scores that
rise late or are huge, weights and values far below or above the others, the largest clusters, NaN payloads, the tail
of GELU. Against plain implementations in 64 bits; tolerances as derived in test_gpu_prompt_ops.py, with what a test
adds to them derived beside it.
"""
import math

import pytest

torch = pytest.importorskip("torch")
from test_gpu_prompt_ops import (DT, attend_ref, attend_tol, be, check_attend, gen, op, randn, u)  # noqa: E402,F401

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
