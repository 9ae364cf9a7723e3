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
