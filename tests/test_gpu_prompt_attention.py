"""GPU test: rows rotated by cb_rope_rotate are what cb_attention takes (16-bit rows that hold their positions already)."""
import pytest

torch = pytest.importorskip("torch")
from test_gpu_prompt_ops import attend_ref, attend_tol, be, gen, op, randn, rotate_ref  # noqa: E402,F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("src", ["f32", "bf16"])
@pytest.mark.parametrize("N", [576, 169])
def test_rotated_rows_into_attention(be, sb, N, src):
    """Queries and keys of fused q | k | v rows rotated by one call (32-bit rows into 16-bit ones, or 16-bit rows in
    place), values copied beside them, then self-attention; against 64 bits on the rotated, rounded rows, which are
    checked themselves: 4 * 2^-24 (|x0| + |x1|) and half a step of the type."""
    nb, h, hd = 2, 16, 64
    E = h * hd
    g = gen(N)
    x = randn(g, nb, N, 3 * E).to(torch.float32 if src == "f32" else torch.bfloat16)
    cs = torch.empty(N, hd // 2, 2, device="cuda")
    be.rope_table(N, hd, 0, None, be.wrap(cs))
    qkv = x.clone() if src == "bf16" else torch.empty(nb, N, 3 * E, device="cuda", dtype=torch.bfloat16)
    qkv[..., 2 * E:] = x[..., 2 * E:].bfloat16()
    m = qkv if src == "bf16" else x
    be.rope_rotate(nb, N, 2 * h, hd, hd, sb.ROPE_PAIRS, op(be, m, 0, 3 * E, N * 3 * E, hd),
                   op(be, qkv, 0, 3 * E, N * 3 * E, hd), be.wrap(cs), N)
    o = torch.empty(nb * N, E, device="cuda")
    be.attention(be.wrap(qkv), nb, N, E, h, hd, None, 0, 0.125, sb.ATTN_TC, be.wrap(o))
    be.sync()
    at = torch.arange(N, device="cuda").expand(nb, N)
    want, e = rotate_ref(x[..., :2 * E].double().reshape(nb, N, 2 * h, hd), cs.double(), at, hd, False, N)
    got = qkv[..., :2 * E].reshape(nb, N, 2 * h, hd).double()
    assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + 1.01 * e).all()
    q, k, v = (qkv[..., i * E:(i + 1) * E].reshape(nb, N, h, hd).double() for i in range(3))
    want, A, big = attend_ref(q, k, v, torch.ones(nb, N, dtype=torch.bool, device="cuda"), 0.125)
    # its exponentials are within 7.5e-5 (2^-13.7) of the weight
    tol = attend_tol(torch.bfloat16, want, A, big, hd, N) + 2.0 ** -13 * A
    assert ((o.view(nb, N, h, hd).double() - want).abs() <= tol).all()
