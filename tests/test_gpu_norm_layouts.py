"""GPU tests of cb_norm_residual over the layouts of its operands: gate, scale and
shift for all rows, for a sample's or row by row, each on its own, in every form of the
kernel on both sides of the row count where rows begin to share their sample's vectors;
and over memory that is read and written, there too.

Against norm_ref, in 64 bits; its tolerances.
"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_block_ops import DT, E8M0, be, ceil, check_quantised, check_rounded, f64, gen, norm_ref, op, randn  # noqa: E402, F401

LAYOUTS = ("all", "sample", "row")
# C, type, columns behind a row, (nb, N) without and with shared vectors on 148 SMs
FORMS = [
    (64, "bf16", 0, (3, 5), (2, 10001)),        # parts of a warp
    (128, "f16", 0, (3, 7), (3, 3301)),
    (256, "bf16", 0, (2, 301), (5, 3003)),      # a warp, aligned
    (512, "f32", 0, (2, 301), (5, 2003)),
    (1024, "bf16", 0, (2, 301), (2, 5001)),
    (1024, "f32", 0, (2, 301), (2, 21501)),     # a CTA, aligned
    (2048, "f16", 0, (2, 33), (2, 19001)),
    (4096, "bf16", 0, (2, 33), (2, 8301)),
    (8192, "f32", 0, (2, 33), (2, 6301)),
    (77, "f32", 0, (2, 301), (2, 19001)),       # a warp, not aligned
    (333, "f32", 0, (2, 301), (3, 2403)),
    (1024, "f32", 1, (2, 101), (2, 16601)),     # a CTA, not aligned
    (2047, "f32", 0, (2, 33), (2, 10701)),
    (3001, "f32", 0, (2, 33), (2, 3601)),
    (5001, "f32", 0, (2, 33), (2, 1503)),
    (77, "bf16", 0, (2, 301), (2, 19001)),      # not aligned, 16 bits: one form
    (1024, "bf16", 1, (2, 101), (2, 4001)),
    (2047, "f16", 0, (2, 33), (2, 701)),
    (5001, "bf16", 0, (2, 33), (3, 301)),
    (9001, "f16", 0, (2, 3), (3, 301)),         # rows of any width
    (12288, "bf16", 0, (2, 3), (3, 301)),
]


def layout(be, g, how, dt, nb, N, C):
    """An operand of the layout: (f64 values that broadcast, descriptor)."""
    shape = {"all": (1, 1, C), "sample": (nb, 1, C), "row": (nb, N, C)}[how]
    t = (0.5 * randn(g, *shape)).to(DT[dt])
    return t.to(f64), op(be, t, C if how == "row" else 0, {"all": 0, "sample": C, "row": N * C}[how])


def call(be, sb, g, nb, N, C, xt, pad, gate=None, scale=None, shift=None, post=0, pre=1, bias=True, yt=None, place=(None, None), h=True):
    """One call and its check. gate, scale, shift: (layout, type) or None; place: what R and Y are (X, H or None)."""
    yt = yt or xt
    ld = C + pad

    def rows(dt, scale, mean):
        t = torch.full((nb, N, ld), 5.0, device="cuda").to(DT[dt])
        t[..., :C] = (randn(g, nb, N, C) * scale + mean).to(DT[dt])
        return t

    def opr(t):
        return op(be, t, ld, N * ld)

    def norm(kind, eps):
        w, b = (1 + 0.3 * randn(g, C), 0.3 * randn(g, C) if bias else None) if kind else (None, None)
        return (kind, w, b, eps), (sb.Norm(kind, eps, be.wrap(w), None if b is None else be.wrap(b)) if kind else None)
    x, hh = rows(xt, 1.5, 0.2), rows(xt, 0.7, 0.1) if h else None
    x64, h64 = x[..., :C].to(f64), hh[..., :C].to(f64) if h else None
    (post64, postn), (pre64, pren) = norm(post, 1e-5), norm(pre, 1e-3)
    v = {n: layout(be, g, *o, nb, N, C) if o else (None, None) for n, o in (("gate", gate), ("scale", scale), ("shift", shift))}
    there = {"X": x, "H": hh}
    r, y = (there[p] if p else torch.full((nb, N, ld), 5.0, device="cuda").to(DT[t]) for p, t in zip(place, (xt, yt)))
    s = torch.zeros(nb, N, ceil(C, 128), device="cuda").to(E8M0) if yt == "e4m3" else None
    be.norm_residual(nb, N, C, opr(x), opr(hh) if h else None, postn, 1.0, None, v["gate"][1], opr(r), pren, v["scale"][1], v["shift"][1], opr(y),
                     None if s is None else op(be, s, ceil(C, 128), N * ceil(C, 128)))
    rr, dr, yy, dy = norm_ref(x64, h64, post64, 1.0, None, v["gate"][0], pre64, v["scale"][0], v["shift"][0], max(32, C / 1024) + 40)
    check_rounded(r[..., :C], rr, dr, DT[xt])
    if yt == "e4m3":
        check_quantised(y[..., :C].reshape(nb * N, C), s.view(nb * N, -1), yy.view(nb * N, C), dy.view(nb * N, C))
    else:
        check_rounded(y[..., :C], yy, dy, DT[yt])
    if pad:
        assert (r[..., C:].float() == 5.0).all() and (y[..., C:].float() == 5.0).all()


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("form", FORMS, ids=lambda f: f"{f[0]}-{f[1]}-{f[2]}")
def test_scale_and_shift_of_any_layout(be, sb, form, many):
    """The nine pairs, each with another gate, norm, type and result than the last."""
    C, dt, pad, few, lot = form
    nb, N = lot if many else few
    g = gen(C + N)
    other = "f32" if dt != "f32" else "bf16"
    i = 0
    for a in LAYOUTS:
        for b in LAYOUTS:
            call(be, sb, g, nb, N, C, dt, pad, gate=(None, (LAYOUTS[i % 3], other))[i % 2], scale=(a, (dt, other)[i % 2]), shift=(b, (other, dt)[i // 2 % 2]),
                 post=i % 3, pre=(1, 2, 0)[i // 2 % 3], bias=i % 4 != 3, yt="e4m3" if i % 3 == 1 else None, h=i != 6)
            i += 1


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("form", FORMS, ids=lambda f: f"{f[0]}-{f[1]}-{f[2]}")
def test_scale_or_shift_alone(be, sb, form, many):
    C, dt, pad, few, lot = form
    nb, N = lot if many else few
    g = gen(C + N + 1)
    for i, a in enumerate(LAYOUTS):
        call(be, sb, g, nb, N, C, dt, pad, scale=(a, "f32"), pre=1 + i % 2)
        call(be, sb, g, nb, N, C, dt, pad, shift=(a, "f16"), pre=i % 3, gate=(a, dt))


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("form", FORMS, ids=lambda f: f"{f[0]}-{f[1]}-{f[2]}")
@pytest.mark.parametrize("place", [("X", None), ("H", None), (None, "X"), (None, "H"), ("X", "H"), ("H", "X")], ids=lambda p: f"R={p[0]},Y={p[1]}")
def test_in_place(be, sb, place, form, many):
    """Every row is read as it was before the call."""
    C, dt, pad, few, lot = form
    nb, N = lot if many else few
    g = gen(C + N + 2)
    call(be, sb, g, nb, N, C, dt, pad, gate=("sample", "f32"), scale=("sample", "f32"), shift=("sample", "f32"), post=2, place=place)


@pytest.mark.parametrize("C,dt,nb,N", [(512, "bf16", 700, 31), (512, "bf16", 700, 32), (4096, "f16", 600, 31), (4096, "f16", 600, 32), (64, "f32", 400, 63),
                                       (64, "f32", 400, 64)])
def test_many_samples_of_few_rows(be, sb, C, dt, nb, N):
    """Around the rows of a sample from which they share its vectors."""
    g = gen(C + N + 3)
    call(be, sb, g, nb, N, C, dt, 0, gate=("sample", "f32"), scale=("sample", "f32"), shift=("row", dt), post=1)
