"""Cases that time and check the operators around attention in a transformer block with 8-bit products: the quantiser to
8-bit floating point with a power-of-two scale per block of 128, the matrix product of such operands, the norms before and after a block
with its gate and residual scale, and rotary positions with several axes.

`own` selects between two forms of the same pass: the plain one in elementary torch operations (32 bits, rounded once at the
end) and the calls a program makes of the library's entry points. `listed()` are the fixed cases, `draw()` gives further ones of
the same ranges, `prepare()` makes a case's inputs on the GPU from a seed, `run()` is one pass, `work()` what the pass cannot do
without, and `exact()` the operator's definition in 64 bits (8-bit results before their rounding, in units of their scales).
"""
import importlib.util
import math
import os
import sys

import torch

own = False

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "e4m3": E4M3, "e8m0": E8M0}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1, "e8m0": 1}
ACT = {"none": 0, "gelu": 1, "relu": 2}
NORM = {"none": 0, "layer": 1, "rms": 2}
BLOCK = 128


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # One new token for each of eight sequences through a 1024 -> 4096 projection: latency counts.
        dict(name="gemm_step", op="gemm", M=8, N=4096, K=1024, wscale="e8m0", out="bf16", act="none", bias=True),
        # The first MLP product of eight crops' 72 x 72 tokens, its GELU quantised for the second one: the largest.
        dict(name="gemm_fc1", op="gemm", M=41472, N=4096, K=1024, wscale="e8m0", out="e4m3", act="gelu", bias=True),
        # The second MLP product, weights of a checkpoint with 32-bit scales.
        dict(name="gemm_fc2", op="gemm", M=41472, N=1024, K=4096, wscale="f32", out="bf16", act="none", bias=True),
        # Patch embedding of one crop: 14 x 14 x 3 columns, no multiple of a block; 32-bit result.
        dict(name="gemm_patch", op="gemm", M=5184, N=1024, K=588, wscale="e8m0", out="f32", act="none", bias=True),
        # Activations of the MLP's hidden layer, one scale for 128 columns of a row.
        dict(name="quant_rows", op="quant", N=41472, K=4096, brows=1, dt="bf16"),
        # A layer's weights at load time, one scale for 128 x 128 values.
        dict(name="quant_weight", op="quant", N=4096, K=1024, brows=128, dt="f32"),
        # Between two blocks for one new token of eight sequences.
        dict(name="norm_step", op="norm", nb=8, N=1, C=1024, dt="bf16", hdt="bf16", out="bf16", post="none", pre="rms", gate="none",
             ls=False, mod=False, nbias=False),
        # Between two blocks of eight crops' tokens: residual scale per channel, gate, shift and scale per sample.
        dict(name="norm_block", op="norm", nb=8, N=5184, C=1024, dt="bf16", hdt="bf16", out="bf16", post="none", pre="layer",
             gate="sample", ls=True, mod=True, nbias=True),
        # Norms on both sides of a block, odd rows and width, quantised for the next product.
        dict(name="norm_sandwich", op="norm", nb=3, N=1801, C=1000, dt="f32", hdt="f32", out="e4m3", post="rms", pre="rms", gate="none",
             ls=False, mod=False, nbias=False),
        # One new token of eight sequences, positions (time, height, width) of their own.
        dict(name="rope_axes_step", op="rope", nb=8, N=1, heads=20, hd=64, rot=64, w0=16, w1=24, w2=24, order="sections", layout="halves",
             dt="bf16", extra=256, npos=8192, pos="given", t=0, h=0, w=0),
        # Queries and keys of two clips of four frames of 72 x 72 tokens, out of the fused q | k | v rows.
        dict(name="rope_axes_video", op="rope", nb=2, N=4 * 5184, heads=24, hd=64, rot=64, w0=16, w1=24, w2=24, order="sections",
             layout="pairs", dt="bf16", extra=768, npos=128, pos="grid", t=4, h=72, w=72),
        # Axes take turns over the pairs, part of the head is turned, odd row count.
        dict(name="rope_axes_turns", op="rope", nb=3, N=3001, heads=7, hd=80, rot=60, w0=24, w1=18, w2=18, order="turns", layout="halves",
             dt="f32", extra=0, npos=4096, pos="given", t=0, h=0, w=0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_once(rng):
    op = rng.choice(["gemm", "gemm", "gemm", "quant", "norm", "norm", "rope"])
    if op == "gemm":
        whole = rng.random() < 0.5
        n, k = _log_int(rng, 16, 4096), _log_int(rng, 16, 4096)
        return dict(op=op, M=_log_int(rng, 1, 41472), N=max(16, n // 16 * 16) if whole else n, K=max(16, k // 16 * 16) if whole else k,
                    wscale=rng.choice(["e8m0", "f32"]), out=rng.choice(["bf16", "bf16", "f16", "f32", "e4m3"]),
                    act=rng.choice(["none", "none", "gelu", "relu"]), bias=rng.random() < 0.7)
    if op == "quant":
        return dict(op=op, N=_log_int(rng, 1, 41472), K=_log_int(rng, 16, 8192), brows=rng.choice([1, 1, 128]),
                    dt=rng.choice(["bf16", "f16", "f32"]))
    if op == "norm":
        c = _log_int(rng, 16, 8192)
        dt = rng.choice(["bf16", "bf16", "f16", "f32"])
        return dict(op=op, nb=rng.randint(1, 9), N=_log_int(rng, 1, 5184), C=c if rng.random() < 0.4 else max(16, c // 64 * 64), dt=dt,
                    hdt=dt if dt != "f32" else rng.choice(["f32", "bf16"]), out=rng.choice([dt, dt, "bf16", "e4m3"]) if dt == "f32" else
                    rng.choice([dt, dt, "e4m3"]), post=rng.choice(["none", "layer", "rms"]), pre=rng.choice(["layer", "rms"]),
                    gate=rng.choice(["none", "sample", "row"]), ls=rng.random() < 0.5, mod=rng.random() < 0.5, nbias=rng.random() < 0.5)
    hd = rng.choice([32, 64, 80, 96, 128])
    axes = rng.choice([2, 3, 3])
    order = rng.choice(["sections", "sections", "turns"])
    pairs = hd // 2 if rng.random() < 0.6 else rng.randint(6, hd // 2)
    each = pairs // axes
    p = [pairs - (axes - 1) * each, each, each if axes == 3 else 0]
    grid = rng.random() < 0.5
    t, h, w = (rng.randint(1, 8) if axes == 3 else 1), rng.randint(1, 72), rng.randint(1, 72)
    return dict(op=op, nb=rng.randint(1, 9), N=t * h * w if grid else _log_int(rng, 1, 8192), heads=rng.randint(1, 32), hd=hd, rot=2 * pairs,
                w0=2 * p[0], w1=2 * p[1], w2=2 * p[2], order=order, layout=rng.choice(["pairs", "halves"]), dt=rng.choice(["bf16", "bf16", "f16", "f32"]),
                extra=rng.choice([0, hd, 4 * hd]), npos=rng.choice([128, 1000, 8192]), pos="grid" if grid else rng.choice(["given", "excluded"]),
                t=t if grid else 0, h=h if grid else 0, w=w if grid else 0)


def draw(rng):
    while True:
        case = _draw_once(rng)
        w = work(case)
        # No more than the largest listed cases.
        if w["bytes"] <= 5.0e8 and w["flops"] <= 3.4e11:
            return case


# ------------------------------------------------------------------------------------------------ blocks of 128
def _ceil(a, b):
    return -(-a // b)


def _spread(s, rows, cols, brows):
    """A scale per block as a value per element: [rows, cols]."""
    s = s.float()
    if brows > 1:
        s = s.repeat_interleave(brows, -2)[..., :rows, :]
    return s.repeat_interleave(BLOCK, -1)[..., :cols]


def _power(e):
    """2^e for whole numbers -126 .. 127, exactly."""
    return ((e + 127) << 23).view(torch.float32)


def _block_scales(x, brows):
    """Exponents of the blocks' scales, int32 [ceil(rows / brows), ceil(cols / 128)]: the smallest e >= -126 with max |x| <= 448 * 2^e."""
    n, k = x.shape
    a = x.abs()
    a = torch.where(torch.isfinite(a), a, 0.0)
    a = torch.nn.functional.pad(a, (0, -k % BLOCK, 0, -n % brows))
    a = a.view(_ceil(n, brows), brows, -1, BLOCK).amax((1, 3))
    m, e = torch.frexp(a)  # a = m 2^e, m in [1/2, 1); 448 = 0.875 * 2^9
    e = torch.where(a > 0, e - 9 + (m > 0.875).int(), -126)
    return e.clamp_min(-126).int()


def _quantised(x, brows):
    """(8-bit values, exponents of their scales) of 32-bit x [rows, cols]."""
    e = _block_scales(x, brows)
    q = (x * _spread(_power(-e), x.shape[0], x.shape[1], brows)).to(E4M3)
    return q, e


def _as_e8m0(e):
    return (e + 127).to(torch.uint8).view(E8M0)


def _padded(q):
    """Rows that start at multiples of 16 bytes, as the product reads them."""
    n, k = q.shape
    store = torch.zeros(n, _ceil(k, 16) * 16, dtype=torch.uint8, device="cuda")
    store[:, :k] = q.view(torch.uint8)
    return store.view(E4M3)


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _widths(c):
    return [w for w in (c["w0"], c["w1"], c["w2"]) if w]


def _axis_of_pairs(c):
    """The axis of each pair: sections one after another, or axis a > 0 at pairs a, a + axes, ... while it has some left, axis 0 elsewhere."""
    pairs = [w // 2 for w in _widths(c)]
    if c["order"] == "sections":
        return [a for a, n in enumerate(pairs) for _ in range(n)]
    k = len(pairs)
    return [j % k if j // k < pairs[j % k] else 0 for j in range(c["rot"] // 2)]


def prepare(case, seed):
    g = _gen(seed)
    dev = "cuda"
    s = {"case": case}

    def randn(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    if case["op"] == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        # Activations with channels of different size, weights of a trained layer's spread.
        x = randn(M, K).mul_(torch.exp(0.5 * randn(K)))
        q, e = _quantised(x, 1)
        s["a"], s["sa"] = _padded(q), _as_e8m0(e)
        w = randn(N, K).mul_(1.0 / math.sqrt(K))
        if case["wscale"] == "e8m0":
            q, e = _quantised(w, BLOCK)
            s["sb"] = _as_e8m0(e)
        else:
            a = torch.nn.functional.pad(w.abs(), (0, -K % BLOCK, 0, -N % BLOCK))
            s["sb"] = a.view(_ceil(N, BLOCK), BLOCK, -1, BLOCK).amax((1, 3)) / 448.0
            q = (w / _spread(s["sb"], N, K, BLOCK)).clamp_(-448.0, 448.0).to(E4M3)
        s["b"] = _padded(q)
        s["bias"] = 0.1 * randn(N) if case["bias"] else None
        s["c"] = torch.empty(M, N, device=dev, dtype=DT[case["out"]])
        s["sc"] = torch.empty(M, _ceil(N, BLOCK), device=dev, dtype=E8M0) if case["out"] == "e4m3" else None
    elif case["op"] == "quant":
        N, K = case["N"], case["K"]
        s["x"] = randn(N, K).mul_(torch.exp(0.5 * randn(K))).to(DT[case["dt"]])
        s["q"] = torch.empty(N, K, device=dev, dtype=E4M3)
        s["s"] = torch.empty(_ceil(N, case["brows"]), _ceil(K, BLOCK), device=dev, dtype=E8M0)
    elif case["op"] == "norm":
        nb, N, C = case["nb"], case["N"], case["C"]
        # A residual stream with a few channels far larger than the others.
        big = torch.where(torch.rand(C, device=dev, generator=g) < 0.01, 20.0, 1.0)
        s["x"] = randn(nb, N, C).add_(0.3 * randn(C)).mul_(big).to(DT[case["dt"]])
        s["h"] = randn(nb, N, C).mul_(0.7).to(DT[case["hdt"]])
        s["ls"] = 0.3 * randn(C) if case["ls"] else None
        # Gate, shift and scale as one projection of a sample's conditioning leaves them: in one row.
        s["mod"] = 0.5 * randn(nb, 3 * C) if case["mod"] or case["gate"] == "sample" else None
        s["gate"] = (0.5 * randn(nb, N, C)).to(DT[case["hdt"]]) if case["gate"] == "row" else None
        for k in ("post", "pre"):
            s[k + "_g"] = 1.0 + 0.2 * randn(C) if case[k] != "none" else None
            s[k + "_b"] = 0.2 * randn(C) if case[k] != "none" and case["nbias"] else None
        s["r"] = torch.empty_like(s["x"])
        s["y"] = torch.empty(nb, N, C, device=dev, dtype=DT[case["out"]])
        s["s"] = torch.empty(nb, N, _ceil(C, BLOCK), device=dev, dtype=E8M0) if case["out"] == "e4m3" else None
    else:
        nb, N, h, hd, rot, dt = case["nb"], case["N"], case["heads"], case["hd"], case["rot"], DT[case["dt"]]
        ld = h * hd + case["extra"]
        s["x"] = randn(nb, N, ld).to(dt)
        s["y"] = torch.empty(nb, N, h, hd, device=dev, dtype=dt)
        inv = 10000.0 ** (-torch.arange(0, rot, 2, device=dev, dtype=torch.float64) / rot)
        ang = torch.arange(case["npos"], device=dev, dtype=torch.float64)[:, None] * inv
        s["cs"] = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()
        s["axis"] = torch.tensor(_axis_of_pairs(case), device=dev)
        s["pos"] = None
        if case["pos"] != "grid":
            axes = len(_widths(case))
            p = torch.randint(0, case["npos"], (nb, N, axes), device=dev, generator=g, dtype=torch.int32)
            if case["pos"] == "excluded":
                p = torch.where(torch.rand(nb, N, axes, device=dev, generator=g) < 0.1, torch.full_like(p, -1), p)
            s["pos"] = p
    return s


# ------------------------------------------------------------------------------------------------ the plain form
def _gelu(z):
    return 0.5 * z * (1.0 + torch.erf(z * 0.7071067811865476))


def _plain_gemm(s):
    c = s["case"]
    M, N, K = c["M"], c["N"], c["K"]
    a = s["a"][:, :K].float().mul_(_spread(s["sa"], M, K, 1))
    b = s["b"][:, :K].float().mul_(_spread(s["sb"], N, K, BLOCK))
    z = a @ b.t()
    if s["bias"] is not None:
        z += s["bias"]
    z = _gelu(z) if c["act"] == "gelu" else (torch.relu(z) if c["act"] == "relu" else z)
    if c["out"] != "e4m3":
        return z.to(DT[c["out"]])
    q, e = _quantised(z, 1)
    return q, _as_e8m0(e)


def _plain_quant(s):
    q, e = _quantised(s["x"].float(), s["case"]["brows"])
    return q, _as_e8m0(e)


def _normed(v, kind, g, b):
    if kind == "none":
        return v
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + 1e-5) * g
    return v if b is None else v + b


def _plain_norm(s):
    c = s["case"]
    C = c["C"]
    h = _normed(s["h"].float(), c["post"], s["post_g"], s["post_b"])
    if s["ls"] is not None:
        h = h * s["ls"]
    if c["gate"] == "sample":
        h = h * s["mod"][:, None, :C]
    elif c["gate"] == "row":
        h = h * s["gate"].float()
    r = s["x"].float() + h
    y = _normed(r, c["pre"], s["pre_g"], s["pre_b"])
    if c["mod"]:
        y = y * (1.0 + s["mod"][:, None, C : 2 * C]) + s["mod"][:, None, 2 * C :]
    r = r.to(s["x"].dtype)
    if c["out"] != "e4m3":
        return r, y.to(DT[c["out"]])
    q, e = _quantised(y.view(-1, C), 1)
    return r, q.view(y.shape), _as_e8m0(e).view(c["nb"], c["N"], -1)


def _positions(s):
    """[nb or 1, N, axes] whole numbers."""
    c = s["case"]
    if s["pos"] is not None:
        return s["pos"].long()
    n = torch.arange(c["N"], device="cuda")
    p = [n // (c["h"] * c["w"]), n // c["w"] % c["h"], n % c["w"]]
    return torch.stack(p[3 - len(_widths(c)) :], -1)[None]


def _plain_rope(s):
    c = s["case"]
    nb, N, h, hd, rot = c["nb"], c["N"], c["heads"], c["hd"], c["rot"]
    x = s["x"][..., : h * hd].view(nb, N, h, hd)
    p = _positions(s)[..., s["axis"]]  # [nb or 1, N, pairs]
    keep = ((p >= 0) & (p < c["npos"]))[:, :, None]
    cs = s["cs"][p.clamp(0, c["npos"] - 1), torch.arange(rot // 2, device="cuda")]
    cos, sin = cs[..., 0][:, :, None], cs[..., 1][:, :, None]
    xf = x.float()
    a, b = (xf[..., 0:rot:2], xf[..., 1:rot:2]) if c["layout"] == "pairs" else (xf[..., : rot // 2], xf[..., rot // 2 : rot])
    u, v = torch.where(keep, a * cos - b * sin, a), torch.where(keep, a * sin + b * cos, b)
    r = torch.stack([u, v], -1).flatten(-2) if c["layout"] == "pairs" else torch.cat([u, v], -1)
    return torch.cat([r, xf[..., rot:]], -1).to(x.dtype)


# ------------------------------------------------------------------------------------------------ the library's calls
_lib = {}


def _backend():
    if "cb" not in _lib:
        name = "sam3_b200"
        mod = sys.modules.get(name)
        if mod is None:
            path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "i.sam3.opencl_b200", name + ".py")
            if not os.path.exists(path):
                path = os.path.join(os.getcwd(), "i.sam3.opencl_b200", name + ".py")
            spec = importlib.util.spec_from_file_location(name, path)
            mod = importlib.util.module_from_spec(spec)
            sys.modules[name] = mod
            spec.loader.exec_module(mod)
        _lib["sb"], _lib["cb"] = mod, mod.Backend(torch.cuda.current_device())
        # Work in the order of torch's current stream (1 is CUDA's name for the default one).
        _lib["cb"].set_stream(torch.cuda.current_stream().cuda_stream or 1)
    return _lib["sb"], _lib["cb"]


def _handles(s):
    """The library's handles of a state's buffers and their layouts, made once as a program keeps them."""
    sb, cb = _backend()
    c = s["case"]
    h = {}

    def op(t, ld=0, s0=0, s1=0, off=0):
        return None if t is None else cb.bmat(cb.wrap(t), off, ld, s0, s1)

    def rows(t):
        return None if t is None else op(t, t.shape[-1], t.shape[-1] * t.shape[-2])

    if c["op"] == "gemm":
        for k in ("a", "sa", "b", "sb", "c", "sc"):
            h[k] = rows(s[k])
        h["bias"] = None if s["bias"] is None else cb.wrap(s["bias"])
        h["act"] = ACT[c["act"]]
    elif c["op"] == "quant":
        for k in ("x", "q", "s"):
            h[k] = rows(s[k])
    elif c["op"] == "norm":
        C = c["C"]
        for k in ("x", "h", "r", "y", "s"):
            h[k] = rows(s[k])
        h["gate"] = rows(s["gate"]) if c["gate"] == "row" else (op(s["mod"], 0, 3 * C) if c["gate"] == "sample" else None)
        h["scale"], h["shift"] = (op(s["mod"], 0, 3 * C, 0, C), op(s["mod"], 0, 3 * C, 0, 2 * C)) if c["mod"] else (None, None)
        h["ls"] = None if s["ls"] is None else cb.wrap(s["ls"])
        for k in ("post", "pre"):
            g, b = s[k + "_g"], s[k + "_b"]
            h[k] = None if c[k] == "none" else sb.Norm(NORM[c[k]], 1e-5, cb.wrap(g), None if b is None else cb.wrap(b))
    else:
        N, w = c["N"], c["heads"] * c["hd"]
        ld = w + c["extra"]
        h["x"], h["y"] = op(s["x"], ld, N * ld, c["hd"]), op(s["y"], w, N * w, c["hd"])
        h["cs"] = cb.wrap(s["cs"])
        h["pos"] = None if s["pos"] is None else cb.wrap(s["pos"])
        h["axes"] = sb.RopeAxes(_widths(c), sb.ROPE_AXES_SECTIONS if c["order"] == "sections" else sb.ROPE_AXES_TURNS)
        h["grid"] = (c["t"], c["h"], c["w"])[3 - len(_widths(c)) :] if s["pos"] is None else None
        h["layout"] = sb.ROPE_PAIRS if c["layout"] == "pairs" else sb.ROPE_HALVES
    return h


def _own(s):
    c = s["case"]
    if "handles" not in s:
        s["handles"] = _handles(s)
    h, cb = s["handles"], _lib["cb"]
    if c["op"] == "gemm":
        cb.gemm_e4m3(c["M"], c["N"], c["K"], h["a"], h["sa"], h["b"], h["sb"], h["c"], h["sc"], h["bias"], h["act"])
        return s["c"] if s["sc"] is None else (s["c"], s["sc"])
    if c["op"] == "quant":
        cb.quantize_e4m3(1, c["N"], c["K"], c["brows"], h["x"], h["q"], h["s"])
        return s["q"], s["s"]
    if c["op"] == "norm":
        cb.norm_residual(c["nb"], c["N"], c["C"], h["x"], h["h"], h["post"], 1.0, h["ls"], h["gate"], h["r"], h["pre"], h["scale"],
                         h["shift"], h["y"], h["s"])
        return (s["r"], s["y"]) if s["s"] is None else (s["r"], s["y"], s["s"])
    cb.rope_rotate_axes(c["nb"], c["N"], c["heads"], c["hd"], c["rot"], h["layout"], h["axes"], h["x"], h["y"], h["cs"], c["npos"],
                        h["pos"], h["grid"])
    return s["y"]


def run(s):
    if own:
        return _own(s)
    return {"gemm": _plain_gemm, "quant": _plain_quant, "norm": _plain_norm, "rope": _plain_rope}[s["case"]["op"]](s)


# ------------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    if case["op"] == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        kb = _ceil(K, BLOCK)
        scales = M * kb + _ceil(N, BLOCK) * kb * SIZE[case["wscale"]] + (M * _ceil(N, BLOCK) if case["out"] == "e4m3" else 0)
        return {"bytes": float(M * K + N * K + scales + M * N * SIZE[case["out"]] + (4 * N if case["bias"] else 0)), "flops": 2.0 * M * N * K}
    if case["op"] == "quant":
        n = case["N"] * case["K"]
        return {"bytes": float(n * (SIZE[case["dt"]] + 1) + _ceil(case["N"], case["brows"]) * _ceil(case["K"], BLOCK)), "flops": 2.0 * n}
    if case["op"] == "norm":
        rows, C = case["nb"] * case["N"], case["C"]
        n = rows * C
        each = 2 * SIZE[case["dt"]] + SIZE[case["hdt"]] + SIZE[case["out"]] + (SIZE[case["hdt"]] if case["gate"] == "row" else 0)
        vectors = 4 * C * ((case["nb"] if case["gate"] == "sample" else 0) + (2 * case["nb"] if case["mod"] else 0) + (1 if case["ls"] else 0) +
                           sum((2 if case["nbias"] else 1) for k in ("post", "pre") if case[k] != "none"))
        return {"bytes": float(n * each + vectors + (rows * _ceil(C, BLOCK) if case["out"] == "e4m3" else 0)), "flops": 12.0 * n}
    rows = case["nb"] * case["N"]
    n = rows * case["heads"] * case["hd"]
    axes = len(_widths(case))
    if case["pos"] == "grid":
        table, pos = max(case["t"], case["h"], case["w"]) * case["rot"] * 4.0, 0.0
    else:
        table, pos = min(case["npos"], rows) * case["rot"] * 4.0, 4.0 * rows * axes
    return {"bytes": 2.0 * n * SIZE[case["dt"]] + table + pos, "flops": 3.0 * rows * case["heads"] * case["rot"]}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_quant(x, brows):
    """x [rows, cols] in 64 bits as (values in units of their block's scale, scales): the definition before the rounding to 8 bits."""
    n, k = x.shape
    up = torch.empty(_ceil(n, brows), _ceil(k, BLOCK), dtype=torch.float64, device=x.device)
    for j in range(up.shape[1]):
        col = x[:, j * BLOCK : (j + 1) * BLOCK].abs().amax(1)
        if brows == 1:
            up[:, j] = col
        else:
            for i in range(up.shape[0]):
                up[i, j] = col[i * brows : (i + 1) * brows].max()
    least = torch.full_like(up, 2.0 ** -126)
    m, e = torch.frexp(up / 448.0)  # the power of two at or above up / 448
    s = torch.maximum(torch.pow(2.0, (e - (m == 0.5).int()).double()), least)
    return x / s.repeat_interleave(brows, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k], s


def _exact_normed(v, kind, g, b):
    if kind == "none":
        return v
    var, mean = torch.var_mean(v, -1, correction=0, keepdim=True)
    if kind == "rms":
        out = v / torch.sqrt(var + mean ** 2 + 1e-5)
    else:
        out = (v - mean) / torch.sqrt(var + 1e-5)
    out = out * g.double()
    return out if b is None else out + b.double()


def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        z = torch.zeros(M, N, dtype=f64, device="cuda")
        for j in range(_ceil(K, BLOCK)):
            k = slice(j * BLOCK, min(K, (j + 1) * BLOCK))
            w = s["b"][:, k].to(f64) * s["sb"][:, j].to(f64).repeat_interleave(BLOCK)[:N, None]
            z += (s["a"][:, k].to(f64) * s["sa"][:, j, None].to(f64)) @ w.t()
        if s["bias"] is not None:
            z += s["bias"].to(f64)
        if case["act"] == "gelu":
            z = z * torch.special.ndtr(z)
        elif case["act"] == "relu":
            z = z.clamp_min(0.0)
        return _exact_quant(z, 1) if case["out"] == "e4m3" else z
    if case["op"] == "quant":
        return _exact_quant(s["x"].to(f64), case["brows"])
    if case["op"] == "norm":
        nb, N, C = case["nb"], case["N"], case["C"]
        mod = None if s["mod"] is None else s["mod"].to(f64).view(nb, 1, 3, C)
        f = torch.ones(1, 1, C, dtype=f64, device="cuda")
        if s["ls"] is not None:
            f = f * s["ls"].to(f64)
        if case["gate"] != "none":
            f = f * (mod[:, :, 0] if case["gate"] == "sample" else s["gate"].to(f64))
        r = torch.addcmul(s["x"].to(f64), f, _exact_normed(s["h"].to(f64), case["post"], s["post_g"], s["post_b"]))
        y = _exact_normed(r, case["pre"], s["pre_g"], s["pre_b"])
        if case["mod"]:
            y = y + y * mod[:, :, 1] + mod[:, :, 2]
        if case["out"] != "e4m3":
            return r, y
        q, e = _exact_quant(y.reshape(nb * N, C), 1)
        return r, q.view(nb, N, C), e.view(nb, N, -1)
    nb, N, h, hd, rot = (case[k] for k in ("nb", "N", "heads", "hd", "rot"))
    y = s["x"][..., : h * hd].reshape(nb, N, h, hd).to(f64)
    n = torch.arange(N, device="cuda")
    dims = [d for d in (case["t"], case["h"], case["w"])][3 - len(_widths(case)) :]
    for j, axis in enumerate(_axis_of_pairs(case)):
        if s["pos"] is not None:
            at = s["pos"][:, :, axis].long()
        else:
            at = (n // math.prod(dims[axis + 1 :]) % dims[axis]).expand(nb, N)
        inside = (at >= 0) & (at < case["npos"])
        t = s["cs"][torch.where(inside, at, 0), j].to(f64)
        t = torch.where(inside[..., None], t, torch.tensor([1.0, 0.0], dtype=f64, device="cuda"))
        turn = torch.complex(t[..., 0].contiguous(), t[..., 1].contiguous())[:, :, None]
        i0, i1 = (2 * j, 2 * j + 1) if case["layout"] == "pairs" else (j, rot // 2 + j)
        z = torch.complex(y[..., i0].contiguous(), y[..., i1].contiguous()) * turn
        y[..., i0], y[..., i1] = z.real, z.imag
    return y
