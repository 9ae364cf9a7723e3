"""Cases that time and check the operators around prompt-conditioned attention: rotary positions (the table of angles and
the rotation of rows), cross attention over an encoder's states of another length, and group norm with an activation over
channels-last maps.

`own` selects between two forms of the same pass: the plain one in elementary torch operations (32 bits, 64 for angles,
rounded once at the end) and the calls a program makes of the library's entry points. `listed()` are the fixed cases,
`draw()` gives further ones of the same ranges, `prepare()` makes a case's inputs on the GPU from a seed, `run()` is one pass,
`work()` what the pass cannot do without, and `exact()` the operator's definition in 64 bits.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ACT = {"none": 0, "gelu": 1, "relu": 2}
SCALING = {"none": 0, "linear": 1, "base": 2, "ramp": 3}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # One coarse map after a prompt's features were added: the smallest call, latency counts.
        dict(name="gn_small", op="groupnorm", nb=1, npix=24 * 24, C=64, groups=8, dt="f32", act="relu"),
        # The mask head's pixel decoder at its finest level for four crops: 288 x 288 pixels, 256 channels, 8 groups.
        dict(name="gn_pixel_decoder", op="groupnorm", nb=4, npix=288 * 288, C=256, groups=8, dt="bf16", act="relu"),
        # Ragged map, groups of ten channels (no 16-byte vector fits a group).
        dict(name="gn_ragged", op="groupnorm", nb=3, npix=77 * 61, C=320, groups=32, dt="f16", act="gelu"),
        # The table of a model run past the length it was trained on: far positions, per-frequency scaling.
        dict(name="rope_table_long", op="rope_table", npos=131072, rot=128, first=65536, theta=500000.0, scaling="ramp",
             factor=16.0, orig=8192.0, amp=1.2772588722239782),
        # One new token for each of eight sequences, queries and shared keys in one fused row.
        dict(name="rope_step", op="rope_rotate", nb=8, N=1, heads=20, hd=64, rot=64, layout="halves", dt="bf16", extra=256,
             npos=8192, pos="random"),
        # Queries and keys of eight crops' 72 x 72 tokens, rotated out of the fused q | k | v rows.
        dict(name="rope_trunk", op="rope_rotate", nb=8, N=5184, heads=24, hd=64, rot=64, layout="pairs", dt="bf16", extra=768,
             npos=5184, pos="rows"),
        # Part of the head is rotated, some rows (positions outside the table) are left as they are, odd row count.
        dict(name="rope_partial", op="rope_rotate", nb=3, N=3001, heads=7, hd=80, rot=32, layout="halves", dt="f32", extra=0,
             npos=4096, pos="excluded"),
        # One query row per sequence over an encoder's states of eight lengths, four query heads to a key head.
        dict(name="xa_step", op="cross_attend", nb=8, Nq=1, Nk=1500, heads=16, kvheads=4, hd=64, dt="bf16", fill=0.6,
             masked=0.0, empty=False),
        # Image tokens of eight crops over the prompt's tokens: few keys, some of them padding.
        dict(name="xa_prompt", op="cross_attend", nb=8, Nq=5184, Nk=39, heads=8, kvheads=8, hd=32, dt="bf16", fill=1.0,
             masked=0.25, empty=True),
        # The detector's 201 queries over the image tokens of eight crops.
        dict(name="xa_queries", op="cross_attend", nb=8, Nq=201, Nk=5184, heads=8, kvheads=8, hd=32, dt="f16", fill=1.0,
             masked=0.0, empty=False),
        # Two crops' tokens over another map's tokens: the largest product.
        dict(name="xa_long", op="cross_attend", nb=2, Nq=5184, Nk=5184, heads=16, kvheads=16, hd=64, dt="bf16", fill=0.9,
             masked=0.0, empty=False),
        # The same kind of call in the library's own 32-bit buffers.
        dict(name="xa_f32", op="cross_attend", nb=2, Nq=201, Nk=5184, heads=8, kvheads=8, hd=32, dt="f32", fill=0.9,
             masked=0.1, empty=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_once(rng):
    op = rng.choice(["groupnorm", "groupnorm", "rope_table", "rope_rotate", "rope_rotate", "cross_attend", "cross_attend",
                     "cross_attend"])
    dt = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "groupnorm":
        groups = rng.choice([1, 4, 8, 16, 32])
        C = groups * rng.choice([1, 2, 3, 4, 8, 10, 12, 16, 32])
        return dict(op=op, nb=rng.randint(1, 9), npix=_log_int(rng, 1, 288 * 288), C=C, groups=groups, dt=dt,
                    act=rng.choice(["none", "gelu", "relu"]))
    if op == "rope_table":
        return dict(op=op, npos=_log_int(rng, 1, 131072), rot=2 * rng.randint(1, 64), first=rng.choice([0, rng.randint(0, 2000000)]),
                    theta=rng.choice([10000.0, 500000.0]), scaling=rng.choice(["none", "linear", "base", "ramp"]),
                    factor=float(rng.choice([2, 4, 16])), orig=float(rng.choice([2048, 8192])), amp=rng.choice([1.0, 1.2]))
    if op == "rope_rotate":
        hd = rng.choice([16, 32, 64, 72, 80, 96, 128])
        return dict(op=op, nb=rng.randint(1, 9), N=_log_int(rng, 1, 8192), heads=rng.randint(1, 32), hd=hd,
                    rot=rng.choice([hd, hd, hd // 2, 2 * rng.randint(1, hd // 2)]), layout=rng.choice(["pairs", "halves"]),
                    dt=dt, extra=rng.choice([0, hd, 4 * hd]), npos=rng.choice([8192, 16384]),
                    pos=rng.choice(["rows", "random", "excluded"]))
    kv = rng.choice([1, 2, 4, 8])
    hd = rng.choice([16, 32, 64, 64, 80, 128])
    return dict(op=op, nb=rng.randint(1, 9), Nq=rng.choice([1, _log_int(rng, 1, 5184)]), Nk=_log_int(rng, 1, 8192),
                heads=kv * rng.choice([1, 1, 2, 4]), kvheads=kv, hd=hd, dt=dt, fill=rng.choice([1.0, 0.6, 0.3]),
                masked=rng.choice([0.0, 0.0, 0.25]), empty=rng.random() < 0.25)


def _cost(case):
    """(bytes, flops, elements of the plain form's largest intermediate) for the bound on drawn cases."""
    w = work(case)
    big = case["nb"] * case["heads"] * case["Nq"] * case["Nk"] if case["op"] == "cross_attend" else 0
    return w["bytes"], w["flops"], big


def draw(rng):
    while True:
        case = _draw_once(rng)
        nbytes, flops, big = _cost(case)
        # No more than the largest listed cases; 32-bit attention no more than a quarter of their products.
        most = 4.5e10 if case.get("dt") == "f32" else 1.9e11
        if nbytes <= 3.4e8 and flops <= most and big <= 8.5e8:
            return case


# ------------------------------------------------------------------------------------------------ inputs
def _key_lengths(case):
    """Valid keys of each sequence, spread evenly between 2 fill - 1 (at least a tenth) and one; prepare() permutes them."""
    nb, Nk, fill = case["nb"], case["Nk"], case["fill"]
    lo = max(0.1, 2.0 * fill - 1.0)
    out = []
    for i in range(nb):
        f = lo + (1.0 - lo) * ((i + 0.5) / nb) if fill < 1.0 else 1.0
        out.append(max(1, min(Nk, int(round(f * Nk)))))
    if case["empty"] and nb > 1:
        out[0] = 0
    return out


def _masked_keys(case):
    return min(case["Nk"] - 1, int(round(case["masked"] * case["Nk"])))


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _frequencies(case):
    """Angle per position of each pair, in 64 bits on the host."""
    rot, theta, kind, factor = case["rot"], case["theta"], case["scaling"], case["factor"]
    half = rot // 2
    if kind == "base" and rot > 2:
        theta = theta * factor ** (rot / (rot - 2.0))
    inv = [theta ** (-2.0 * j / rot) for j in range(half)]
    if kind == "linear":
        return [w / factor for w in inv]
    if kind == "ramp":
        def at(turns):
            return rot * math.log(case["orig"] / (2.0 * math.pi * turns)) / (2.0 * math.log(case["theta"]))
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        keep = [1.0 - min(1.0, max(0.0, (j - lo) / max(hi - lo, 1e-3))) for j in range(half)]
        return [w * k + w / factor * (1.0 - k) for w, k in zip(inv, keep)]
    return inv


def prepare(case, seed):
    g = _gen(seed)
    dev = "cuda"
    s = {"case": case}
    if case["op"] == "groupnorm":
        nb, n, C, dt = case["nb"], case["npix"], case["C"], DT[case["dt"]]
        # Activations with a mean of their own per channel, as a convolution with bias leaves them.
        mean = torch.randn(C, device=dev, generator=g)
        s["x"] = torch.randn(nb, n, C, device=dev, generator=g).add_(mean).to(dt)
        s["gamma"] = 1.0 + 0.2 * torch.randn(C, device=dev, generator=g)
        s["beta"] = 0.2 * torch.randn(C, device=dev, generator=g)
        s["y"] = torch.empty_like(s["x"])
    elif case["op"] == "rope_table":
        # Nothing but sizes and scalars enters this operator; the seed moves the first position.
        s["first"] = case["first"] + int(seed) % 1009
        s["cs"] = torch.empty(case["npos"], case["rot"] // 2, 2, device=dev)
    elif case["op"] == "rope_rotate":
        nb, N, h, hd, rot, dt = case["nb"], case["N"], case["heads"], case["hd"], case["rot"], DT[case["dt"]]
        ld = h * hd + case["extra"]
        s["x"] = torch.randn(nb, N, ld, device=dev, generator=g).to(dt)
        s["y"] = torch.empty(nb, N, h, hd, device=dev, dtype=dt)
        inv = 10000.0 ** (-torch.arange(0, rot, 2, device=dev, dtype=torch.float64) / rot)
        ang = torch.arange(case["npos"], device=dev, dtype=torch.float64)[:, None] * inv
        s["cs"] = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()
        if case["pos"] == "rows":
            s["pos"] = None
        else:
            p = torch.randint(0, case["npos"], (nb, N), device=dev, generator=g, dtype=torch.int32)
            if case["pos"] == "excluded":
                out = torch.rand(nb, N, device=dev, generator=g) < 0.1
                p = torch.where(out, torch.full_like(p, -1), p)
            s["pos"] = p
    else:
        nb, Nq, Nk, h, kv, hd, dt = (case[k] for k in ("nb", "Nq", "Nk", "heads", "kvheads", "hd", "dt"))
        dt = DT[dt]
        s["q"] = torch.randn(nb, Nq, h, hd, device=dev, generator=g).to(dt)
        # Keys and values as one projection leaves them: k | v in one row.
        s["kv"] = torch.randn(nb, Nk, 2 * kv, hd, device=dev, generator=g).to(dt)
        s["o"] = torch.empty_like(s["q"])
        lens = torch.tensor(_key_lengths(case), dtype=torch.int32)
        order = torch.randperm(nb, generator=torch.Generator().manual_seed(int(seed) & 0x7FFFFFFF))
        s["klen"] = lens[order].to(dev) if case["fill"] < 1.0 or case["empty"] else None
        s["kmask"] = None
        if _masked_keys(case) > 0:
            rank = torch.rand(nb, Nk, device=dev, generator=g).argsort(1).argsort(1)
            s["kmask"] = (rank < _masked_keys(case)).to(torch.uint8)
    return s


# ------------------------------------------------------------------------------------------------ the plain form
def _plain_groupnorm(s):
    c = s["case"]
    nb, n, C, G = c["nb"], c["npix"], c["C"], c["groups"]
    x = s["x"].float().view(nb, n, G, C // G)
    mean = x.mean((1, 3), keepdim=True)
    d = x - mean
    var = (d * d).mean((1, 3), keepdim=True)
    y = (d * torch.rsqrt(var + 1e-5)).view(nb, n, C) * s["gamma"] + s["beta"]
    if c["act"] == "gelu":
        y = 0.5 * y * (1.0 + torch.erf(y * 0.7071067811865476))
    elif c["act"] == "relu":
        y = torch.relu(y)
    return y.to(s["x"].dtype)


def _plain_table(s):
    c = s["case"]
    w = torch.tensor(_frequencies(c), dtype=torch.float64, device="cuda")
    p = torch.arange(s["first"], s["first"] + c["npos"], dtype=torch.float64, device="cuda")
    a = p[:, None] * w
    return (torch.stack([a.cos(), a.sin()], -1) * c["amp"]).float()


def _turned(x, cos, sin, rot, layout):
    """x [nb, N, heads, hd]; cos, sin [nb or 1, N, 1, rot / 2]."""
    if layout == "pairs":
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        r = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = x[..., : rot // 2], x[..., rot // 2 : rot]
        r = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([r, x[..., rot:]], -1)


def _plain_rotate(s):
    c = s["case"]
    nb, N, h, hd = c["nb"], c["N"], c["heads"], c["hd"]
    x = s["x"][..., : h * hd].view(nb, N, h, hd)
    if s["pos"] is None:
        cs, keep = s["cs"][:N][None], None
    else:
        keep = (s["pos"] >= 0) & (s["pos"] < c["npos"])
        cs = s["cs"][s["pos"].clamp(0, c["npos"] - 1).long()]
    y = _turned(x.float(), cs[..., 0][:, :, None], cs[..., 1][:, :, None], c["rot"], c["layout"]).to(x.dtype)
    return y if keep is None else torch.where(keep[:, :, None, None], y, x)


def _visible(s, nb, Nk):
    """[nb, Nk] truth values: which keys a sequence's queries see."""
    see = torch.ones(nb, Nk, dtype=torch.bool, device="cuda")
    if s["klen"] is not None:
        see &= torch.arange(Nk, device="cuda")[None] < s["klen"][:, None]
    if s["kmask"] is not None:
        see &= s["kmask"] == 0
    return see


def _plain_attend(s):
    c = s["case"]
    nb, Nq, Nk, h, kv, hd = (c[k] for k in ("nb", "Nq", "Nk", "heads", "kvheads", "hd"))
    see = _visible(s, nb, Nk)
    q = s["q"].float().view(nb, Nq, kv, h // kv, hd).permute(0, 2, 3, 1, 4).reshape(nb * kv, h // kv * Nq, hd)
    k = s["kv"][:, :, :kv].float().permute(0, 2, 3, 1).reshape(nb * kv, hd, Nk)
    v = torch.where(see[:, :, None, None], s["kv"][:, :, kv:].float(), 0.0).permute(0, 2, 1, 3).reshape(nb * kv, Nk, hd)
    a = torch.bmm(q, k).mul_(1.0 / math.sqrt(hd)).view(nb, kv, h // kv * Nq, Nk)
    a.masked_fill_(~see[:, None, None], float("-inf"))
    m = a.amax(-1, keepdim=True)
    a.sub_(torch.where(m == float("-inf"), 0.0, m)).exp_()
    t = a.sum(-1, keepdim=True)
    o = torch.bmm(a.view(nb * kv, -1, Nk), v).view(nb, kv, h // kv * Nq, hd)
    o = torch.where(t > 0, o / t, 0.0)
    return o.view(nb, kv, h // kv, Nq, hd).permute(0, 3, 1, 2, 4).reshape(nb, Nq, h, hd).to(s["q"].dtype)


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
    if c["op"] == "groupnorm":
        n, C = c["npix"], c["C"]
        h["x"], h["y"] = (cb.bmat(cb.wrap(s[k]), 0, C, n * C) for k in ("x", "y"))
        h["g"], h["b"] = cb.wrap(s["gamma"]), cb.wrap(s["beta"])
        h["act"] = ACT[c["act"]]
    elif c["op"] == "rope_table":
        h["cs"] = cb.wrap(s["cs"])
        h["scaling"] = sb.RopeScaling(theta=c["theta"], kind=SCALING[c["scaling"]], factor=c["factor"], orig_len=c["orig"],
                                      turns_fast=32.0, turns_slow=1.0, amplitude=c["amp"])
    elif c["op"] == "rope_rotate":
        N, w = c["N"], c["heads"] * c["hd"]
        ld = w + c["extra"]
        h["x"] = cb.bmat(cb.wrap(s["x"]), 0, ld, N * ld, c["hd"])
        h["y"] = cb.bmat(cb.wrap(s["y"]), 0, w, N * w, c["hd"])
        h["cs"] = cb.wrap(s["cs"])
        h["pos"] = None if s["pos"] is None else cb.wrap(s["pos"])
        h["layout"] = sb.ROPE_PAIRS if c["layout"] == "pairs" else sb.ROPE_HALVES
    else:
        wq, wk = c["heads"] * c["hd"], 2 * c["kvheads"] * c["hd"]
        kv = cb.wrap(s["kv"])
        h["q"], h["o"] = (cb.bmat(cb.wrap(s[k]), 0, wq, c["Nq"] * wq, c["hd"]) for k in ("q", "o"))
        h["k"] = cb.bmat(kv, 0, wk, c["Nk"] * wk, c["hd"])
        h["v"] = cb.bmat(kv, wk // 2, wk, c["Nk"] * wk, c["hd"])
        h["klen"], h["kmask"] = (None if s[k] is None else cb.wrap(s[k]) for k in ("klen", "kmask"))
        h["scale"] = 1.0 / math.sqrt(c["hd"])
    return h


def run(s):
    c = s["case"]
    op = c["op"]
    if own:
        if "h" not in s:
            s["h"] = _handles(s)
        h, cb = s["h"], _lib["cb"]
        if op == "groupnorm":
            cb.groupnorm(c["nb"], c["npix"], c["C"], c["groups"], h["x"], h["y"], h["g"], h["b"], 1e-5, h["act"])
            return s["y"]
        if op == "rope_table":
            cb.rope_table(c["npos"], c["rot"], s["first"], h["scaling"], h["cs"])
            return s["cs"]
        if op == "rope_rotate":
            cb.rope_rotate(c["nb"], c["N"], c["heads"], c["hd"], c["rot"], h["layout"], h["x"], h["y"], h["cs"], c["npos"],
                           h["pos"])
            return s["y"]
        cb.cross_attend(c["nb"], c["Nq"], c["Nk"], c["heads"], c["kvheads"], c["hd"], h["q"], h["k"], h["v"], h["o"],
                        h["klen"], h["kmask"], h["scale"])
        return s["o"]
    if op == "groupnorm":
        return _plain_groupnorm(s)
    if op == "rope_table":
        return _plain_table(s)
    if op == "rope_rotate":
        return _plain_rotate(s)
    return _plain_attend(s)


# ------------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if case["op"] == "groupnorm":
        n = case["nb"] * case["npix"] * case["C"]
        return {"bytes": 2.0 * n * size[case["dt"]] + 8.0 * case["C"], "flops": 8.0 * n}
    if case["op"] == "rope_table":
        n = case["npos"] * (case["rot"] // 2)
        return {"bytes": 8.0 * n, "flops": 2.0 * n}
    if case["op"] == "rope_rotate":
        rows = case["nb"] * case["N"]
        n = rows * case["heads"] * case["hd"]
        table = min(case["npos"], case["N"] if case["pos"] == "rows" else rows) * case["rot"] * 4.0
        return {"bytes": 2.0 * n * size[case["dt"]] + table + (0.0 if case["pos"] == "rows" else 4.0 * rows),
                "flops": 3.0 * rows * case["heads"] * case["rot"]}
    keys = sum(_key_lengths(case)) * (1.0 - _masked_keys(case) / case["Nk"])
    q = case["nb"] * case["Nq"] * case["heads"] * case["hd"]
    return {"bytes": size[case["dt"]] * (2.0 * q + 2.0 * keys * case["kvheads"] * case["hd"]),
            "flops": 4.0 * case["Nq"] * keys * case["heads"] * case["hd"]}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_frequencies(case):
    rot, f = case["rot"], case["factor"]
    j = torch.arange(rot // 2, dtype=torch.float64)
    base = case["theta"] * (f ** (rot / (rot - 2)) if case["scaling"] == "base" and rot > 2 else 1.0)
    w = torch.exp(-2.0 * j / rot * math.log(base))
    if case["scaling"] == "linear":
        w = w / f
    if case["scaling"] == "ramp":
        # The pair that makes n turns over the trained length has the index rot / 2 * log_theta(orig / (2 pi n)).
        pair = [rot / 2.0 * math.log(case["orig"] / (2.0 * math.pi * n), case["theta"]) for n in (32.0, 1.0)]
        first, last = max(0, math.floor(pair[0])), min(rot - 1, math.ceil(pair[1]))
        share = ((j - first) / max(last - first, 0.001)).clamp(0.0, 1.0)
        w = w * (1.0 - share * (1.0 - 1.0 / f))
    return w.tolist()


def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "groupnorm":
        nb, n, C, G = case["nb"], case["npix"], case["C"], case["groups"]
        y = torch.empty(nb, n, C, dtype=f64, device="cuda")
        for i in range(nb):
            for k in range(G):
                cols = slice(k * (C // G), (k + 1) * (C // G))
                x = s["x"][i, :, cols].to(f64)
                var, mean = torch.var_mean(x, correction=0)
                z = (x - mean) / torch.sqrt(var + 1e-5) * s["gamma"][cols].to(f64) + s["beta"][cols].to(f64)
                if case["act"] == "gelu":
                    z = z * torch.special.ndtr(z)
                y[i, :, cols] = z.clamp_min(0.0) if case["act"] == "relu" else z
        return y
    if case["op"] == "rope_table":
        half = case["rot"] // 2
        out = torch.empty(case["npos"], half, 2, dtype=f64, device="cuda")
        p = torch.arange(case["npos"], dtype=f64, device="cuda") + float(s["first"])
        for j, w in enumerate(_exact_frequencies(case)):
            z = torch.polar(torch.full_like(p, case["amp"]), torch.remainder(p * w, 2.0 * math.pi))
            out[:, j, 0], out[:, j, 1] = z.real, z.imag
        return out
    if case["op"] == "rope_rotate":
        nb, N, h, hd, rot = (case[k] for k in ("nb", "N", "heads", "hd", "rot"))
        y = s["x"][..., : h * hd].reshape(nb, N, h, hd).to(f64)
        t = s["cs"].to(f64)
        t = torch.complex(t[..., 0].contiguous(), t[..., 1].contiguous())
        one = torch.ones(1, rot // 2, dtype=t.dtype, device="cuda")
        t = torch.cat([t, one])  # the last row turns by nothing
        if s["pos"] is None:
            idx = torch.arange(N, device="cuda").expand(nb, N)
        else:
            idx = s["pos"].long()
            idx = torch.where((idx < 0) | (idx >= case["npos"]), case["npos"], idx)
        for i in range(h):
            a, b = (y[:, :, i, 0:rot:2], y[:, :, i, 1:rot:2]) if case["layout"] == "pairs" else (
                y[:, :, i, : rot // 2], y[:, :, i, rot // 2 : rot])
            z = torch.complex(a.contiguous(), b.contiguous()) * t[idx]
            a.copy_(z.real)
            b.copy_(z.imag)
        return y
    nb, Nq, Nk, h, kv, hd = (case[k] for k in ("nb", "Nq", "Nk", "heads", "kvheads", "hd"))
    o = torch.zeros(nb, Nq, h, hd, dtype=f64, device="cuda")
    for i in range(nb):
        at = torch.arange(Nk if s["klen"] is None else int(s["klen"][i]), device="cuda")
        if s["kmask"] is not None:
            at = at[s["kmask"][i, at] == 0]
        if at.numel() == 0:
            continue
        for j in range(h):
            k = s["kv"][i, at, j // (h // kv)].to(f64)
            v = s["kv"][i, at, kv + j // (h // kv)].to(f64)
            p = torch.softmax(s["q"][i, :, j].to(f64) @ k.t() / math.sqrt(hd), -1)
            o[i, :, j] = p @ v
    return o
