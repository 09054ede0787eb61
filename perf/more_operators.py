"""Operators of video transformer blocks beside the 8-bit linears, as calls of this package and as plain formulas.

* ``fp4``     linear on microscaled 4-bit values, the activation quantised in the call; with ``train`` also the activation gradient
* ``qk``      norm of every head of queries and keys with the rotation by position; with ``train`` also all gradients
* ``axial``   rotation of queries and keys by positions with several axes (time, height, width); with ``train`` also both gradients

Definitions, as far as they are choices.

4 bits: values 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives, rounded to nearest, halves to the even code, beyond 6 to 6.

* "mxfp4": blocks of 32 along a row share a power of two, 2^(floor(log2 absmax) - 2), held as its exponent, -127 at least.
* "nvfp4": blocks of 16 share an e4m3 scale, rows an fp32 scale.  In fp32, each operation rounded: the row's scale is r = A / 2688
  (= 6 * 448) with A the row's absmax; a block of absmax a has the scale s = e4m3(a * (448 / A)) and its values are rounded from
  x * (1 / (s * r)); a block with s = 0 holds zeros.

The weight is held in 4 bits, quantised by rows of input channels in the same way; the product adds in fp32, scales, adds the bias, takes
the tanh-GELU where the case says so, and rounds once.  In the backward pass (weights are frozen) the gradient is quantised per token and the
de-quantised weight (fp32) per input channel to e4m3 with the factor 448 / absmax, as the 8-bit linears do.

Norm: x / sqrt(mean(x^2) + eps) * weight over a head's channels, unrounded into the rotation.  Rotation: pair i of the rotated channels turns by
position[axis(i)] * frequency(i); channel 2i is paired with 2i + 1 ("interleaved") or i with i + rotated / 2 ("half").  With the "own" spectrum an
axis of c channels has the frequencies base^(-2j/c), with the "shared" one pair i has base^(-2i/rotated) whatever its axis.
"""
import math

import torch

own = False

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
E4M3 = torch.float8_e4m3fn
EPS = 1e-6
_TYPES = {"bf16": BF16, "fp16": F16, "fp32": F32}
_BLOCK = {"mxfp4": 32, "nvfp4": 16}


# ------------------------------------------------------------------------------------------ the cases

def _fp4(fmt, dtype, m, k, n, gelu, train):
    return {"kind": "fp4", "format": fmt, "dtype": dtype, "m": m, "k": k, "n": n, "gelu": gelu, "train": train}


def _qk(dtype, b, s, hq, hk, d, axes, layout, affine, train):
    """axes: channels of each axis as text, "64" or "16,24,24"; together the rotated ones."""
    return {"kind": "qk", "dtype": dtype, "b": b, "s": s, "hq": hq, "hk": hk, "d": d, "axes": axes, "layout": layout, "spectrum": "own",
            "positions": "int64", "affine": affine, "train": train}


def _axial(dtype, b, s, hq, hk, d, axes, layout, spectrum, positions, train):
    return {"kind": "axial", "dtype": dtype, "b": b, "s": s, "hq": hq, "hk": hk, "d": d, "axes": axes, "layout": layout,
            "spectrum": spectrum, "positions": positions, "train": train}


def listed():
    cases = {
        # one token (a modulation vector, a generated token) through an up projection: the weights are all there is to read
        "fp4_token_nv": _fp4("nvfp4", "bf16", 1, 2048, 8192, False, False),
        # a text encoder's layer on one prompt of odd length
        "fp4_prompt_mx": _fp4("mxfp4", "fp16", 77, 4096, 10240, True, False),
        # the tokens of one clip through the down projection
        "fp4_clip_mx": _fp4("mxfp4", "bf16", 6144, 8192, 2048, False, False),
        # the largest: four clips through the up projection with its activation
        "fp4_clips_nv": _fp4("nvfp4", "bf16", 24576, 2048, 8192, True, False),
        # fine-tuning step on two short clips of odd length, output and activation gradient; a width that no tile divides
        "fp4_train_nv": _fp4("nvfp4", "bf16", 2002, 2048, 5504, False, True),
        # one generated token of eight requests, grouped heads
        "qk_token": _qk("bf16", 8, 1, 32, 8, 128, "128", "half", True, False),
        # the tokens of one clip with the framework's heads, positions in time, height and width
        "qk_clip": _qk("bf16", 1, 6144, 32, 32, 64, "16,24,24", "interleaved", True, False),
        # odd prompt lengths, two fifths of a head rotated; output and all gradients
        "qk_train_odd": _qk("fp16", 3, 1001, 20, 4, 80, "8,12,12", "half", True, True),
        # training step over long sequences
        "qk_train": _qk("bf16", 2, 8192, 32, 8, 128, "32,48,48", "interleaved", True, True),
        # the patches of one image of odd size in a vision encoder
        "axial_image": _axial("fp16", 1, 1023, 16, 16, 72, "36,36", "half", "own", "int32", False),
        # the tokens of one clip at fractional places in time and space
        "axial_clip": _axial("bf16", 1, 6144, 32, 32, 64, "16,24,24", "interleaved", "own", "float32", False),
        # training step over long sequences of text, images and video in one spectrum
        "axial_train": _axial("bf16", 2, 8192, 32, 8, 128, "32,48,48", "half", "shared", "int64", True),
    }
    return [{"name": name, **c} for name, c in cases.items()]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _split(rng, r, axes):
    """r channels on so many axes, each an even number of them."""
    if axes == 1:
        return str(r)
    if axes == 2:
        first = r // 4 * 2 if rng.random() < 0.6 else 2 * rng.randint(1, r // 2 - 1)
        return f"{first},{r - first}"
    time = max(2, r // 8 * 2) if rng.random() < 0.6 else 2 * rng.randint(1, r // 2 - 2)
    height = max(2, (r - time) // 4 * 2)
    return f"{time},{height},{r - time - height}"


def draw(rng):
    kind = rng.choice(["fp4", "qk", "axial"])
    if kind == "fp4":
        train = rng.random() < 0.35
        k = rng.choice([1024, 2048, 4096, 8192]) if rng.random() < 0.4 else 32 * _log_int(rng, 2, 320)
        n = rng.choice([2048, 4096, 8192, 10240]) if rng.random() < 0.4 else 16 * _log_int(rng, 4, 640)
        m = max(1, min(_log_int(rng, 1, 24576), 24576 * 2048 * 8192 // (k * n) // (4 if train else 1)))
        return _fp4(rng.choice(["mxfp4", "nvfp4"]), rng.choice(["bf16", "bf16", "fp16"]), m, k, n, rng.random() < 0.4 and not train, train)
    d = rng.choice([64, 64, 72, 80, 96, 128, 128, 192, 256])
    r = d if rng.random() < 0.6 else 2 * rng.randint(3, d // 2)
    axes = rng.choice([1, 2, 3, 3]) if kind == "qk" else rng.choice([2, 3, 3])
    hk = rng.choice([1, 2, 4, 8, 16, 32])
    hq = hk * rng.choice([1, 1, 2, 4, 5, 8])
    b = rng.choice([1, 1, 2, 3, 8, 64])
    s = 1 if rng.random() < 0.2 else max(1, min(_log_int(rng, 2, 8192), 2 * 8192 * 40 * 128 // (2 * b * (hq + hk) * d)))
    dtype, layout = rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.choice(["half", "interleaved"])
    if kind == "qk":
        return _qk(dtype, b, s, hq, hk, d, _split(rng, r, axes), layout, rng.random() < 0.8, rng.random() < 0.5)
    return _axial(dtype, b, s, hq, hk, d, _split(rng, r, axes), layout, rng.choice(["own", "shared"]),
                  rng.choice(["int32", "int64", "float32", "float64"]), rng.random() < 0.4)


# ------------------------------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _activations(g, rows, dim):
    """~N(0,1) with 0.1 % of the channels twenty times as large."""
    x = _randn(g, rows, dim)
    x[:, torch.randperm(dim, generator=g, device="cuda")[:max(1, dim // 1000)]] *= 20.0
    return x


def _sections(case):
    return [int(c) for c in case["axes"].split(",")]


def _positions(case, g):
    """Places of the tokens: clips of frames of 16:9 that each begin at a time of their own; one axis: the end of a sequence."""
    b, s, axes = case["b"], case["s"], len(_sections(case))
    start = torch.randint(0, 4096, (b, 1), generator=g, device="cuda")
    i = torch.arange(s, device="cuda").expand(b, s)
    if axes == 1:
        return start * 8 + i
    area = s if axes == 2 else max(1, s // 13)
    width = max(1, round(math.sqrt(area * 16 / 9)))
    height = max(1, -(-area // width))
    place = [i // width % height, i % width] if axes == 2 else [start + i // (height * width), i // width % height, i % width]
    p = torch.stack(place, -1)
    if case["positions"].startswith("float"):                   # seconds at 25 frames a second, centres of patches in pixels
        p = (p.double() + 0.5) * torch.tensor(([0.04] if axes == 3 else []) + [32.0, 32.0], dtype=torch.float64, device="cuda")
    return p.to(getattr(torch, case["positions"]))


def _inputs(case, seed):
    g = _gen(seed)
    t = _TYPES[case["dtype"]]
    if case["kind"] == "fp4":
        m, k, n = case["m"], case["k"], case["n"]
        s = {"x": _activations(g, m, k).to(t), "w": (_randn(g, n, k) * 0.02).to(t), "bias": _randn(g, n) * 0.02}
        if case["train"]:
            s["g"] = (_randn(g, m, n) * 0.1).to(t)
        return s
    b, n, hq, hk, d = (case[i] for i in ("b", "s", "hq", "hk", "d"))
    # queries and keys as they lie in the output of a joint projection, tokens of different sizes
    qkv = (_randn(g, b, n, hq + 2 * hk, d) * (0.5 + 2.0 * torch.rand(b, n, 1, 1, generator=g, device="cuda"))).to(t)
    s = {"q": qkv[:, :, :hq], "k": qkv[:, :, hq:hq + hk], "positions": _positions(case, g)}
    if case["kind"] == "qk" and case["affine"]:
        s["wq"], s["wk"] = 1.0 + 0.1 * _randn(g, d), 1.0 + 0.1 * _randn(g, d)
    if case["train"]:
        s["gq"], s["gk"] = (_randn(g, b, n, hq, d) * 0.1).to(t), (_randn(g, b, n, hk, d) * 0.1).to(t)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    return _prepare_own(s) if own else _prepare_plain(s)


# ------------------------------------------------------------------------------------------ the package's calls

def _prepare_own(s):
    c = s["case"]
    if c["kind"] == "fp4":
        from q8_kernels_b200.modules import FP4Linear
        full = torch.nn.Linear(c["k"], c["n"], device="cuda", dtype=s["w"].dtype)         # a checkpoint's layer
        full.weight.data, full.bias.data = s.pop("w"), s.pop("bias")
        s["linear"] = FP4Linear.from_linear(full, c["format"])
        s["leaves"] = [s["x"]]
    else:
        from q8_kernels_b200.modules import AxialRotaryEmbedding, HeadNormRotary, RotaryEmbedding
        sections = _sections(c)
        rotary = (RotaryEmbedding(c["d"], sections[0], layout=c["layout"]) if len(sections) == 1
                  else AxialRotaryEmbedding(c["d"], sections, layout=c["layout"], spectrum=c["spectrum"]))
        s["leaves"] = [s["q"], s["k"]]
        if c["kind"] == "qk":
            s["module"] = HeadNormRotary(c["d"], rotary, eps=EPS, elementwise_affine=c["affine"]).cuda()
            if c["affine"]:
                s["module"].q_weight.data, s["module"].k_weight.data = s["wq"], s["wk"]
                s["leaves"] += [s["module"].q_weight, s["module"].k_weight]
        else:
            s["module"] = rotary.cuda()
    if c["train"]:
        for leaf in s["leaves"]:
            leaf.requires_grad_(True)
    else:
        for leaf in s["leaves"]:
            leaf.requires_grad_(False)
    return s


def _run_own(s):
    c = s["case"]
    if c["kind"] == "fp4":
        y = s["linear"](s["x"], fuse_gelu=c["gelu"])
        return (y.detach(), torch.autograd.grad(y, s["leaves"], s["g"])[0]) if c["train"] else y
    q, k = s["module"](s["q"], s["k"], s["positions"])
    if not c["train"]:
        return q, k
    return (q.detach(), k.detach()) + torch.autograd.grad([q, k], s["leaves"], [s["gq"], s["gk"]])


# ------------------------------------------------------------------------------------------ the plain forms

def _to_fp4(y):
    """fp32 to the nearest 4-bit value, halves to the even code."""
    a = y.abs()
    v = 0.5 * (a > 0.25) + 0.5 * (a >= 0.75) + 0.5 * (a > 1.25) + 0.5 * (a >= 1.75) + (a > 2.5) + (a >= 3.5) + 2.0 * (a > 5.0)
    return torch.where(y < 0, -v, v)


def _blocks(x, fmt):
    """Rows x [rows, k] in fp32 as 4-bit values (in fp32), the scales of their blocks [rows, k / block] and of the rows [rows, 1]."""
    rows, k = x.shape
    v = x.view(rows, k // _BLOCK[fmt], _BLOCK[fmt])
    a = v.abs().amax(dim=2)
    if fmt == "mxfp4":
        e = (torch.frexp(a)[1] - 3).clamp(min=-127)             # frexp: a = f 2^e with f in [0.5, 1)
        e = torch.where(a > 0, e, torch.full_like(e, -127))
        scale = torch.where(e > -127, (e + 127) << 23, torch.full_like(e, 1 << 22)).view(F32)        # 2^e
        q = _to_fp4(v * ((127 - e) << 23).view(F32).unsqueeze(2))
        return q.view(rows, k), scale, torch.ones(rows, 1, device=x.device)
    top = a.amax(dim=1, keepdim=True)
    r = top / torch.full_like(top, 2688.0)
    scale = (a * torch.where(top > 0, torch.full_like(top, 448.0) / top, torch.zeros_like(top))).to(E4M3).float()
    unit = scale * r
    inverse = torch.where(scale > 0, torch.ones_like(unit) / unit, torch.zeros_like(unit))
    return _to_fp4(v * inverse.unsqueeze(2)).view(rows, k), scale, r


def _spread(q, scale):
    rows, k = q.shape
    return (q.view(rows, scale.shape[1], -1) * scale.unsqueeze(2)).view(rows, k)


def _rows_e4m3(x):
    """Rows as e4m3 values (in fp32) and what each stands for."""
    amax = x.abs().amax(dim=1, keepdim=True)
    factor = torch.where(amax > 0, torch.full_like(amax, 448.0) / amax, torch.zeros_like(amax))
    return (x * factor).to(E4M3).float(), torch.where(amax > 0, torch.ones_like(amax) / factor, torch.zeros_like(amax))


def _plain_fp4(s):
    c = s["case"]
    t = s["x"].dtype
    q, qs, qr = _blocks(s["x"].float(), c["format"])
    w = _spread(s["wq"].float() * 0.5, s["wscale"])
    y = (_spread(q, qs) @ w.T) * (qr * s["wr"].T) + s["bias"]
    if c["gelu"]:
        y = 0.5 * y * (1.0 + torch.tanh(0.7978845608028654 * (y + 0.044715 * y * y * y)))
    if not c["train"]:
        return y.to(t)
    g, gs = _rows_e4m3(s["g"].float())
    wt, wts = _rows_e4m3((w * s["wr"]).T)
    return y.to(t), ((g @ wt.T) * (gs * wts.T)).to(t)


def _frequencies(case):
    """Radians per position of each pair, and the pair's axis."""
    sections, freq, axis = _sections(case), [], []
    i = torch.arange(sum(sections) // 2, device="cuda", dtype=torch.float64)
    for n, c in enumerate(sections):
        freq.append(10000.0 ** (-2.0 * i[:c // 2] / c))
        axis += [n] * (c // 2)
    freq = torch.cat(freq) if case["spectrum"] == "own" else 10000.0 ** (-2.0 * i / sum(sections))
    return freq, torch.tensor(axis, device="cuda")


def _prepare_plain(s):
    c = s["case"]
    if c["kind"] == "fp4":                                      # the weight as a program holds it: values (doubled) and scales
        q, s["wscale"], s["wr"] = _blocks(s.pop("w").float(), c["format"])
        s["wq"] = (2.0 * q).to(torch.int8)
    else:
        s["freq"], s["axis"] = _frequencies(c)
    return s


def _turn(x, cos, sin, layout):
    """x in fp32 with its first channels turned."""
    r = 2 * cos.shape[-1]
    y = x.clone()
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if layout == "interleaved" else (x[..., :r // 2], x[..., r // 2:r])
    a, b = a * cos - b * sin, b * cos + a * sin
    if layout == "interleaved":
        y[..., 0:r:2], y[..., 1:r:2] = a, b
    else:
        y[..., :r // 2], y[..., r // 2:r] = a, b
    return y


def _plain_qk(s):
    c, t = s["case"], s["q"].dtype
    p = s["positions"].double()
    p = p[..., s["axis"]] if p.dim() == 3 else p.unsqueeze(-1)
    angle = (p * s["freq"]).unsqueeze(2)                        # far positions need 64 bits
    cos, sin = angle.cos().float(), angle.sin().float()
    outs, grads, weights = [], [], []
    for x, w, g in ((s["q"], s.get("wq"), s.get("gq")), (s["k"], s.get("wk"), s.get("gk"))):
        z = x.float()
        if c["kind"] == "qk":
            rstd = torch.rsqrt((z * z).mean(dim=-1, keepdim=True) + EPS)
            z = z * rstd
        outs.append(_turn(z if w is None else z * w, cos, sin, c["layout"]).to(t))
        if c["train"]:
            d = _turn(g.float(), cos, -sin, c["layout"])
            if c["kind"] == "qk":
                if w is not None:
                    weights.append((d * z).double().sum(dim=(0, 1, 2)).float())     # a sum over all tokens and heads
                    d = d * w
                d = rstd * (d - z * (d * z).mean(dim=-1, keepdim=True))
            grads.append(d.to(t))
    return tuple(outs + grads + weights)


def run(state):
    if own:
        return _run_own(state)
    return _plain_fp4(state) if state["case"]["kind"] == "fp4" else _plain_qk(state)


# ------------------------------------------------------------------------------------------ what it takes

def work(case):
    if case["kind"] == "fp4":
        m, k, n = case["m"], case["k"], case["n"]
        w = {"bytes": 2 * m * k + n * k // 2 + n * k // _BLOCK[case["format"]] + 8 * n + 2 * m * n, "flops": 2 * m * n * k}
        if case["train"]:                                       # the output's gradient comes in, the input's goes out
            w = {"bytes": w["bytes"] + 2 * m * n + 2 * m * k, "flops": 2 * w["flops"]}
        return w
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    tokens, heads, axes = case["b"] * case["s"], case["hq"] + case["hk"], _sections(case)
    passes = 2 if case["train"] else 1                          # forward reads x and writes y; backward takes the gradient to dx
    place = {"int32": 4, "float32": 4, "int64": 8, "float64": 8}[case["positions"]] * len(axes) * tokens
    flops = tokens * heads * (3 * sum(axes) + (4 * case["d"] if case["kind"] == "qk" else 0))
    return {"bytes": passes * 2 * tokens * heads * case["d"] * size + place + 4 * sum(axes) + 16 * case["d"], "flops": passes * flops}


# ------------------------------------------------------------------------------------------ in 64 bits

def _grid64(x, fmt):
    """What rows of x stand for once they are in 4 bits.  Scales and values go by fp32 where the definition does; the nearest value is looked up."""
    x = x.float()
    rows, k = x.shape
    v = x.reshape(rows, -1, _BLOCK[fmt])
    a = v.abs().max(dim=2).values
    if fmt == "mxfp4":
        exponent = ((a.view(torch.int32) >> 23) - 127 - 2).clamp(min=-127).double()
        unit = torch.exp2(exponent)
        y = v.double() / unit.unsqueeze(2)
    else:
        top = a.max(dim=1).values.unsqueeze(1)
        r = torch.div(top, torch.tensor(2688.0, device="cuda").expand_as(top))
        s = torch.mul(a, torch.nan_to_num(torch.div(torch.tensor(448.0, device="cuda").expand_as(top), top), posinf=0.0)).to(E4M3).float()
        inverse = torch.div(torch.tensor(1.0, device="cuda").expand_as(s), s * r)
        y = torch.nan_to_num((v * inverse.unsqueeze(2)), nan=0.0, posinf=0.0, neginf=0.0).double()
        unit = s.double() * r.double()
    values = torch.tensor([0.0, 1.0, 2.0, 4.0, 0.5, 1.5, 3.0, 6.0], dtype=torch.float64, device="cuda")      # even codes first: they win ties
    best, away = torch.zeros_like(y), torch.full_like(y, math.inf)
    for w in values:
        far = (y.abs() - w).abs()
        best, away = torch.where(far < away, w, best), torch.minimum(far, away)
    return (best * y.sign() * unit.unsqueeze(2)).reshape(rows, k)


def _rows64(x):
    """What rows of fp32 values stand for in e4m3."""
    amax = x.abs().max(dim=1).values.unsqueeze(1)
    factor = torch.div(torch.tensor(448.0, device="cuda").expand_as(amax), amax)
    return torch.nan_to_num((x * factor).to(E4M3).double() / factor.double(), nan=0.0)


def _exact_fp4(case, s):
    w = _grid64(s["w"], case["format"])
    y = _grid64(s["x"], case["format"]) @ w.T + s["bias"].double()
    if case["gelu"]:
        y = torch.nn.functional.gelu(y, approximate="tanh")
    if not case["train"]:
        return y
    return y, _rows64(s["g"].float()) @ _rows64(w.T.float()).T


def _exact_qk(case, s):
    sections, total = _sections(case), sum(_sections(case))
    freq, axis, i = [], [], 0
    for n, c in enumerate(sections):
        for j in range(c // 2):
            freq.append(math.exp(math.log(10000.0) * (-2.0 * j / c if case["spectrum"] == "own" else -2.0 * i / total)))
            axis.append(n)
            i += 1
    p = s["positions"].double()
    p = p[..., None] if p.dim() == 2 else p
    angle = torch.stack([p[..., n] * f for n, f in zip(axis, freq)], dim=-1)[:, :, None]
    rot = torch.polar(torch.ones_like(angle), angle)
    first, second = (torch.arange(0, total, 2), torch.arange(1, total, 2)) if case["layout"] == "interleaved" else \
        (torch.arange(total // 2), torch.arange(total // 2, total))

    def forward(x, w):
        if case["kind"] == "qk":
            x = x / torch.sqrt(x.square().mean(dim=-1, keepdim=True) + EPS)
            x = x if w is None else x * w
        z = torch.complex(x[..., first], x[..., second]) * rot
        out = x.clone()
        out[..., first], out[..., second] = z.real, z.imag
        return out

    with torch.set_grad_enabled(case["train"]):
        names = ["q", "k"] + (["wq", "wk"] if "wq" in s else [])
        leaf = {n: s[n].double().detach().requires_grad_(case["train"]) for n in names}
        outs = [forward(leaf["q"], leaf.get("wq")), forward(leaf["k"], leaf.get("wk"))]
        if not case["train"]:
            return tuple(outs)
        return tuple(o.detach() for o in outs) + torch.autograd.grad(outs, [leaf[n] for n in names], [s["gq"].double(), s["gk"].double()])


def exact(case, seed):
    with torch.no_grad():
        s = _inputs(case, seed)
        return _exact_fp4(case, s) if case["kind"] == "fp4" else _exact_qk(case, s)
