"""Operators of transformer blocks beside the 8-bit linears, as calls of this package and as plain formulas.

* ``gated``   gate and up projection with 8-bit weights, ``act(gate) * up``; with ``train`` also the activation gradient
* ``rotary``  rotary embedding of queries and keys from positions; with ``train`` also both gradients
* ``norm``    layer norm with weight and bias; with ``train`` also the gradients of input, weight and bias

Definitions, as far as they are choices.  Activations are quantised per token (int8: halves away from zero, rotated by the
Sylvester-Hadamard matrix and rounded to bf16 before; e4m3: nearest even), weights are held in 8 bits with one scale per
output channel, gate rows first.  Between forward and backward pass gate and up are held in bf16.  The backward pass quantises
the gradient of gate and up per token, and the de-quantised weight per input channel, to e4m3.  The quantiser is the package's:
``top / absmax`` and its product with each value are rounded to fp32 before the value is rounded to 8 bits.
"""
import math

import torch

own = False

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
E4M3 = torch.float8_e4m3fn
_TYPES = {"bf16": BF16, "fp16": F16, "fp32": F32}


# ------------------------------------------------------------------------------------------ the cases

def _gated(dtype, m, k, f, act, rotate, train):
    return {"kind": "gated", "dtype": dtype, "m": m, "k": k, "f": f, "act": act, "rotate": rotate, "train": train}


def _rotary(dtype, b, s, hq, hk, d, r, layout, scaling, last, train):
    return {"kind": "rotary", "dtype": dtype, "b": b, "s": s, "hq": hq, "hk": hk, "d": d, "r": r, "layout": layout,
            "scaling": scaling, "last": last, "train": train}


def _norm(dtype, rows, dim, train):
    return {"kind": "norm", "dtype": dtype, "rows": rows, "dim": dim, "train": train}


def listed():
    cases = {
        # one generated token through the gated projections of a layer: the weights are all there is to read
        "gated_token_int8": _gated("int8", 1, 2048, 8192, "gelu_tanh", True, False),
        # a text encoder's layer on one prompt of odd length, FP8 without rotation
        "gated_encoder_fp8": _gated("fp8", 77, 4096, 10240, "gelu_tanh", False, False),
        # the tokens of one clip: the tensor cores bound it
        "gated_clip_int8": _gated("int8", 6144, 2048, 8192, "silu", True, False),
        # fine-tuning step on two short clips of odd length, output and activation gradient; a width that no tile divides
        "gated_train_int8": _gated("int8", 2002, 2048, 5504, "silu", True, True),
        # the largest: fine-tuning step on one clip
        "gated_train_fp8": _gated("fp8", 6144, 2048, 8192, "silu", False, True),
        # one generated token of eight requests far into a long context, grouped heads, positions scaled by frequency
        "rotary_token": _rotary("bf16", 8, 1, 32, 8, 128, 128, "half", "yarn", 131071, False),
        # the tokens of one clip, the framework's heads and pair layout
        "rotary_clip": _rotary("bf16", 1, 6144, 32, 32, 64, 64, "interleaved", "none", 6143, False),
        # odd prompt lengths, a third of each head rotated
        "rotary_part_fp16": _rotary("fp16", 3, 1001, 20, 4, 96, 32, "half", "linear", 4003, False),
        # training step over long sequences
        "rotary_train": _rotary("bf16", 2, 8192, 32, 8, 128, 128, "half", "ntk", 32767, True),
        # the norm before one generated token's projections
        "norm_token": _norm("bf16", 1, 2048, False),
        # odd sizes, every row off the vector boundary
        "norm_train_odd": _norm("fp16", 1001, 1537, True),
        # training step over four clips
        "norm_train": _norm("bf16", 24576, 2048, True),
    }
    return [{"name": name, **c} for name, c in cases.items()]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["gated", "rotary", "norm"])
    if kind == "gated":
        dtype = rng.choice(["int8", "fp8"])
        rotate = dtype == "int8" or rng.random() < 0.3
        k = rng.choice([512, 1024, 2048, 4096]) if rotate else 16 * _log_int(rng, 16, 320)
        f = 16 * _log_int(rng, 16, 640) if rng.random() < 0.6 else rng.choice([2048, 4096, 8192, 10240])
        m = min(_log_int(rng, 1, 6144), 6144 * 2048 * 8192 // (k * f))
        return _gated(dtype, m, k, f, rng.choice(["silu", "gelu_tanh"]), rotate, rng.random() < 0.4)
    if kind == "rotary":
        d = rng.choice([64, 64, 80, 96, 128, 128, 192, 256])
        r = d if rng.random() < 0.5 else 2 * rng.randint(1, d // 2)
        hk = rng.choice([1, 2, 4, 8, 16, 32])
        hq = hk * rng.choice([1, 1, 2, 4, 5, 8])
        b = rng.choice([1, 1, 2, 3, 8, 64])
        s = 1 if rng.random() < 0.3 else max(1, min(_log_int(rng, 2, 8192), 2 * 8192 * 40 * 128 // (2 * b * (hq + hk) * d)))
        last = _log_int(rng, max(s, 2), 1 << 20)
        return _rotary(rng.choice(["bf16", "bf16", "fp16", "fp32"]), b, s, hq, hk, d, r, rng.choice(["half", "interleaved"]),
                       rng.choice(["none", "linear", "ntk", "yarn"]) if r > 2 else "none", last, rng.random() < 0.4)
    dim = rng.choice([512, 768, 1024, 1536, 2048, 4096, 8192]) if rng.random() < 0.5 else _log_int(rng, 16, 10240)
    rows = max(1, min(_log_int(rng, 1, 32768), 24576 * 2048 // (2 * dim)))
    return _norm(rng.choice(["bf16", "bf16", "fp16", "fp32"]), rows, dim, rng.random() < 0.5)


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


def _weight(g, n, k, dtype):
    """A checkpoint's weight: 8-bit values and one scale per row."""
    w = _randn(g, n, k) * 0.02
    top = 127.0 if dtype == "int8" else 448.0
    amax = w.abs().amax(dim=1)
    q = w * (top / amax).unsqueeze(1)
    return (q.round().to(torch.int8) if dtype == "int8" else q.to(E4M3)), amax / top


def _scaling(case):
    """What a user writes down for the positions' scaling."""
    return {"none": None, "linear": {"type": "linear", "factor": 4.0}, "ntk": {"type": "ntk", "factor": 8.0},
            "yarn": {"type": "yarn", "factor": 32.0, "original_length": 4096}}[case["scaling"]]


def _inputs(case, seed):
    g = _gen(seed)
    if case["kind"] == "gated":
        m, k, f = case["m"], case["k"], case["f"]
        w, ws = _weight(g, 2 * f, k, case["dtype"])
        s = {"x": _activations(g, m, k).to(BF16), "w": w, "ws": ws, "bias": _randn(g, 2 * f) * 0.02}
        if case["train"]:
            s["g"] = (_randn(g, m, f) * 0.1).to(BF16)
        return s
    t = _TYPES[case["dtype"]]
    if case["kind"] == "rotary":
        b, n, hq, hk, d = (case[i] for i in ("b", "s", "hq", "hk", "d"))
        # queries and keys as they lie in the output of a joint projection
        qkv = _randn(g, b, n, hq + 2 * hk, d).to(t)
        # every sequence ends at its own place, the longest at `last`
        end = torch.randint(n - 1, case["last"] + 1, (b, 1), generator=g, device="cuda")
        end[0] = case["last"]
        s = {"q": qkv[:, :, :hq], "k": qkv[:, :, hq:hq + hk], "positions": end - torch.arange(n - 1, -1, -1, device="cuda")}
        if case["train"]:
            s["gq"], s["gk"] = (_randn(g, b, n, hq, d) * 0.1).to(t), (_randn(g, b, n, hk, d) * 0.1).to(t)
        return s
    rows, dim = case["rows"], case["dim"]
    s = {"x": (_activations(g, rows, dim) + 0.5 * _randn(g, rows, 1)).to(t), "w": 1.0 + 0.1 * _randn(g, dim),
         "b": 0.1 * _randn(g, dim)}
    if case["train"]:
        s["g"] = (_randn(g, rows, dim) * 0.1).to(t)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["kind"] == "rotary":
        if own:
            from q8_kernels_b200.modules import RotaryEmbedding
            s["rotary"] = RotaryEmbedding(case["d"], case["r"], layout=case["layout"], scaling=_scaling(case)).cuda()
        else:
            s["freq"], s["amplitude"] = _frequencies(case)
    elif case["kind"] == "gated" and not own and case["rotate"]:
        s["h"] = _hadamard(case["k"], F32)
    if own and case["train"]:
        for name in {"gated": ("x",), "rotary": ("q", "k"), "norm": ("x", "w", "b")}[case["kind"]]:
            s[name].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------ the package's calls

def _run_own(s):
    c = s["case"]
    if c["kind"] == "gated":
        from q8_kernels_b200.functional.gated import fp8_gated_linear, q8_gated_linear
        if c["dtype"] == "int8":
            y = q8_gated_linear(s["x"], s["w"], s["bias"], None, s["ws"], c["act"])
        else:
            y = fp8_gated_linear(s["x"], s["w"], s["bias"], None, s["ws"], c["act"], c["rotate"])
        return (y.detach(), torch.autograd.grad(y, [s["x"]], s["g"])[0]) if c["train"] else y
    if c["kind"] == "rotary":
        q, k = s["rotary"](s["q"], s["k"], s["positions"])
        if c["train"]:
            return (q.detach(), k.detach()) + torch.autograd.grad([q, k], [s["q"], s["k"]], [s["gq"], s["gk"]])
        return q, k
    from q8_kernels_b200.functional.layer_norm import layer_norm
    y = layer_norm(s["x"], s["w"], s["b"], 1e-5)
    if c["train"]:
        return (y.detach(),) + torch.autograd.grad(y, [s["x"], s["w"], s["b"]], s["g"])
    return y


# ------------------------------------------------------------------------------------------ the plain forms

def _hadamard(n, dtype):
    """Sylvester-Hadamard matrix over sqrt(n), n a power of two."""
    h = torch.ones(1, 1, device="cuda", dtype=dtype)
    while h.shape[0] < n:
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    return h * n ** -0.5


def _quantise(x, dtype):
    """Rows as 8-bit values (held in fp32) and their scales."""
    amax = x.abs().amax(dim=1, keepdim=True)
    scale = (127.0 if dtype == "int8" else 448.0) / amax
    y = torch.where(amax > 0, x * scale, torch.zeros_like(x))
    q = torch.sign(y) * torch.floor(y.abs() + 0.5) if dtype == "int8" else y.to(E4M3).float()
    return q, 1.0 / scale


def _act(g, act):
    if act == "silu":
        return g / (1.0 + torch.exp(-g))
    u = 0.7978845608028654 * (g + 0.044715 * g * g * g)
    return 0.5 * g * (1.0 + torch.tanh(u))


def _act_grad(g, act):
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return s * (1.0 + g * (1.0 - s))
    t = torch.tanh(0.7978845608028654 * (g + 0.044715 * g * g * g))
    return 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * 0.7978845608028654 * (1.0 + 3.0 * 0.044715 * g * g)


def _plain_gated(s):
    c, f = s["case"], s["case"]["f"]
    x, w = s["x"].float(), s["w"].float()
    if c["rotate"]:
        x = (x @ s["h"]).to(BF16).float()          # the rotated activation is a bf16 tensor
    q, qs = _quantise(x, c["dtype"])
    y = (q @ w.T) * (qs * s["ws"]) + s["bias"]
    gate, up = y[:, :f], y[:, f:]
    h = (_act(gate, c["act"]) * up).to(BF16)
    if not c["train"]:
        return h
    gate, up, g = gate.to(BF16).float(), up.to(BF16).float(), s["g"].float()
    d, ds = _quantise(torch.cat([g * up * _act_grad(gate, c["act"]), g * _act(gate, c["act"])], 1), "fp8")
    wt, wts = _quantise((w * s["ws"].unsqueeze(1)).T, "fp8")
    dx = (d @ wt.T) * (ds * wts.T)
    return h, (dx @ s["h"] if c["rotate"] else dx).to(BF16)


def _frequencies(case):
    """Radians per position of every pair in 64 bits, and the factor on cosine and sine."""
    r, sc = case["r"], case["scaling"]
    i = torch.arange(r // 2, device="cuda", dtype=torch.float64)
    base = 10000.0 * (8.0 ** (r / (r - 2)) if sc == "ntk" else 1.0)
    freq = base ** (-2.0 * i / r)
    if sc == "linear":
        freq = freq / 4.0
    if sc != "yarn":
        return freq, 1.0
    # pairs that turn more than 32 times within the original length keep their frequency, those that turn less than once
    # are slowed down by the factor, those between by a linear mix over the pair's number
    def pair(turns):
        return r * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(10000.0))
    low, high = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), r - 1)
    slow = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
    return freq * (1 - slow) + freq / 32.0 * slow, 0.1 * math.log(32.0) + 1.0


def _plain_rotary(s):
    c, r = s["case"], s["case"]["r"]
    angle = (s["positions"].double().unsqueeze(-1) * s["freq"]).unsqueeze(2)     # far positions need 64 bits
    cos, sin = (angle.cos() * s["amplitude"]).float(), (angle.sin() * s["amplitude"]).float()

    def turn(x, sin):
        y = x.float().clone()
        a, b = (y[..., 0:r:2], y[..., 1:r:2]) if c["layout"] == "interleaved" else (y[..., :r // 2], y[..., r // 2:r])
        a, b = a * cos - b * sin, b * cos + a * sin
        if c["layout"] == "interleaved":
            y[..., 0:r:2], y[..., 1:r:2] = a, b
        else:
            y[..., :r // 2], y[..., r // 2:r] = a, b
        return y.to(x.dtype)

    out = (turn(s["q"], sin), turn(s["k"], sin))
    return out + (turn(s["gq"], -sin), turn(s["gk"], -sin)) if c["train"] else out


def _plain_norm(s):
    c, x = s["case"], s["x"].float()
    mean = x.mean(dim=1, keepdim=True)
    z = x - mean
    rstd = torch.rsqrt((z * z).mean(dim=1, keepdim=True) + 1e-5)
    z = z * rstd
    y = (z * s["w"] + s["b"]).to(s["x"].dtype)
    if not c["train"]:
        return y
    g = s["g"].float()
    gw = g * s["w"]
    dx = rstd * (gw - gw.mean(dim=1, keepdim=True) - z * (gw * z).mean(dim=1, keepdim=True))
    return y, dx.to(s["x"].dtype), (g * z).sum(dim=0), g.sum(dim=0)


def run(state):
    if own:
        return _run_own(state)
    return {"gated": _plain_gated, "rotary": _plain_rotary, "norm": _plain_norm}[state["case"]["kind"]](state)


# ------------------------------------------------------------------------------------------ what it takes

def work(case):
    if case["kind"] == "gated":
        m, k, n = case["m"], case["k"], 2 * case["f"]
        w = {"bytes": 2 * m * k + n * k + 8 * n + m * n, "flops": 2 * m * n * k}
        if case["train"]:                          # the output's gradient comes in, the input's goes out
            w = {"bytes": w["bytes"] + m * n + 2 * m * k, "flops": 2 * w["flops"]}
        return w
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    if case["kind"] == "rotary":
        tokens, heads = case["b"] * case["s"], case["hq"] + case["hk"]
        passes = 2 if case["train"] else 1
        return {"bytes": passes * 2 * tokens * heads * case["d"] * size + 8 * tokens + 4 * case["r"],
                "flops": passes * tokens * heads * case["r"] * 3}
    n, d = case["rows"] * case["dim"], case["dim"]
    if case["train"]:                              # x and the gradient in, output and gradients out
        return {"bytes": 4 * n * size + 16 * d, "flops": 20 * n}
    return {"bytes": 2 * n * size + 8 * d, "flops": 8 * n}


# ------------------------------------------------------------------------------------------ in 64 bits

def _rows64(x, top, whole):
    """Rows of x on the 8-bit grid: values that stand for x, i.e. with the scale in them.  The grid goes by fp32, as defined: a
    bf16 value may lie on the very border between two steps, where the rounding of the scale decides."""
    x = x.float()
    scale = top / x.abs().amax(dim=1, keepdim=True)
    y = torch.nan_to_num(x * scale, nan=0.0).double()
    y = torch.trunc(y + 0.5 * y.sign()) if whole else y.float().to(E4M3).double()
    return torch.nan_to_num(y / scale.double(), nan=0.0)


def _turned64(x):
    """Butterflies of the Hadamard transform, over sqrt(n)."""
    n, step = x.shape[1], 1
    while step < n:
        a, b = x.view(x.shape[0], -1, 2, step).unbind(2)
        x = torch.stack([a + b, a - b], 2).view(x.shape[0], n)
        step *= 2
    return x / math.sqrt(n)


def _exact_gated(case, s):
    f, int8 = case["f"], case["dtype"] == "int8"
    x, w = s["x"].double(), s["w"].double() * s["ws"].double().unsqueeze(1)
    if case["rotate"]:
        x = _turned64(x).to(BF16).double()
    y = _rows64(x, 127.0 if int8 else 448.0, int8) @ w.T + s["bias"].double()

    def act(g):
        if case["act"] == "silu":
            return g * torch.sigmoid(g)
        return torch.nn.functional.gelu(g, approximate="tanh")

    h = act(y[:, :f]) * y[:, f:]
    if not case["train"]:
        return h
    y = y.to(BF16).double()
    with torch.enable_grad():                      # the gradient of the formula itself
        gate, up = y[:, :f].clone().requires_grad_(True), y[:, f:].clone().requires_grad_(True)
        d = torch.autograd.grad(act(gate) * up, [gate, up], s["g"].double())
    dx = _rows64(torch.cat(d, 1), 448.0, False) @ _rows64(w.T.contiguous(), 448.0, False).T
    return h, _turned64(dx) if case["rotate"] else dx


def _exact_rotary(case, s):
    r, d = case["r"], case["d"]
    base, amplitude, freq = 10000.0, 1.0, []
    if case["scaling"] == "ntk":
        base = base * 8.0 ** (r / (r - 2.0))
    for i in range(r // 2):
        w = math.exp(-2.0 * i / r * math.log(base))
        if case["scaling"] == "linear":
            w /= 4.0
        if case["scaling"] == "yarn":
            lo, hi = (r / 2.0 * math.log(4096 / (2 * math.pi * t)) / math.log(base) for t in (32.0, 1.0))
            lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), r - 1)
            m = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            w = m * w / 32.0 + (1.0 - m) * w
            amplitude = 1.0 + 0.1 * math.log(32.0)
        freq.append(w)
    angle = s["positions"].double()[..., None] * torch.tensor(freq, dtype=torch.float64, device="cuda")
    rot = torch.polar(torch.full_like(angle, amplitude), angle)[:, :, None]
    if case["layout"] == "interleaved":
        first, second = torch.arange(0, r, 2), torch.arange(1, r, 2)
    else:
        first, second = torch.arange(r // 2), torch.arange(r // 2, r)

    def turn(x, rot):
        x = x.double()
        z = torch.complex(x[..., first], x[..., second]) * rot
        out = x.clone()
        out[..., first], out[..., second] = z.real, z.imag
        return out

    out = (turn(s["q"], rot), turn(s["k"], rot))
    return out + (turn(s["gq"], rot.conj()), turn(s["gk"], rot.conj())) if case["train"] else out


def _exact_norm(case, s):
    with torch.enable_grad():
        x, w, b = (s[i].double().requires_grad_(True) for i in ("x", "w", "b"))
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        y = (x - mean) / torch.sqrt(var + 1e-5) * w + b
        if not case["train"]:
            return y.detach()
        return (y.detach(),) + torch.autograd.grad(y, [x, w, b], s["g"].double())


def exact(case, seed):
    with torch.no_grad():
        s = _inputs(case, seed)
        return {"gated": _exact_gated, "rotary": _exact_rotary, "norm": _exact_norm}[case["kind"]](case, s)
