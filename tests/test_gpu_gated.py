"""Gated 8-bit projections against their formulas in 64 bits.

The kernel's products are exact and its sums fp32 (u = 2^-24): a chain of K / 32 partial sums of 32 products, K / 32 + 8 roundings of
the sum of the magnitudes A = sum |a||w| sa sw + |bias|, which bounds the error of gate and up.  act and its derivative are formed of five
or six roundings and two approximate instructions good to 2^-22: 16 u relative in all.  Then one rounding to bf16, whose 8 significant
bits leave eps / 2 = 2^-7 / 2 = 2^-8 of the value.  Quantised values are compared bit by bit with the definition where their input is exact, and by half a step of e4m3 (2^-4 of the
value, 2^-10 of the row's step below its normal range) where it is not.
"""
import pytest
import torch

from helpers import bits

pytestmark = pytest.mark.gpu
BF16, F16, F32, E4M3, I8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn, torch.int8
U = 2.0 ** -24


def act64(g, act):
    return g * torch.sigmoid(g) if act == "silu" else torch.nn.functional.gelu(g, approximate="tanh")


def quantise(x, t):
    """The operators' quantizer on fp32 rows: top * (1 / absmax), each rounded; halves away from zero or nearest even."""
    amax = x.abs().amax(-1, keepdim=True)
    f = torch.reciprocal(amax) * (127.0 if t == I8 else 448.0)
    y = torch.where(amax > 0, x * f, torch.zeros_like(x))
    q = (torch.sign(y).double() * torch.floor(y.double().abs() + 0.5)).to(I8) if t == I8 else y.to(E4M3)
    return q, torch.reciprocal(f).squeeze(-1)


def inputs(m, k, f, t, seed, bias=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(m, k, generator=g, device="cuda")
    x[:, torch.randperm(k, generator=g, device="cuda")[:max(1, k // 1000)]] *= 20
    w, ws = quantise(torch.randn(2 * f, k, generator=g, device="cuda") * k ** -0.5, t)
    return x.to(BF16), w, ws, (0.3 * torch.randn(2 * f, generator=g, device="cuda") if bias else None)


def products(q, qs, w, ws, bias):
    """gate and up in 64 bits, and the bound on their error."""
    f = w.shape[0] // 2
    scale = qs.double().unsqueeze(-1) * ws.double()
    y = (q.double() @ w.double().T) * scale
    size = (q.double().abs() @ w.double().abs().T) * scale
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    err = (q.shape[-1] / 32 + 8) * U * size
    return y[:, :f], y[:, f:], err[:, :f], err[:, f:]


def check_out(out, gate, up, eg, eu, act):
    ref = act64(gate, act) * up
    err = 1.2 * up.abs() * eg + act64(gate, act).abs() * eu + eg * eu + 16 * U * (ref.abs() + gate.abs() * up.abs() * 2.0 ** -20)
    bad = (out.double() - ref).abs() > ref.abs() * 2.0 ** -8 * 1.001 + 1e-38 + 1.01 * err
    assert out.dtype == BF16 and not bad.any(), f"{int(bad.sum())} of {bad.numel()}"


def near_bf16(a, ref, err):
    return ((a.double() - ref).abs() <= ref.abs() * 2.0 ** -8 * 1.001 + 1.01 * err + 1e-38).all()


# rows around the tiles' 128 and 256, columns around 32, 64, 96 and 128 and with tails of 16, K around slabs of 128
SIZES = [(1, 16, 16), (1, 2048, 8192), (3, 48, 32), (16, 512, 48), (77, 272, 144), (128, 128, 128), (129, 1024, 112), (255, 144, 272), (256, 4096, 1408),
         (257, 256, 528), (300, 640, 96), (1001, 2048, 688), (700, 128, 4112), (2002, 512, 5504), (40, 8192, 256)]


@pytest.mark.parametrize("m,k,f", SIZES)
@pytest.mark.parametrize("t", [I8, E4M3])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_products(m, k, f, t, act):
    from q8_kernels_b200 import check_status, native
    x, w, ws, bias = inputs(m, k, f, t, m + k + f)
    q, qs = native.gated_quant(x, False, t)
    gate, up, eg, eu = products(q, qs, w, ws, bias)
    out, pre = native.gated_mm(q, w, bias, qs, ws, act, True)
    check_out(out, gate, up, eg, eu, act)
    assert pre.shape == (m, 2, f) and near_bf16(pre[:, 0], gate, eg) and near_bf16(pre[:, 1], up, eu)
    plain, none = native.gated_mm(q, w, bias, qs, ws, act, False)
    assert none is None and torch.equal(bits(plain), bits(out))
    gate, up, eg, eu = products(q, qs, w, ws, None)
    check_out(native.gated_mm(q, w, None, qs, ws, act)[0], gate, up, eg, eu, act)
    check_status()


@pytest.mark.parametrize("t", [I8, E4M3])
def test_a_row_has_the_same_bits_in_every_call(t):
    from q8_kernels_b200 import native
    x, w, ws, bias = inputs(900, 512, 1056, t, 3)
    q, qs = native.gated_quant(x, False, t)
    whole = native.gated_mm(q, w, bias, qs, ws, "silu", True)
    for a, b in ((0, 1), (5, 140), (100, 900)):
        part = native.gated_mm(q[a:b], w, bias, qs[a:b], ws, "silu", True)
        assert torch.equal(bits(part[0]), bits(whole[0][a:b])) and torch.equal(bits(part[1]), bits(whole[1][a:b]))


def test_extreme_gates():
    """silu and GELU of gates far out: 0 and the gate itself, no NaN; a row of zeros; NaN stays in its row."""
    from q8_kernels_b200 import native
    q = torch.zeros(6, 128, dtype=I8, device="cuda")
    q[0], q[1], q[2, 0], q[3, 0] = 127, -127, 1, -1
    w = torch.full((64, 128), 127, dtype=I8, device="cuda")
    qs = torch.tensor([1e3, 1e3, 1.0, 1.0, 0.0, float("nan")], device="cuda")
    ws = torch.full((64,), 1e2, device="cuda")
    for act in ("silu", "gelu_tanh"):
        out, pre = native.gated_mm(q, w, None, qs, ws, act, True)
        g = pre[:, 0].double()
        assert torch.isfinite(out[:5]).all() and (out[4] == 0).all() and out[5].isnan().all()
        assert (out[1].double().abs() == 0).all() and (out[3].double().abs() <= 1e-30).all()
        assert near_bf16(out[0], (g[0] * pre[0, 1].double()), (g[0] ** 2).abs() * 2.0 ** -7)
        d8, ds = native.gated_backward_quant(torch.ones(5, 32, device="cuda", dtype=BF16), pre[:5].contiguous(), act)
        assert torch.isfinite(d8.float()).all() and torch.isfinite(ds).all() and (d8[4].float() == 0).all() and ds[4] == 0


@pytest.mark.parametrize("rotate", [False, True])
@pytest.mark.parametrize("t", [I8, E4M3])
@pytest.mark.parametrize("k", [16, 128, 256, 512, 2048, 4096, 16384])
def test_activation_quantiser(rotate, t, k):
    from q8_kernels_b200 import native
    x = inputs(37, k, 16, t, k)[0]
    x[5] = 0
    for src in (x, x.to(E4M3)):
        q, s = native.gated_quant(src, rotate, t)
        y = src
        if rotate:
            y = native.fast_hadamard_transform(src, k ** -0.5)     # the rotation by itself, rounded to its input's type
        rq, rs = quantise(y.float(), t)
        assert torch.equal(bits(q), bits(rq)) and torch.equal(bits(s), bits(rs))
    wide = torch.cat([x, x], 1)[:, :k]                          # strided rows
    assert torch.equal(bits(native.gated_quant(wide, rotate, t)[0]), bits(native.gated_quant(x, rotate, t)[0]))


@pytest.mark.parametrize("f,k", [(16, 16), (16, 144), (48, 64), (144, 128), (496, 528), (5504, 2048), (1024, 96)])
@pytest.mark.parametrize("t", [I8, E4M3])
def test_weight_operand(f, k, t):
    from q8_kernels_b200 import native
    _, w, ws, _ = inputs(1, k, f, t, f + k)
    w[:, 3] = 0
    w[0], w[1, 5] = (127 if t == I8 else 448.0), (-128 if t == I8 else -448.0)
    q, s = native.gated_weight_operand(w, ws)
    rq, rs = quantise((w.float() * ws.unsqueeze(1)).T.contiguous(), E4M3)
    assert torch.equal(bits(q), bits(rq)) and torch.equal(bits(s), bits(rs))


@pytest.mark.parametrize("m,f", [(1, 16), (3, 528), (65, 1024), (7, 1040), (9, 2048), (5, 4096), (4, 8192), (3, 8208), (2, 16384)])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_gradient_operand(m, f, act):
    from q8_kernels_b200 import native
    g = torch.Generator(device="cuda").manual_seed(m + f)
    pre = (3 * torch.randn(m, 2, f, generator=g, device="cuda")).to(BF16)
    grad = torch.randn(m, f, generator=g, device="cuda").to(BF16)
    q, s = native.gated_backward_quant(grad, pre, act)
    gate, up = pre[:, 0].double().requires_grad_(True), pre[:, 1].double().requires_grad_(True)
    d = torch.cat(torch.autograd.grad(act64(gate, act) * up, [gate, up], grad.double()), 1)
    size = torch.cat([grad.double().abs() * up.detach().abs(), grad.double().abs() * gate.detach().abs()], 1)   # of the terms that are added
    err = 32 * U * size * 2
    top = d.abs().amax(1, keepdim=True)
    assert ((s.double().unsqueeze(1) * 448 - top).abs() <= top * 4 * U + err.amax(1, keepdim=True)).all()
    bound = d.abs() * 2.0 ** -4 + (top / 448) * 2.0 ** -10
    assert ((q.double() * s.double().unsqueeze(1) - d).abs() <= bound * 1.001 + 2 * err).all()


@pytest.mark.parametrize("kind,rotate", [("int8", True), ("fp8", False), ("fp8", True)])
@pytest.mark.parametrize("m,k,f,act", [(1, 512, 16, "silu"), (77, 1024, 272, "gelu_tanh"), (300, 256, 1040, "silu")])
def test_training(kind, rotate, m, k, f, act):
    from q8_kernels_b200 import native
    from q8_kernels_b200.functional import gated
    from q8_kernels_b200.functional.fast_hadamard import hadamard_transform
    t = I8 if kind == "int8" else E4M3
    x, w, ws, bias = inputs(m, k, f, t, m)
    x.requires_grad_(True)
    grad = torch.randn(m, f, device="cuda").to(BF16)

    def call(a, scale=None):
        return (gated.q8_gated_linear(a, w, bias, scale, ws, act) if kind == "int8"
                else gated.fp8_gated_linear(a, w, bias, scale, ws, act, rotate))

    y = call(x)
    dx, = torch.autograd.grad(y, [x], grad)
    with torch.no_grad():
        q, qs = native.gated_quant(x, rotate, t)
        assert torch.equal(bits(call(x)), bits(y)) and torch.equal(bits(call(q, qs)), bits(y))
        _, pre = native.gated_mm(q, w, bias, qs, ws, act, True)
        g8, gs = native.gated_backward_quant(grad, pre, act)
        w8, wsc = native.gated_weight_operand(w, ws)
    # the product in 64 bits, rounded to bf16, and the rotation back: fp32 sums of K values of about one size, rounded again
    ref = (g8.double() @ w8.double().T) * gs.double().unsqueeze(-1) * wsc.double()
    size = (g8.double().abs() @ w8.double().abs().T) * gs.double().unsqueeze(-1) * wsc.double()
    err = ref.abs() * 2.0 ** -8 + (2 * f / 32 + 8) * U * size
    if rotate:
        h = hadamard_transform(torch.eye(k, device="cuda").to(BF16), scale=1.0).double()
        err = (err @ h.abs()) * k ** -0.5
        ref = (ref @ h) * k ** -0.5
        err = err + 16 * U * err.amax(1, keepdim=True) + ref.abs() * 2.0 ** -8
    assert dx.dtype == BF16 and ((dx.double() - ref).abs() <= err * 1.01 + 1e-38).all()


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_gradient_against_differences(kind, act):
    """The un-quantised function of the de-quantised weight in 64 bits, differenced along the gradient: what the activation's and the
    gradient's 8-bit grids leave.  A value is off by at most 2^-4 of itself (e4m3; int8 less), gate and up by the activation's grid, the
    gradient's and the weight's values by one more each: (1 + 2^-4)^3 - 1 < 0.2 of the whole if all pulled one way."""
    from q8_kernels_b200.functional import gated
    t = I8 if kind == "int8" else E4M3
    m, k, f = 64, 512, 1024
    x, w, ws, bias = inputs(m, k, f, t, 9)
    x.requires_grad_(True)
    grad = torch.randn(m, f, device="cuda").to(BF16)
    y = gated.q8_gated_linear(x, w, bias, None, ws, act) if kind == "int8" else gated.fp8_gated_linear(x, w, bias, None, ws, act)
    dx = torch.autograd.grad(y, [x], grad)[0].double()
    wd = w.double() * ws.double().unsqueeze(1)
    if kind == "int8":                                          # the weight belongs to rotated activations
        from q8_kernels_b200.functional.fast_hadamard import hadamard_transform
        wd = wd @ (hadamard_transform(torch.eye(k, device="cuda").to(BF16), scale=1.0).double() * k ** -0.5)

    def loss(a):
        v = a @ wd.T + bias.double()
        return (act64(v[:, :f], act) * v[:, f:] * grad.double()).sum()

    v = dx / dx.norm()
    h = 1e-4
    diff = (loss(x.detach().double() + h * v) - loss(x.detach().double() - h * v)) / (2 * h)
    assert abs(diff / dx.norm() - 1) <= 0.2


def test_types_shapes_and_zero_rows():
    from q8_kernels_b200.functional import gated
    x, w, ws, bias = inputs(24, 512, 64, I8, 5)
    y = gated.q8_gated_linear(x, w, bias, None, ws)
    assert torch.equal(bits(gated.q8_gated_linear(x.view(2, 3, 4, 512), w, bias, None, ws)), bits(y.view(2, 3, 4, 64)))
    assert torch.equal(bits(gated.q8_gated_linear(x[0], w, bias, None, ws)), bits(y[0]))
    half = x.to(F16).requires_grad_(True)
    z = gated.q8_gated_linear(half, w, bias, None, ws)
    assert z.dtype == BF16 and torch.autograd.grad(z, [half], torch.ones_like(z))[0].dtype == F16
    assert torch.equal(bits(z), bits(gated.q8_gated_linear(half.detach().to(BF16), w, bias, None, ws)))
    assert gated.q8_gated_linear(x.to(E4M3), w, bias, None, ws).shape == (24, 64)
    e = x[:0].detach().requires_grad_(True)
    z = gated.q8_gated_linear(e, w, bias, None, ws)
    assert z.shape == (0, 64) and torch.autograd.grad(z, [e], torch.empty_like(z))[0].shape == (0, 512)
    strided = torch.cat([x, x], 1)[:, :512].detach().requires_grad_(True)
    z = gated.q8_gated_linear(strided, w, bias, None, ws)
    assert torch.equal(bits(z), bits(y))
    g = torch.randn(24, 128, device="cuda").to(BF16)[:, ::2]
    assert torch.equal(bits(torch.autograd.grad(z, [strided], g, retain_graph=True)[0]), bits(torch.autograd.grad(z, [strided], g.contiguous())[0]))


def test_captured_and_on_another_stream():
    from q8_kernels_b200.functional import gated
    x, w, ws, bias = inputs(200, 1024, 528, I8, 6)
    x.requires_grad_(True)
    grad = torch.randn(200, 528, device="cuda").to(BF16)

    def step():
        y = gated.q8_gated_linear(x, w, bias, None, ws, "gelu_tanh")
        return y.detach(), torch.autograd.grad(y, [x], grad)[0]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = step()
        other = step()
    torch.cuda.current_stream().wait_stream(s)
    eager = step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        x.copy_(torch.randn_like(x))
    graph.replay()
    fresh = step()
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(eager, other))
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(out, fresh))


@pytest.mark.parametrize("linear,dim,inner", [("int8", 512, 256), ("fp8", 512, 256), ("fp8", 528, 272)])
def test_modules(linear, dim, inner):
    from q8_kernels_b200.modules import GatedFeedForward, GatedLinear, FP8Linear, Q8Linear
    gate, up = (torch.nn.Linear(dim, inner).cuda().to(BF16) for _ in range(2))
    down = torch.nn.Linear(inner, dim).cuda().to(BF16)
    rotate = dim == 512
    m = GatedLinear.from_linears(gate, up, "gelu_tanh", linear, rotate)
    assert set(m.state_dict()) == {"weight", "bias", "scales"} and m.weight.shape == (2 * inner, dim)
    one = Q8Linear.from_linear(gate) if linear == "int8" else FP8Linear.from_linear(gate, use_hadamard=rotate)
    assert torch.equal(bits(m.weight.data[:inner]), bits(one.weight.data)) and torch.equal(m.scales[:inner], one.scales)
    x = torch.randn(3, 40, dim, device="cuda").to(BF16)
    # 8 bits of weights and activations: int8 rows of N(0,1) have steps of 4 sigma / 127, 1 % rms, e4m3 2.6 %; of both operands of gate and
    # up, of the product and the last weight: at most six of them as squares, and as much again for the sums' cancellation
    bound = 12 ** 0.5 * (0.01 if linear == "int8" else 0.026)
    ref = torch.nn.functional.gelu(gate(x).float(), approximate="tanh") * up(x).float()
    y = m(x)
    assert ((y.float() - ref).norm() / ref.norm()).item() <= bound
    ff = GatedFeedForward.from_linears(gate, up, down, "gelu_tanh", linear)
    assert torch.equal(bits(ff(x)), bits(ff.proj_down(y, out_dtype=BF16)))
    whole = ref @ down.weight.float().T + down.bias.float()
    assert ((ff(x).view_as(whole).float() - whole).norm() / (whole - down.bias.float()).norm()).item() <= bound
    other = GatedFeedForward(dim, inner, "gelu_tanh", linear=linear).cuda()
    other.load_state_dict(ff.state_dict())
    assert torch.equal(bits(other(x)), bits(ff(x)))
    x.requires_grad_(True)
    assert torch.autograd.grad(ff(x).float().sum(), [x])[0].shape == x.shape


def test_modules_refuse():
    from q8_kernels_b200.modules import GatedFeedForward, GatedLinear
    for bad in (lambda: GatedLinear(64, 64, act="relu"), lambda: GatedLinear(64, 64, linear="int4"), lambda: GatedFeedForward(64, 96),
                lambda: GatedFeedForward(96, 64),
                lambda: GatedLinear.from_linears(*(torch.nn.Linear(96, 64).cuda().to(BF16) for _ in range(2)), "silu", "int8"),
                lambda: GatedLinear.from_linears(torch.nn.Linear(64, 64).cuda().to(BF16), torch.nn.Linear(64, 32).cuda().to(BF16))):
        with pytest.raises(ValueError):
            bad()


def test_misaligned_tensors():
    """Dense tensors that begin off the 16 bytes of the kernels' accesses."""
    from q8_kernels_b200 import native
    from q8_kernels_b200.functional import gated
    for m in (5, 40):
        x, w, ws, bias = inputs(m, 512, 64, I8, 8)

        def off(t):
            o = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape)
            return o.copy_(t)

        want = gated.q8_gated_linear(x, w, bias, None, ws)
        leaf = off(x).requires_grad_(True)
        y = gated.q8_gated_linear(leaf, off(w), off(bias), None, off(ws))
        assert torch.equal(bits(y), bits(want))
        q, qs = native.gated_quant(x, True, I8)
        assert torch.equal(bits(gated.q8_gated_linear(off(q), off(w), bias, off(qs), ws)), bits(want))
        y = gated.q8_gated_linear(leaf, w, bias, None, ws)
        g = torch.randn(m, 64, device="cuda").to(BF16)
        assert torch.equal(bits(torch.autograd.grad(y, [leaf], off(g), retain_graph=True)[0]), bits(torch.autograd.grad(y, [leaf], g)[0]))


def test_under_checkpointing():
    from torch.utils.checkpoint import checkpoint
    from q8_kernels_b200.functional import gated, layer_norm
    x, w, ws, bias = inputs(33, 512, 64, I8, 10)
    nw = torch.ones(512, device="cuda", requires_grad=True)
    x.requires_grad_(True)
    g = torch.randn(33, 64, device="cuda").to(BF16)

    def f(a):
        return gated.q8_gated_linear(layer_norm.layer_norm(a, nw), w, bias, None, ws)

    plain = torch.autograd.grad(f(x), [x, nw], g)
    again = torch.autograd.grad(checkpoint(f, x, use_reentrant=False), [x, nw], g)
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(plain, again))


def test_refusals():
    from q8_kernels_b200 import Q8KernelError
    from q8_kernels_b200.functional import gated
    x, w, ws, bias = inputs(4, 64, 32, I8, 7)
    x8, xs = torch.zeros(4, 64, dtype=I8, device="cuda"), torch.zeros(4, device="cuda")
    f8 = w.float().to(E4M3)
    q8, fp8 = gated.q8_gated_linear, gated.fp8_gated_linear
    for bad in (lambda: q8(x, w, bias, None, ws, "relu"), lambda: q8(x, w, bias, None, None), lambda: q8(x, f8, bias, None, ws), lambda: fp8(x, w, bias, None, ws),
                lambda: q8(x[:, :48], w, bias, None, ws), lambda: q8(x, w[:48], bias, None, ws), lambda: q8(x, w, bias[:63], None, ws),
                lambda: q8(x, w, bias.to(BF16), None, ws), lambda: q8(x, w, bias, None, ws[:32]), lambda: q8(x8, w, bias, None, ws),
                lambda: q8(x8, w, bias, xs[:3], ws), lambda: q8(x, w, bias, xs, ws), lambda: fp8(x8, f8, bias, xs, ws), lambda: fp8(x.float(), f8, bias, None, ws),
                lambda: q8(x.float(), w, bias, None, ws), lambda: q8(x.cpu(), w, bias, None, ws), lambda: q8(x, w.cpu(), bias, None, ws),
                lambda: q8(x[:, :24], w[:, :24], bias, None, ws), lambda: q8(x, w.view(64, 8, 8), bias, None, ws)):
        with pytest.raises(Q8KernelError):
            bad()
    big = torch.zeros(2 * 16400, 64, dtype=I8, device="cuda")
    bs = torch.ones(2 * 16400, device="cuda")
    assert q8(x, big, None, None, bs).shape == (4, 16400)
    with pytest.raises(Q8KernelError):                          # refused before the forward pass, not in the backward pass
        q8(x.detach().requires_grad_(True), big, None, None, bs)
