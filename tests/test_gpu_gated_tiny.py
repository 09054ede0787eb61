"""Gated projections of rows, gradients and weight columns whose largest value is below 448 / FLT_MAX, where 448 / absmax has no fp32 value, with
exact zeros among them: no NaN, and the values that the 8-bit grid holds."""
import pytest
import torch

from helpers import bits

pytestmark = pytest.mark.gpu
BF16, F32, E4M3, I8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.int8
TINY = [1.2e-36, 1e-37, 1e-38, 1e-39, 3e-40]                    # the last two are subnormal in bf16 and fp32


def close(q, s, ref, t):
    """q * s against the values that were quantised: half a step of int8; of e4m3 2^-4 of the value, or 2^-10 steps of the row below its normal
    range.  The scale is off by up to 2^-22 of itself at 1 / FLT_MAX (a subnormal number of 22 bits) and the factor by two roundings."""
    step = s.double().unsqueeze(1)
    half = step / 2 if t == I8 else torch.maximum(ref.abs() * 2.0 ** -4, step * 2.0 ** -10)
    return ((q.double() * step - ref).abs() <= half * (1 + 2.0 ** -20) + ref.abs() * 2.0 ** -20).all()


@pytest.mark.parametrize("rotate", [False, True])
@pytest.mark.parametrize("t", [I8, E4M3])
@pytest.mark.parametrize("k", [16, 128, 256, 512, 2048, 4096, 16384])
def test_activations(rotate, t, k):
    from q8_kernels_b200 import native
    x = torch.zeros(len(TINY) + 2, k, device="cuda")
    for i, v in enumerate(TINY):
        x[i, 1], x[i, 5], x[i, k // 2] = v * (k ** 0.5 if rotate else 1.0), -v / 3, v / 7
    x[-2] = torch.randn(k, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    x = x.to(BF16)
    q, s = native.gated_quant(x, rotate, t)
    ref = native.fast_hadamard_transform(x, k ** -0.5).double() if rotate else x.double()
    assert torch.isfinite(q.float()).all() and torch.isfinite(s).all() and (s[:-1] > 0).all() and s[-1] == 0 and (q[-1].float() == 0).all()
    assert close(q[:-1], s[:-1], ref[:-1], t)


@pytest.mark.parametrize("m", [7, 8, 40])
@pytest.mark.parametrize("k", [128, 512, 2048])
@pytest.mark.parametrize("kind", ["int8", "fp8", "fp8_rotated"])
def test_projections(m, k, kind):
    """A product of such a row vanishes against the bias: the output of a row of zeros."""
    from q8_kernels_b200 import native
    from q8_kernels_b200.functional import gated
    g = torch.Generator(device="cuda").manual_seed(k)
    t = I8 if kind == "int8" else E4M3
    f = 64
    w, ws = native.tokenwise_quant(torch.randn(2 * f, k, generator=g, device="cuda").to(BF16), t)
    bias = torch.randn(2 * f, generator=g, device="cuda")
    x = torch.zeros(m, k, device="cuda")
    for i, v in enumerate(TINY):
        x[i, 1], x[i, k // 2] = v, -v / 3
    x = x.to(BF16).requires_grad_(True)
    y = gated.q8_gated_linear(x, w, bias, None, ws) if t == I8 else gated.fp8_gated_linear(x, w, bias, None, ws, "silu", kind != "fp8")
    assert torch.isfinite(y).all() and torch.equal(bits(y), bits(y[-1:].expand_as(y).contiguous()))
    # gradients of that size, single values among zeros and whole rows
    grad = torch.zeros(m, f, device="cuda")
    for i, v in enumerate(TINY):
        grad[i, 3] = v
    grad[5] = 1e-37 * torch.randn(f, generator=g, device="cuda")
    dx = torch.autograd.grad(y, [x], grad.to(BF16))[0]
    # |dx| <= sum of gradient * up * act' * w, all but the first a few units: less than 1e-33 of 64 * 2048 terms
    assert torch.isfinite(dx).all() and (dx.abs() < 1e-33).all() and (dx[5] != 0).any() and (dx[6:] == 0).all()


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("f", [16, 528, 2048, 16384])
def test_gradient_operand(f, act):
    from q8_kernels_b200 import native
    g = torch.Generator(device="cuda").manual_seed(f)
    m = len(TINY)
    pre = torch.randn(m, 2, f, generator=g, device="cuda").to(BF16)
    pre[:, :, f // 2] = 2.0
    grad = torch.zeros(m, f, device="cuda")
    for i, v in enumerate(TINY):
        grad[i, f // 2], grad[i, 0] = v, v / 5
    grad = grad.to(BF16)
    q, s = native.gated_backward_quant(grad, pre, act)
    gate, up = pre[:, 0].double().requires_grad_(True), pre[:, 1].double().requires_grad_(True)
    a = gate * torch.sigmoid(gate) if act == "silu" else torch.nn.functional.gelu(gate, approximate="tanh")
    ref = torch.cat(torch.autograd.grad(a * up, [gate, up], grad.double()), 1)
    assert torch.isfinite(q.float()).all() and torch.isfinite(s).all() and (s > 0).all()
    step = s.double().unsqueeze(1)
    # half a step as above; before it 2^-18 of the value for act and its derivative, and three products that are rounded to whole 2^-149
    bound = torch.maximum(ref.abs() * 2.0 ** -4, step * 2.0 ** -10) * (1 + 2.0 ** -20) + ref.abs() * 2.0 ** -18 + 16 * 2.0 ** -149
    assert ((q.double() * step - ref).abs() <= bound).all()


@pytest.mark.parametrize("t", [I8, E4M3])
def test_weight_columns(t):
    """Input channels that only rows of a tiny scale use."""
    from q8_kernels_b200 import native
    g = torch.Generator(device="cuda").manual_seed(2)
    w, ws = native.tokenwise_quant(torch.randn(96, 144, generator=g, device="cuda").to(BF16), t)
    w = w.float()
    w[:, :len(TINY) + 1] = 0
    for i, v in enumerate(TINY):
        w[i, i], w[i, i + 8] = 64.0, 0.0
        ws[i] = v / 64
    w = w.to(t)
    q, s = native.gated_weight_operand(w, ws)
    ref = (w.double() * ws.double().unsqueeze(1)).T
    assert torch.isfinite(q.float()).all() and torch.isfinite(s).all() and s[len(TINY)] == 0 and (s[:len(TINY)] > 0).all()
    # the scale itself may be subnormal: w * scale is rounded to whole 2^-149
    bound = torch.maximum(ref.abs() * 2.0 ** -4, s.double().unsqueeze(1) * 2.0 ** -10) * (1 + 2.0 ** -20) + ref.abs() * 2.0 ** -20 + 2.0 ** -149
    assert ((q.double() * s.double().unsqueeze(1) - ref).abs() <= bound).all()


@pytest.mark.parametrize("rotate", [False, True])
@pytest.mark.parametrize("src", [BF16, E4M3])
@pytest.mark.parametrize("t", [I8, E4M3])
@pytest.mark.parametrize("k", [16, 32, 64, 128, 256, 272, 512, 1024, 2048, 3088, 4096, 5504, 8192, 16384])
def test_rows_of_zeros(rotate, src, t, k):
    from q8_kernels_b200 import native
    x = torch.randn(40, k, generator=torch.Generator(device="cuda").manual_seed(k), device="cuda").to(BF16).to(src)
    x[::3], x[4] = 0.0, -0.0
    rows = list(range(0, 40, 3)) + [4]
    linears = native.hadamard_quant(x, k ** -0.5, t) if rotate else native.tokenwise_quant(x, t)
    for q, s in (native.gated_quant(x, rotate, t), linears):
        assert (q[rows].float() == 0).all() and (s[rows] == 0).all() and (s[1] > 0) and (q[1].float() != 0).any()
