"""The sweeps over sizes, layouts and types of 4-bit linears, head norms and rotations by several axes again, with conditions that an output of NaN does
not meet: |y - ref| <= bound has to hold.  Sizes, references and bounds are those of the tests that these stand beside.
"""
import pytest
import torch

import test_gpu_axial_rotary as axial
import test_gpu_fp4 as fp4
import test_gpu_head_norm as norm
from helpers import bits
from test_gpu_head_norm_without_eps import near

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def params(test):
    """The parametrisation of another test."""
    def again(f):
        for mark in test.pytestmark:
            if mark.name == "parametrize":
                f = pytest.mark.parametrize(*mark.args, **mark.kwargs)(f)
        return f
    return again


def within(y, ref, bound):
    good = (y.double() - ref).abs() <= bound
    # beyond the type: an infinity of the right sign
    good |= torch.isinf(y) & (ref.abs() >= torch.finfo(y.dtype).max) & (torch.signbit(y) == torch.signbit(ref))
    assert good.all(), f"{int((~good).sum())} of {good.numel()}, {int(torch.isnan(y).sum())} NaN"


@params(fp4.test_products)
def test_products(fmt, gelu, bias, out, m, n, k):
    from q8_kernels_b200 import check_status, native
    a, b = fp4.sample(m, k, BF16, 1).cuda(), fp4.sample(n, k, BF16, 2).cuda()
    qa, qb = native.fp4_quant(a, fmt), native.fp4_quant(b, fmt)
    c = torch.randn(n, device="cuda") if bias else None
    y = native.fp4_mm(qa[0], qb[0], c, qa[1:], qb[1:], gelu, out)
    check_status()
    wa, wb = fp4.wide(*qa, fmt), fp4.wide(*qb, fmt)
    ref, slack = wa @ wb.T, (k // 64 + 8) * 2.0 ** -23 * (wa.abs() @ wb.abs().T)
    if bias:
        ref, slack = ref + c.double(), slack + 2.0 ** -22 * c.double().abs()
    if gelu:
        slack = 1.13 * slack + 2.0 ** -11.9 * ref.abs() + 2.0 ** -22 * ref.abs()    # |gelu'| < 1.13
        ref = torch.nn.functional.gelu(ref, approximate="tanh")
    f = torch.finfo(out)
    within(y, ref.clamp(-2 * f.max, 2 * f.max), slack + (ref.abs() + slack) * f.eps / 2 * 1.001 + f.tiny * f.eps)


@params(fp4.test_linear_and_gradient)
def test_linear_and_gradient(fmt, t, shape, n):
    from q8_kernels_b200 import check_status, native
    from q8_kernels_b200.functional.fp4 import fp4_dequantize, fp4_linear, fp4_quantize
    k = shape[-1]
    x = fp4.sample(torch.Size(shape[:-1]).numel(), k, t, 4).cuda().clamp(-1e3, 1e3).view(shape).requires_grad_(True)
    w, ws = fp4_quantize((fp4.sample(n, k, BF16, 5) * 0.02).to(t).cuda(), fmt)
    bias = torch.randn(n, device="cuda")
    y = fp4_linear(x, w, bias, None, ws)
    g = torch.randn(y.shape, device="cuda").to(t)
    dx, = torch.autograd.grad(y, [x], g)
    check_status()
    f = torch.finfo(t)
    qx, qs = fp4_quantize(x, fmt)
    wx, ww = fp4_dequantize(qx, qs, F32).double().view(-1, k), fp4_dequantize(w, ws, F32).double()
    # (values are rounded to fp32 by the row's scale: 2^-24 of each on both sides)
    ref, slack = wx @ ww.T + bias.double(), (k // 64 + 10) * 2.0 ** -23 * (wx.abs() @ ww.abs().T) + 2.0 ** -22 * bias.double().abs()
    within(y.detach().reshape(-1, n), ref, slack + (ref.abs() + slack) * f.eps / 2 * 1.001 + f.tiny * f.eps)
    g8, gs = fp4.rows_e4m3(g.reshape(-1, n).float())
    w8, wsc = native.fp4_weight_operand(w, ws)
    a, b = g8.double() * gs.double(), w8.double() * wsc.double().unsqueeze(1)
    ref, slack = a @ b.T, (n // 32 + 12) * 2.0 ** -23 * (a.abs() @ b.abs().T)
    within(dx.reshape(-1, k), ref, slack + (ref.abs() + slack) * f.eps / 2 * 1.001 + f.tiny * f.eps)


@params(norm.test_layouts_types_and_sizes)
def test_head_norm(monkeypatch, kind, layout, t, d, r):
    monkeypatch.setattr(norm, "near", near)
    norm.test_layouts_types_and_sizes(kind, layout, t, d, r)


@params(norm.test_strides_shapes_and_parts)
def test_head_norm_strides(monkeypatch, layout, d):
    monkeypatch.setattr(norm, "near", near)
    norm.test_strides_shapes_and_parts(layout, d)


def test_head_norm_long_offsets_parts_and_values(monkeypatch):
    monkeypatch.setattr(norm, "near", near)
    norm.test_long_offsets_and_many_tokens()
    norm.test_parts_of_the_gradient()
    norm.test_values_that_are_not_finite()


def numbers(y, x, positions, freq, axes, amplitude, layout, sign=1.0):
    """As axial.check."""
    ref, size = axial.turned(x, positions, freq, axes, amplitude, layout, sign)
    f = torch.finfo(x.dtype)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    good = (y.double() - ref).abs() <= ref.abs() * (f.eps / 2) * 1.001 + f.tiny * f.eps + 8 * axial.U * size
    assert good.all(), f"{int((~good).sum())} of {good.numel()}, {int(torch.isnan(y).sum())} NaN"
    assert torch.equal(bits(y[..., 2 * freq.numel():]), bits(x[..., 2 * freq.numel():]))


@params(axial.test_layouts_types_and_sizes)
def test_axial_rotary(monkeypatch, layout, t, d, sections):
    monkeypatch.setattr(axial, "check", numbers)
    axial.test_layouts_types_and_sizes(layout, t, d, sections)


@params(axial.test_strides_empty_and_long_offsets)
def test_axial_rotary_strides(monkeypatch, layout):
    monkeypatch.setattr(axial, "check", numbers)
    axial.test_strides_empty_and_long_offsets(layout)


@params(axial.test_gradients)
def test_axial_rotary_gradients(monkeypatch, layout, t, d):
    monkeypatch.setattr(axial, "check", numbers)
    axial.test_gradients(layout, t, d)


def test_axial_rotary_positions(monkeypatch):
    monkeypatch.setattr(axial, "check", numbers)
    axial.test_positions_and_axes()


def test_casts_of_a_linear_with_a_bias():
    """A cast of the model rounds the bias and leaves weight and scales alone: the output is that of the rounded bias, widened."""
    from q8_kernels_b200.functional.fp4 import fp4_linear
    from q8_kernels_b200.modules import FP4Linear
    for fmt in fp4.FORMATS:
        full = torch.nn.Linear(512, 208, device="cuda", dtype=BF16)
        full.bias.data.mul_(1.0 + 2.0 ** -9)
        x = torch.randn(3, 50, 512, device="cuda").to(BF16)
        m = FP4Linear.from_linear(full, fmt)
        m.bias.data.add_(2.0 ** -14)                           # not a number of 16 bits
        bias, weight, scales = m.bias.data.clone(), m.weight.data.clone(), m.weight_scales
        for types in ((F16,), (BF16,), (F16, BF16), (torch.float64, F32)):
            cast = FP4Linear.from_linear(full, fmt)
            cast.bias.data.copy_(bias)
            expected = bias
            for t in types:
                cast, expected = cast.to(t), expected.to(t)
            assert cast.bias.dtype == types[-1] and torch.equal(cast.weight, weight)
            assert torch.equal(bits(cast(x)), bits(fp4_linear(x, weight, expected.float(), None, scales)))
        assert not torch.equal(bias.to(BF16).float(), bias)
