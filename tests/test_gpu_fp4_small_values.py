"""Gradients of 4-bit linears at the lower end of fp32's range: columns of the weight and rows of the output's gradient whose factor
448 / absmax fp32 does not hold (absmax below 1.3e-36) have FLT_MAX in its place, and their zeros stay zeros.

Tolerances.  The operands are defined operation by operation in fp32: none.  Products as in test_gpu_fp4.py; the product of the two scales may
be subnormal, and is then off by up to half of fp32's smallest step, 2^-150, times the sum of the operands' sizes.
"""
import pytest
import torch

from helpers import bits
from test_gpu_fp4 import FORMATS, sample, wide

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
E4M3 = torch.float8_e4m3fn
MAX = torch.finfo(F32).max


def rows_e4m3(x):
    """Rows of fp32 values as e4m3 and what each step stands for, by the definition."""
    x = x.cpu()
    amax = x.abs().amax(1, keepdim=True)
    f = torch.full_like(amax, 448.0) / amax
    f = torch.where(amax > 0, f.clamp(max=MAX), f)
    return (x * torch.where(amax > 0, f, torch.zeros_like(f))).to(E4M3), torch.ones_like(f) / f


def weights(fmt):
    """Some output channels by 96 input channels; a block's worth of input channels is near the smallest values, with zeros among them."""
    small = torch.randn(48, 96, generator=torch.Generator().manual_seed(1))
    if fmt == "nvfp4":                                          # (a row's values are within 2^-20 of its largest one)
        w = (small * 1e-37).to(BF16)
        w[:, 3:9] = 0
        w[::3, 11] = 0
    else:
        w = sample(48, 96, BF16, 7)
        w[:, 32:64] = (small[:, 32:64] * 1e-38).to(BF16)
        w[::2, 32:40] = 0
        w[:, 45] = 0
        w[:, 50] = 0
        w[7, 50] = 9.2e-41
    return w


@pytest.mark.parametrize("fmt", FORMATS)
def test_weight_operand(fmt):
    from q8_kernels_b200 import native
    q = native.fp4_quant(weights(fmt).cuda(), fmt)
    got, scales = native.fp4_weight_operand(q[0], q[1:])
    full = wide(*q[:2], None, fmt).float()
    full = full if q[2] is None else full * q[2].unsqueeze(1)
    ref, rs = rows_e4m3(full.T.contiguous())
    amax = full.abs().amax(0).cpu()
    assert ((amax > 0) & (amax < 448.0 / MAX)).any() and (full.cpu()[:, (amax > 0) & (amax < 448.0 / MAX)] == 0).any()
    assert torch.equal(got.cpu().float(), ref.float()) and torch.equal(bits(scales.cpu()), bits(rs[:, 0]))


def gradient(y, x, g, w, ws, k):
    """dx against the e4m3 operands' product in 64 bits."""
    from q8_kernels_b200 import check_status, native
    dx, = torch.autograd.grad(y, [x], g)
    check_status()
    n = w.shape[0]
    g8, gs = (t.cuda() for t in rows_e4m3(g.reshape(-1, n).float()))
    w8, wsc = native.fp4_weight_operand(w, ws)
    a, b = g8.double() * gs.double(), w8.double() * wsc.double().unsqueeze(1)
    a, b = torch.where(g8.double() == 0, 0.0, a), torch.where(w8.double() == 0, 0.0, b)
    f = torch.finfo(BF16)
    ref = a @ b.T
    slack = (n // 32 + 12) * 2.0 ** -23 * (a.abs() @ b.abs().T) + 2.0 ** -150 * (g8.double().abs() @ w8.double().abs().T)
    good = (dx.reshape(-1, k).double() - ref).abs() <= slack + (ref.abs() + slack) * f.eps / 2 * 1.001 + f.tiny * f.eps
    assert good.all(), f"{int((~good).sum())} of {good.numel()}, {int(torch.isnan(dx).sum())} NaN"


@pytest.mark.parametrize("fmt", FORMATS)
def test_gradient_through_a_weight_of_small_values(fmt):
    from q8_kernels_b200.functional.fp4 import fp4_linear, fp4_quantize
    w, ws = fp4_quantize(weights(fmt).cuda(), fmt)
    x = torch.randn(5, 96, device="cuda").to(BF16).requires_grad_(True)
    y = fp4_linear(x, w, None, None, ws)
    assert torch.isfinite(y).all()
    gradient(y, x, torch.randn(5, 48, device="cuda").to(BF16), w, ws, 96)


@pytest.mark.parametrize("native_host", [True, False])
@pytest.mark.parametrize("gelu", [False, True])
@pytest.mark.parametrize("fmt", FORMATS)
def test_gradient_rows_of_small_values(monkeypatch, fmt, gelu, native_host):
    """Rows of an ordinary size, of 1e-30, 1e-37 and the smallest bf16, each with zeros, and a row of zeros; a training step of 16-bit gradients has
    such rows where a loss hardly depends on a token."""
    from q8_kernels_b200 import _host, native
    from q8_kernels_b200.functional.fp4 import fp4_linear, fp4_quantize
    if not native_host:
        monkeypatch.setattr(_host, "_fp4_linear", lambda *a: None)
    w, ws = fp4_quantize(sample(272, 512, BF16, 5).cuda(), fmt)
    x = torch.randn(2, 6, 512, device="cuda").to(BF16).requires_grad_(True)
    g = torch.randn(2, 6, 272, device="cuda")
    g *= torch.tensor([1.0, 1e-30, 1e-36, 1e-37, 1e-38, 0.0], device="cuda").view(1, 6, 1)
    g[:, :, ::3] = 0
    g[1, 5, 4] = 9.2e-41
    g = g.to(BF16)
    y = fp4_linear(x, w, None, None, ws, gelu)
    if gelu:
        dx, = torch.autograd.grad(y, [x], g)
        assert torch.isfinite(dx).all() and not dx[0, 5].any()
        pre = fp4_linear(x.detach(), w, None, None, ws, out_dtype=BF16)
        x2 = x.detach().requires_grad_(True)
        inner = native.gelu_backward(pre, g, BF16)
        ref, = torch.autograd.grad(fp4_linear(x2, w, None, None, ws), [x2], inner)
        assert torch.equal(bits(dx), bits(ref))
    else:
        gradient(y, x, g, w, ws, 512)


def test_gradient_operand():
    """Bit by bit, and that of tokenwise_quant where rows are of an ordinary size; its refusals."""
    from q8_kernels_b200 import Q8KernelError, native
    for t in (BF16, torch.float16):
        for n in (16, 48, 272, 1040, 4112, 20000, 32768):
            g = sample(7, n, t, 2).clamp(-1e4, 1e4)
            g[1] = 0
            if t == BF16:
                g[2] = (g[2].float().clamp(-8, 8) * 1e-38).to(t)
                g[3] = 0
                g[3, n // 2] = -9.2e-41
                g[2, ::5] = 0
            q, s = native.fp4_backward_quant(g.cuda())
            ref, rs = rows_e4m3(g.float())
            assert torch.equal(q.cpu().float(), ref.float()) and torch.equal(bits(s.cpu()), bits(rs[:, 0])), (t, n)
            plain = g[[0, 1, 4, 5, 6]].cuda()
            for a, b in zip(native.fp4_backward_quant(plain), native.tokenwise_quant(plain, E4M3)):
                assert torch.equal(bits(a), bits(b))
    q, s = native.fp4_backward_quant(torch.tensor([[float("nan")] + [1.0] * 15, [float("inf")] + [1.0] * 15], device="cuda").to(BF16))
    assert torch.isnan(q[0, 0].float()) and torch.isnan(q[1, 0].float()) and torch.isinf(s[1])
    assert native.fp4_backward_quant(torch.zeros(0, 32, device="cuda", dtype=BF16))[0].shape == (0, 32)
    x = torch.zeros(2, 32, device="cuda", dtype=BF16)
    for bad in (x.float(), x.cpu(), x[:, :24], torch.zeros(1, 32784, device="cuda", dtype=BF16)):
        with pytest.raises(Q8KernelError):
            native.fp4_backward_quant(bad)
