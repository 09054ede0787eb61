"""The gradient's quantizer of gated projections with more rows than its grid and its rings hold: every CTA walks over several, with slots and the
arrays of partial maxima used again."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
U = 2.0 ** -24


def act64(g, act):
    return g * torch.sigmoid(g) if act == "silu" else torch.nn.functional.gelu(g, approximate="tanh")


# 148 SMs with 16, 8, 4, 3, 2 and 1 CTAs and rings of 4, 4, 4, 3, 2 and 2 rows: five to seven turns at the full width of each layout and at one in it
@pytest.mark.parametrize("m,f", [(12001, 512), (12001, 400), (6007, 1024), (6007, 912), (3001, 2048), (3001, 1040), (2221, 4096), (2221, 2064), (1483, 8192),
                                 (1483, 5504), (741, 16384), (741, 8208)])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_many_rows(m, f, act):
    from q8_kernels_b200 import native
    g = torch.Generator(device="cuda").manual_seed(m + f)
    pre = (3 * torch.randn(m, 2, f, generator=g, device="cuda")).to(BF16)
    grad = torch.randn(m, f, generator=g, device="cuda")
    # neighbouring rows, and those of one CTA, far apart in size: a row's maximum or elements in another's place show
    size = torch.exp2(torch.randint(-60, 60, (m, 1), generator=g, device="cuda").float())
    grad = (grad * size).to(BF16)
    q, s = native.gated_backward_quant(grad, pre, act)
    for lo in range(0, m, 500):                                 # in parts, for the 64-bit copies
        part = slice(lo, min(lo + 500, m))
        gate, up = pre[part, 0].double().requires_grad_(True), pre[part, 1].double().requires_grad_(True)
        gr = grad[part].double()
        d = torch.cat(torch.autograd.grad(act64(gate, act) * up, [gate, up], gr), 1)
        # act and act' are off by 2^-24 times a few units and the exponent's size, |v| up to 2 * 0.8 * (16 + 0.045 * 16^3) = 320 in GELU, of
        # the terms that are added; where |v| is above 20 the sigmoid is 1 or below 2^-28, so 64 units cover it
        err = 64 * U * torch.cat([gr.abs() * up.detach().abs(), gr.abs() * gate.detach().abs()], 1) * 2
        top = d.abs().amax(1, keepdim=True)
        step = s[part].double().unsqueeze(1)
        assert ((step * 448 - top).abs() <= top * 4 * U + err.amax(1, keepdim=True)).all()
        bound = d.abs() * 2.0 ** -4 + (top / 448) * 2.0 ** -10
        assert ((q[part].double() * step - d).abs() <= bound * 1.001 + 2 * err).all()
