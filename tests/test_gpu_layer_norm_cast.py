"""The LayerNorm module in a model that is cast to 16 bits."""
import pytest
import torch

from helpers import bits

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_layer_norm_of_a_cast_model(dtype):
    """Weight and bias rounded with the model; the rest of the arithmetic is that of fp32 parameters with these values."""
    from q8_kernels_b200.functional.layer_norm import layer_norm
    from q8_kernels_b200.modules import LayerNorm
    g = torch.Generator(device="cuda").manual_seed(4)
    m = LayerNorm(96).cuda()
    m.weight.data, m.bias.data = 1 + 0.1 * torch.randn(96, generator=g, device="cuda"), torch.randn(96, generator=g, device="cuda")
    m = m.to(dtype)
    x = torch.randn(7, 96, generator=g, device="cuda").to(dtype).requires_grad_(True)
    grad = torch.randn(7, 96, generator=g, device="cuda").to(dtype)
    y = m(x)
    wide = [t.detach().float().requires_grad_(True) for t in (m.weight, m.bias)]
    z = layer_norm(x, *wide)
    assert torch.equal(bits(y), bits(z))
    got = torch.autograd.grad(y, [x, m.weight, m.bias], grad)
    want = torch.autograd.grad(z, [x, *wide], grad)
    assert torch.equal(bits(got[0]), bits(want[0]))
    for a, b in zip(got[1:], want[1:]):
        assert a.dtype == dtype and torch.equal(bits(a), bits(b.to(dtype)))
    for kwargs in ({"bias": False}, {"elementwise_affine": False}):
        assert torch.isfinite(LayerNorm(96, **kwargs).cuda().to(dtype)(x)).all()
