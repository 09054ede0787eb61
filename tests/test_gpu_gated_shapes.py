"""The gated feed-forward module keeps the leading dims of its input, so that it can stand in a residual sum: rows without a batch, one row, no
rows, more dims; forward and backward."""
import pytest
import torch

from helpers import bits

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def filled(ff, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    for m in (ff.gate_up, ff.proj_down):
        n, k = m.weight.shape
        w = 0.1 * torch.randn(n, k, generator=g, device="cuda")
        m.weight.data = (w * 500).clamp(-127, 127).to(m.weight.dtype)
        m.scales.data = torch.full((n,), 0.01, device="cuda")
        m.bias.data = torch.randn(n, generator=g, device="cuda")
    return ff


@pytest.mark.parametrize("linear", ["int8", "fp8"])
@pytest.mark.parametrize("lead", [(), (6,), (1, 6), (2, 3), (2, 1, 3), (0,), (2, 0)])
def test_feed_forward_keeps_the_shape(linear, lead):
    from q8_kernels_b200.modules import GatedFeedForward, LayerNorm
    ff, norm = filled(GatedFeedForward(512, 256, linear=linear).cuda()), LayerNorm(512).cuda()
    x = torch.randn(*lead, 512, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").to(BF16)
    flat = x.reshape(1, -1, 512)
    y = ff(norm(x))
    assert y.shape == x.shape and y.dtype == BF16
    if x.numel():
        assert torch.equal(bits(y), bits(ff(norm(flat)).view(x.shape)))
    leaf = x.clone().requires_grad_(True)
    z = leaf + ff(norm(leaf))
    assert z.shape == x.shape
    g = torch.randn(x.shape, device="cuda").to(BF16)
    dx, = torch.autograd.grad(z, [leaf], g)
    assert dx.shape == x.shape
    if x.numel():
        leaf = flat.clone().requires_grad_(True)
        assert torch.equal(bits(dx), bits(torch.autograd.grad(leaf + ff(norm(leaf)), [leaf], g.view(flat.shape))[0].view(x.shape)))


@pytest.mark.parametrize("linear", ["int8", "fp8"])
def test_output_types_without_rows(linear):
    from q8_kernels_b200.modules import GatedFeedForward
    ff = filled(GatedFeedForward(512, 256, linear=linear).cuda())
    x = torch.randn(4, 512, device="cuda").to(BF16)
    for kwargs in ({}, {"out_dtype": BF16}, {"out_dtype": None}):
        y, none = ff(x, **kwargs), ff(x[:0], **kwargs)
        assert y.shape == (4, 512) and none.shape == (0, 512) and none.dtype == y.dtype
