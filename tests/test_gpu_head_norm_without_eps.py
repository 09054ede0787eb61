"""Head norms with eps = 0: the places of a CTA that no token or head fills stay out of the weights' gradients.

Tolerances as in test_gpu_head_norm.py, whose formulas in 64 bits these use; for the weights' gradients: a thread adds up at most 16 heads of each of
two tokens, a CTA 32 of its groups, the last kernel 47 rows a thread and 18 of its warps, with 26 u for a term: below 256 u of the sum of sizes.
"""
import pytest
import torch

import test_gpu_head_norm as norm

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def near(y, ref, slack):
    """As norm.near, with a condition that NaN does not meet."""
    f = torch.finfo(y.dtype)
    good = (y.double() - ref).abs() <= ref.abs() * (f.eps / 2) * 1.001 + f.tiny * f.eps + slack * 1.01
    assert good.all(), f"{int((~good).sum())} of {good.numel()}, {int(torch.isnan(y).sum())} NaN"


# tokens and heads that fill the last CTA, or leave a part of it, in the forms for heads of 64, 128 and 256 channels and in the general one
@pytest.mark.parametrize("t", [BF16, F16, F32])
@pytest.mark.parametrize("kind,layout", [("none", "half"), ("one", "half"), ("axes", "interleaved")])
@pytest.mark.parametrize("b,s,hq,hk,d,r", [(3, 1001, 20, 4, 80, 32), (1, 1, 1, 1, 64, 64), (1, 1023, 8, 2, 64, 64), (2, 67, 12, 5, 128, 96), (1, 333, 7, 3, 72, 72),
                                           (1, 2047, 9, 1, 256, 256), (1, 6143, 40, 8, 128, 128), (2, 5, 3, 1, 65, 10)])
def test_gradients(monkeypatch, t, kind, layout, b, s, hq, hk, d, r):
    from q8_kernels_b200.functional.head_norm import head_norm
    monkeypatch.setattr(norm, "near", near)
    g = torch.Generator(device="cuda").manual_seed(d + s)
    q, k = (torch.randn(b, s, h, d, generator=g, device="cuda").to(t).requires_grad_(True) for h in (hq, hk))
    wq, wk = ((1 + 0.3 * torch.randn(d, generator=g, device="cuda")).requires_grad_(True) for _ in range(2))
    angle = norm.angles(kind, r, b, s, layout)
    y, z = head_norm(q, k, wq, wk, 0.0, *angle[:4], layout)
    norm.check(y.detach(), q.detach(), wq, 0.0, angle)
    norm.check(z.detach(), k.detach(), wk, 0.0, angle)
    gy, gz = torch.randn(y.shape, generator=g, device="cuda").to(t), torch.randn(z.shape, generator=g, device="cuda").to(t)
    dq, dk, dwq, dwk = torch.autograd.grad([y, z], [q, k, wq, wk], [gy, gz])
    norm.check_grads(dq, dwq, q, wq, gy, 0.0, angle)
    norm.check_grads(dk, dwk, k, wk, gz, 0.0, angle)


def test_a_head_of_zeros_spoils_the_weights_gradient_and_no_other_head():
    """0 / 0 is no number: its own elements' and the sums that it is a part of."""
    from q8_kernels_b200.functional.head_norm import head_norm
    q, k = torch.randn(1, 9, 3, 64, device="cuda"), torch.randn(1, 9, 2, 64, device="cuda")
    q[0, 4, 1] = 0
    leaves = [t.requires_grad_(True) for t in (q, k, torch.ones(64, device="cuda"), torch.ones(64, device="cuda"))]
    y, z = head_norm(*leaves, 0.0)
    dq, dk, dwq, dwk = torch.autograd.grad([y, z], leaves, [torch.ones_like(y), torch.ones_like(z)])
    for t in (y, dq):
        assert torch.isnan(t).any(-1)[0].nonzero().tolist() == [[4, 1]] and torch.isnan(t[0, 4, 1]).all()
    assert torch.isnan(dwq).all() and torch.isfinite(dwk).all() and torch.isfinite(dk).all() and torch.isfinite(z).all()
