"""Gated projections of rows with NaN or infinity: such a row's output and gradient are NaN throughout, whatever the type, the rotation and the
number of rows (up to eight are quantised in the product's kernel), and the other rows keep their bits."""
import pytest
import torch

from helpers import bits

pytestmark = pytest.mark.gpu
BF16, E4M3, I8 = torch.bfloat16, torch.float8_e4m3fn, torch.int8
NAN, INF = float("nan"), float("inf")


def spoilt(x):
    """x with a NaN in row 1, only NaN in row 2, an infinity in row 3 and two of opposite signs in row 4."""
    x = x.clone()
    x[1, 7], x[2], x[3, 0], x[4, 1], x[4, 2] = NAN, NAN, INF, INF, -INF
    return x


@pytest.mark.parametrize("m", [5, 8, 9, 40])
@pytest.mark.parametrize("k,f", [(16, 16), (128, 48), (512, 96), (2048, 64), (4096, 32), (8192, 16), (16384, 16)])
@pytest.mark.parametrize("kind", ["int8", "fp8", "fp8_rotated"])
def test_rows_that_are_not_finite(m, k, f, kind):
    from q8_kernels_b200 import check_status, native
    from q8_kernels_b200.functional import gated
    g = torch.Generator(device="cuda").manual_seed(m + k)
    t = I8 if kind == "int8" else E4M3
    w, ws = native.tokenwise_quant(torch.randn(2 * f, k, generator=g, device="cuda").to(BF16), t)
    bias = torch.randn(2 * f, generator=g, device="cuda")
    x = torch.randn(m, k, generator=g, device="cuda").to(BF16)
    grad = torch.randn(m, f, generator=g, device="cuda").to(BF16)

    def step(a):
        a = a.clone().requires_grad_(True)
        y = gated.q8_gated_linear(a, w, bias, None, ws) if t == I8 else gated.fp8_gated_linear(a, w, bias, None, ws, "silu", kind != "fp8")
        return y.detach(), torch.autograd.grad(y, [a], grad)[0]

    rest = [0] + list(range(5, m))
    for clean, got in zip(step(x), step(spoilt(x))):
        assert got[1:5].isnan().all()
        assert torch.isfinite(got[rest]).all() and torch.equal(bits(got[rest]), bits(clean[rest]))
    check_status()


@pytest.mark.parametrize("rotate", [False, True])
@pytest.mark.parametrize("src", [BF16, E4M3])
@pytest.mark.parametrize("t", [I8, E4M3])
@pytest.mark.parametrize("k", [16, 48, 128, 256, 272, 512, 1024, 1536, 2048, 4096, 8192, 16384])
def test_scales_of_rows_with_nan(rotate, src, t, k):
    """The row's scale is NaN; the quantizers of the linears leave NaN out of the maximum, as before."""
    from q8_kernels_b200 import native
    x = torch.randn(33, k, generator=torch.Generator(device="cuda").manual_seed(k), device="cuda").to(BF16).to(src)
    bad = x.clone()
    bad[1, 3], bad[4], bad[32, k - 1] = NAN, NAN, NAN
    q, s = native.gated_quant(x, rotate, t)
    qb, sb = native.gated_quant(bad, rotate, t)
    rest = [i for i in range(33) if i not in (1, 4, 32)]
    assert sb[[1, 4, 32]].isnan().all() and torch.equal(sb[rest], s[rest]) and torch.equal(bits(qb)[rest], bits(q)[rest])
    if rotate:
        q, s = native.hadamard_quant(bad, k ** -0.5, t)
        assert (s[[1, 4, 32]] == 0).all()
    else:
        q, s = native.tokenwise_quant(bad, t)
        left = native.tokenwise_quant(torch.where(bad.float().isnan(), 0.0, bad.float()).to(src), t)
        assert torch.equal(s, left[1])
        if t == E4M3:
            assert q.float()[1, 3].isnan() and q.float()[32, k - 1].isnan()


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("f", [16, 528, 1024, 4096, 16384])
def test_gradients_with_nan(f, act):
    """A NaN anywhere in a gradient's row, or only NaN: the row of the product has it."""
    from q8_kernels_b200 import native
    g = torch.Generator(device="cuda").manual_seed(f)
    pre = torch.randn(6, 2, f, generator=g, device="cuda").to(BF16)
    grad = torch.randn(6, f, generator=g, device="cuda").to(BF16)
    clean = native.gated_backward_quant(grad, pre, act)
    grad[1, f // 2], grad[2] = NAN, NAN
    pre[4, 1, f - 1] = NAN
    q, s = native.gated_backward_quant(grad, pre, act)
    real = q.float() * s.unsqueeze(1)
    assert real[[1, 2, 4]].isnan().any(1).all() and real[2].isnan().all()
    rest = [0, 3, 5]
    assert torch.equal(bits(q)[rest], bits(clean[0])[rest]) and torch.equal(s[rest], clean[1][rest])
