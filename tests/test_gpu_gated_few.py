"""One call of the gated projection with few rows, which rotates and quantises them in the product's kernel: the bits of the two separate
steps, for every number of rows around the limit, columns that are no power of two, short and long K."""
import pytest
import torch

from helpers import bits

pytestmark = pytest.mark.gpu
BF16, E4M3, I8 = torch.bfloat16, torch.float8_e4m3fn, torch.int8


@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 7, 8, 9])
@pytest.mark.parametrize("k,f", [(16, 16), (48, 32), (64, 48), (128, 272), (144, 16), (256, 1040), (272, 96), (512, 688), (1024, 112), (1040, 64), (2048, 1408),
                                 (3088, 160), (4096, 528), (8192, 144), (8208, 48)])
@pytest.mark.parametrize("kind", ["int8", "fp8", "fp8_rotated"])
def test_bits_of_the_two_steps(m, k, f, kind):
    from q8_kernels_b200 import check_status, native
    from q8_kernels_b200.functional import gated
    g = torch.Generator(device="cuda").manual_seed(m * k + f)
    x = torch.randn(m, k, generator=g, device="cuda").to(BF16)
    x[:, k // 3] *= 20
    if m > 2:
        x[1] = 0
    t = I8 if kind == "int8" else E4M3
    rotate = kind != "fp8"
    w, ws = native.gated_quant(torch.randn(2 * f, k, generator=g, device="cuda").to(BF16), False, t)
    bias = torch.randn(2 * f, generator=g, device="cuda")
    q, qs = native.gated_quant(x, rotate, t)
    want = native.gated_mm(q, w, bias, qs, ws, "silu", True)

    def call(a):
        return gated.q8_gated_linear(a, w, bias, None, ws) if t == I8 else gated.fp8_gated_linear(a, w, bias, None, ws, "silu", rotate)

    assert torch.equal(bits(call(x)), bits(want[0]))
    leaf = x.clone().requires_grad_(True)
    y = call(leaf)
    assert torch.equal(bits(y), bits(want[0]))
    # what the backward pass finds is what the two steps leave
    grad = torch.randn(m, f, generator=g, device="cuda").to(BF16)
    g8, gs = native.gated_backward_quant(grad, want[1], "silu")
    w8, wsc = native.gated_weight_operand(w, ws)
    dx = native.fp8_mm(g8, w8, gs, wsc, False, BF16)[0]
    if rotate:
        dx = native.fast_hadamard_transform(dx, k ** -0.5)
    assert torch.equal(bits(torch.autograd.grad(y, [leaf], grad)[0]), bits(dx))
    check_status()


def test_not_finite_rows_stay_alone():
    from q8_kernels_b200 import native
    from q8_kernels_b200.functional import gated
    x = torch.randn(5, 512, device="cuda").to(BF16)
    w, ws = native.gated_quant(torch.randn(96, 512, device="cuda").to(BF16), False, E4M3)
    clean = gated.fp8_gated_linear(x, w, None, None, ws)
    x[1, 7], x[3] = float("nan"), float("inf")
    y = gated.fp8_gated_linear(x, w, None, None, ws)
    assert y[1].isnan().all() and not y[3].isfinite().any()
    assert torch.equal(bits(y[[0, 2, 4]]), bits(clean[[0, 2, 4]]))
