"""The native path of the differentiable ops (layer norm, rotary positions, gated projection) against their Python bodies: the same bits and
gradients, what is left to Python, gradients of gradients."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _plain_calls():
    """(native call, call that takes the Python body: a tensor of another kind with the same values) of the differentiable ops."""
    from q8_kernels_b200 import native
    from q8_kernels_b200.functional import gated, layer_norm, rotary
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(6, 40, 512, generator=g, device="cuda").to(BF16)
    w, b = 1 + 0.1 * torch.randn(512, generator=g, device="cuda"), 0.1 * torch.randn(512, generator=g, device="cuda")
    w8, ws = native.tokenwise_quant(torch.randn(288, 512, generator=g, device="cuda").to(BF16))
    f8, fs = native.tokenwise_quant(torch.randn(288, 512, generator=g, device="cuda").to(BF16), torch.float8_e4m3fn)
    freq = rotary.rotary_frequencies(32)[0].cuda()
    pos = torch.arange(40, device="cuda")
    return [(lambda t: layer_norm.layer_norm(t, w, b), x), (lambda t: layer_norm.layer_norm(t, w), x.float()),
            (lambda t: rotary.apply_rotary(t.view(6, 40, 8, 64), None, pos, freq, 1.5, "interleaved")[0], x),
            (lambda t: torch.cat(rotary.apply_rotary(t.view(6, 40, 8, 64)[:, :, :6], t.view(6, 40, 8, 64)[:, :, 6:], pos, freq), 2), x.half()),
            (lambda t: gated.q8_gated_linear(t, w8, None, None, ws, "gelu_tanh"), x),
            (lambda t: gated.fp8_gated_linear(t, f8, None, None, fs, "silu", True), x)]


@pytest.mark.parametrize("i", range(6))
def test_differentiable_ops_native_and_python_body(i):
    from q8_kernels_b200 import _host
    call, x = _plain_calls()[i]
    seen = []

    def run(native):
        leaf = x.clone().requires_grad_(True)
        names = ("_layer_norm", "_rotary", "_gated_linear")
        kept = {n: getattr(_host, n) for n in names}
        for n in names:
            def watch(*a, fn=kept[n]):
                out = fn(*a) if native else None
                seen.append(out is not None)
                return out
            setattr(_host, n, watch)
        try:
            y = call(leaf)
            with torch.no_grad():
                plain = call(leaf)
        finally:
            for n in names:
                setattr(_host, n, kept[n])
        grad = torch.randn(y.shape, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(y.dtype)
        return y.detach(), plain, torch.autograd.grad(y, [leaf], grad)[0]

    a, b = run(True), run(False)
    assert seen == [True, True, False, False]
    for p, q in zip(a, b):
        assert p.dtype == q.dtype and torch.equal(p.view(torch.uint8), q.view(torch.uint8))
    assert torch.equal(a[0].view(torch.uint8), a[1].view(torch.uint8))


@pytest.mark.parametrize("i", range(6))
def test_differentiable_ops_once(i):
    """Gradients of gradients are refused when they are asked for, and not before."""
    call, x = _plain_calls()[i]
    leaf = x.clone().requires_grad_(True)
    y = call(leaf)
    grad = torch.ones_like(y).requires_grad_(True)
    dx, = torch.autograd.grad(y, [leaf], grad, create_graph=True)
    assert torch.isfinite(dx.float()).all()
    with pytest.raises(RuntimeError, match="twice|once"):
        dx.float().sum().backward()


def test_differentiable_ops_leave_others_to_python():
    from q8_kernels_b200 import _host
    from q8_kernels_b200.functional.rotary import rotary_frequencies
    x = torch.zeros(4, 6, 2, 64, device="cuda", dtype=BF16)
    freq = rotary_frequencies(64)[0].cuda()
    assert _host._layer_norm(x, None, None, 1e-5, None) is not None and _host._rotary(x, None, None, freq, 1.0, True) is not None
    assert _host._layer_norm(x[..., ::2], None, None, 1e-5, None) is None and _host._layer_norm(x, None, None, 1e-5, torch.float16) is None
    assert _host._layer_norm(x.cpu(), None, None, 1e-5, None) is None and _host._layer_norm(x, None, None, 1, None) is None
    assert _host._rotary(x[..., ::2], None, None, freq[:16], 1.0, True) is None and _host._rotary(x, x.half(), None, freq, 1.0, True) is None
    assert _host._rotary(x, None, None, freq.float(), 1.0, True) is None
    assert torch.func.vmap(lambda t: torch.tensor(_host._layer_norm(t, None, None, 1e-5, None) is None))(x).all()
    w, s = torch.zeros(64, 64, dtype=torch.int8, device="cuda"), torch.zeros(64, device="cuda")
    a = x.view(-1, 64)
    assert _host._gated_linear(a, w, None, s, 1, True, True) is not None
    assert _host._gated_linear(a, w, None, s, 0, True, True) is None and _host._gated_linear(a, w, None, s, 1, False, True) is None
    assert _host._gated_linear(a, w[:48], None, s[:48], 1, True, True) is None and _host._gated_linear(a, w, s[:3], s, 1, True, True) is None
