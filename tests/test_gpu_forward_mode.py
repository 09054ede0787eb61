"""Forward-mode derivatives, which layer norm, rotary positions and gated projections do not have: an input that carries one is refused, with and
without a gradient of its own, instead of an output that has lost it."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu
BF16, I8, E4M3 = torch.bfloat16, torch.int8, torch.float8_e4m3fn


def calls():
    """(call, the tensors that may carry a tangent)"""
    from q8_kernels_b200 import native
    from q8_kernels_b200.functional import gated, layer_norm, rotary
    x = torch.randn(4, 64, device="cuda").to(BF16)
    w = torch.ones(64, device="cuda")
    q, k = torch.randn(2, 3, 4, 64, device="cuda").to(BF16).unbind(0)
    freq = rotary.rotary_frequencies(64)[0].cuda()
    w8, ws = native.tokenwise_quant(torch.randn(64, 64, device="cuda").to(BF16), I8)
    f8, fs = native.tokenwise_quant(torch.randn(64, 64, device="cuda").to(BF16), E4M3)
    return [(lambda x, w, b: layer_norm.layer_norm(x, w, b), (x, w, w.clone())),
            (lambda q, k: rotary.apply_rotary(q, k, None, freq), (q, k)),
            (lambda x: gated.q8_gated_linear(x, w8, None, None, ws), (x,)),
            (lambda x: gated.fp8_gated_linear(x, f8, None, None, fs), (x,)),
            (lambda x: gated.q8_gated_linear(x.to(torch.float16), w8, None, None, ws), (x,))]


@pytest.mark.parametrize("i", range(5))
@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("leaf", [False, True])
def test_tangents_are_refused(i, strided, leaf):
    from q8_kernels_b200 import Q8KernelError
    call, tensors = calls()[i]
    if strided:                                                # the Python bodies' inputs
        tensors = tuple(torch.stack([t, t], -1)[..., 0] for t in tensors)
    with fwd.dual_level():
        call(*tensors)                                         # a level alone refuses nothing
        for j, t in enumerate(tensors):
            t = t.clone().requires_grad_(True) if leaf else t
            dual = fwd.make_dual(t, torch.ones_like(t))
            with pytest.raises(Q8KernelError, match="forward-mode"):
                call(*tensors[:j], dual, *tensors[j + 1:])
    call(*tensors)


def test_module():
    from q8_kernels_b200 import Q8KernelError
    from q8_kernels_b200.modules import RotaryEmbedding
    m = RotaryEmbedding(64).cuda()
    q = torch.randn(3, 4, 64, device="cuda").to(BF16)
    with fwd.dual_level(), pytest.raises(Q8KernelError, match="forward-mode"):
        m(fwd.make_dual(q, torch.ones_like(q)))


def test_tangents_of_what_is_frozen():
    from q8_kernels_b200 import Q8KernelError, native
    from q8_kernels_b200.functional import gated, rotary
    x = torch.randn(12, 64, device="cuda").to(BF16)
    w, ws = native.tokenwise_quant(torch.randn(64, 64, device="cuda").to(BF16), I8)
    bias, freq = torch.zeros(64, device="cuda"), rotary.rotary_frequencies(64)[0].cuda()
    with fwd.dual_level():
        def dual(t):
            return fwd.make_dual(t, torch.ones_like(t))

        for bad in (lambda: gated.q8_gated_linear(x, w, dual(bias), None, ws), lambda: gated.q8_gated_linear(x, w, bias, None, dual(ws)),
                    lambda: rotary.apply_rotary(x.view(1, 3, 4, 64), None, None, dual(freq))):
            with pytest.raises(Q8KernelError, match="forward-mode"):
                bad()
