"""q8k_rotary with the output in the place of the input: the bits of a call with an output of its own, for both layouts, parts of a head, every
width of access, and more heads than a thread holds at a time; strides that overlap are refused there."""
import ctypes

import pytest
import torch

from helpers import bits

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
Strides = ctypes.c_int64 * 3


def rotate_in_place(q, k, pos, freq, half, backward=0):
    from q8_kernels_b200 import _lib
    b, s, _, d = q.shape
    code = {BF16: _lib.DT_BF16, F16: _lib.DT_F16, F32: _lib.DT_F32}[q.dtype]
    args = []
    for t in (q, k):
        args += [t.data_ptr(), Strides(*t.stride()[:3]), t.data_ptr(), Strides(*t.stride()[:3]), t.shape[2]]
    return _lib.lib.q8k_rotary(*args, code, pos.data_ptr(), 1, pos.stride(0), 1, freq.data_ptr(), 1.25, b, s, d, 2 * freq.numel(), half, backward,
                               torch.cuda.current_stream().cuda_stream)


# 16-, 8-, 4- and 2-byte accesses; whole heads and parts, odd heads; 40 and 24 heads: up to eight a thread, four loaded ahead
@pytest.mark.parametrize("d,r", [(64, 64), (128, 96), (96, 32), (80, 72), (100, 60), (66, 22), (67, 34)])
@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("b,s,hq,hk", [(2, 700, 40, 24), (3, 5, 3, 1)])
def test_in_place(d, r, half, dtype, b, s, hq, hk):
    from q8_kernels_b200 import native
    from q8_kernels_b200.functional.rotary import rotary_frequencies
    g = torch.Generator(device="cuda").manual_seed(d + r)
    qkv = torch.randn(b, s, hq + 2 * hk, d, generator=g, device="cuda").to(dtype)
    freq = rotary_frequencies(r)[0].cuda()
    pos = torch.randint(0, 5000, (b, s), generator=g, device="cuda")
    want = native.rotary(qkv[:, :, :hq], qkv[:, :, hq:hq + hk], pos, freq, 1.25, bool(half))
    own = qkv.clone()
    q, k = own[:, :, :hq], own[:, :, hq:hq + hk]
    assert rotate_in_place(q, k, pos, freq, half) == 0
    assert torch.equal(bits(q.contiguous()), bits(want[0])) and torch.equal(bits(k.contiguous()), bits(want[1]))
    assert torch.equal(bits(own[:, :, hq + hk:].contiguous()), bits(qkv[:, :, hq + hk:].contiguous()))
