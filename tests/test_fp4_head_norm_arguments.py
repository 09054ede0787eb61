"""Axial frequencies, and refusals of the 4-bit linears', head norms' and axial rotary's entry points that need no GPU."""
import ctypes
import math

import pytest
import torch

from q8_kernels_b200 import Q8KernelError, _lib
from q8_kernels_b200.functional.rotary import axial_frequencies, grid_positions, rotary_frequencies


def test_axial_frequencies():
    f, a = axial_frequencies((16, 24, 24))
    assert f.dtype == torch.float64 and a.dtype == torch.int32 and f.shape == a.shape == (32,)
    assert a.tolist() == [0] * 8 + [1] * 12 + [2] * 12
    for n, (lo, c) in enumerate(((0, 16), (8, 24), (20, 24))):
        for j in range(c // 2):
            assert math.isclose(f[lo + j].item(), 10000.0 ** (-2 * j / c), rel_tol=1e-14)
    f, _ = axial_frequencies((16, 24, 24), 100.0, "shared")
    assert torch.equal(f, rotary_frequencies(64, 100.0)[0])
    f, _ = axial_frequencies((4, 4), (100.0, 10000.0))
    assert torch.equal(f, torch.cat([rotary_frequencies(4, 100.0)[0], rotary_frequencies(4, 10000.0)[0]]))


@pytest.mark.parametrize("args", [((),), ((16, 23),), ((0, 16),), ((16.0,),), ((16, 16), 1.0), ((16, 16), (1e4,)), ((16, 16), (1e4, 1e3), "shared"),
                                  ((16, 16), 1e4, "each"), ((-2, 4),)])
def test_refused_axial_frequencies(args):
    with pytest.raises(Q8KernelError):
        axial_frequencies(*args)


def test_grid_positions():
    p = grid_positions(2, 3, 4)
    assert p.shape == (24, 3) and p.dtype == torch.int64
    assert all(p[i].tolist() == [i // 12, i // 4 % 3, i % 4] for i in range(24))
    for bad in ((), (0, 3), (2.0, 3)):
        with pytest.raises(Q8KernelError):
            grid_positions(*bad)


def test_refusals_of_the_c_entries():
    lib = _lib.lib
    buf = (torch.zeros(8192, dtype=torch.uint8).data_ptr() + 255) // 256 * 256
    bf, f16, f32 = _lib.DT_BF16, _lib.DT_F16, _lib.DT_F32
    s = (ctypes.c_int64 * 3)(64, 64, 64)

    def axial(kind=2, axes=buf, n_axes=3, pos=buf, freq=buf, part=64, strides=s, batch=1):
        return lib.q8k_axial_rotary(buf, s, buf, s, 1, None, None, None, None, 0, bf, pos, kind, strides, n_axes, axes, freq, 1.0, batch, 1, 64, part, 1, 0,
                                    None)

    assert axial(kind=0) == -1 and axial(kind=5) == -1 and axial(axes=None) == -1 and axial(axes=buf + 2) == -1 and axial(n_axes=0) == -1
    assert axial(pos=None) == -1 and axial(pos=buf + 4) == -1 and axial(freq=None) == -1 and axial(part=63) == -1 and axial(strides=None) == -1
    assert axial(batch=0) == 0

    def norm(dtype=bf, q=buf, out=buf, head=64, part=64, heads=1, batch=1, pos=buf, strides=s, freq=buf, w=buf, qs=s):
        return lib.q8k_head_norm(q, qs, w, out, s, heads, None, None, None, None, None, 0, dtype, 1e-6, pos, 2, strides, 1, None, freq, 1.0, batch, 1, head,
                                 part, 1, None)

    assert norm(dtype=_lib.DT_E4M3) == -2 and norm(q=None) == -1 and norm(out=None) == -1 and norm(q=buf + 1) == -1 and norm(qs=None) == -1
    assert norm(head=520) == -2 and norm(part=66) == -1 and norm(part=63) == -1 and norm(part=-2) == -1 and norm(heads=-1) == -1 and norm(batch=-1) == -1
    assert norm(strides=None) == -1 and norm(freq=None) == -1 and norm(w=buf + 2) == -1 and norm(heads=1 << 20) == -2
    assert norm(batch=0) == 0 and norm(heads=0) == 0
    need = lib.q8k_head_norm_backward_workspace_bytes(64)
    assert need > 0 and lib.q8k_head_norm_backward_workspace_bytes(0) == 0

    def back(dw=buf, g=buf, work=buf, size=need):
        return lib.q8k_head_norm_backward(buf, s, buf, g, s, buf, s, dw, 1, None, None, None, None, None, None, None, None, 0, bf, 1e-6, buf, 2, s, 1, None,
                                          buf, 1.0, 1, 1, 64, 64, 1, work, size, None)

    assert back(work=None) == -1 and back(work=buf + 4) == -1 and back(size=need - 1) == -3 and back(g=None) == -1
    # 4 bits
    assert lib.q8k_fp4_scale_bytes(1, 129, 288) == 2 * 2 * 1024 and lib.q8k_fp4_scale_bytes(2, 128, 256) == 2048
    assert lib.q8k_fp4_scale_bytes(3, 128, 256) == 0 and lib.q8k_fp4_scale_bytes(2, 0, 256) == 0

    def quant(x=buf, dtype=bf, stride=64, fmt=2, q=buf, rs=buf, rows=4, k=64):
        return lib.q8k_fp4_quant(x, dtype, stride, fmt, q, buf, rs, rows, k, None)

    assert quant(fmt=0) == -2 and quant(fmt=3) == -2 and quant(dtype=f32) == -2 and quant(k=48) == -1 and quant(k=0) == -1 and quant(k=65568) == -2
    assert quant(x=None) == -1 and quant(x=buf + 8) == -1 and quant(q=buf + 4) == -1 and quant(rs=None) == -1 and quant(stride=60) == -1
    assert quant(stride=68) == -1 and quant(rows=-1) == -1 and quant(rows=0) == 0
    assert lib.q8k_fp4_dequant(buf, buf, None, 2, buf, bf, 4, 64, None) == -1 and lib.q8k_fp4_dequant(buf, buf, buf, 2, buf, _lib.DT_I8, 4, 64, None) == -2
    assert lib.q8k_fp4_dequant(buf, buf, buf, 2, buf, bf, 0, 64, None) == 0

    def mm(fmt=2, a=buf, rs=buf, out=buf, dtype=bf, m=4, n=32, k=64):
        return lib.q8k_fp4_mm(fmt, a, buf, rs, buf, buf, rs, None, out, dtype, m, n, k, 0, None, None)

    assert mm(fmt=9) == -2 and mm(a=None) == -1 and mm(a=buf + 8) == -1 and mm(rs=None) == -1 and mm(out=buf + 2) == -1 and mm(dtype=f32) == -2
    assert mm(n=24) == -1 and mm(k=48) == -1 and mm(m=-1) == -1 and mm(m=0) == 0
    need = lib.q8k_fp4_linear_workspace_bytes(2, 40, 32, 64)
    assert need >= 40 * 32 + 2048 + 160 and lib.q8k_fp4_linear_workspace_bytes(2, 0, 32, 64) == 0
    assert [lib.q8k_fp4_linear_workspace_bytes(1, m, n, k) == 0 for m, n, k in ((8, 32, 1024), (8, 32, 1056), (9, 32, 64), (1, 64, 8192), (1, 64, 8224),
                                                                               (1, 28416, 64), (1, 28432, 64))] == [True, False, False, True, False, True, False]

    def linear(x=buf, dtype=bf, out_dtype=f16, m=40, n=32, k=64, work=buf, size=need):
        return lib.q8k_fp4_linear(2, x, dtype, buf, buf, buf, None, buf, out_dtype, m, n, k, 0, work, size, None, None)

    assert linear(x=None) == -1 and linear(dtype=f32) == -2 and linear(n=24) == -1 and linear(k=48) == -1
    assert linear(work=None) == -1 and linear(work=buf + 16) == -1 and linear(size=need - 1) == -3 and linear(m=0) == 0
    # a few rows, without a workspace
    for bad, rc in ((dict(x=None), -1), (dict(x=buf + 8), -1), (dict(dtype=f32), -2), (dict(out_dtype=f32), -2), (dict(n=24), -1), (dict(k=48), -1)):
        assert linear(**{"m": 4, "work": None, "size": 0, **bad}) == rc, bad
    need = lib.q8k_fp4_weight_operand_workspace_bytes(32, 64)
    assert need > 0 and lib.q8k_fp4_weight_operand_workspace_bytes(0, 64) == 0

    def operand(fmt=2, n=32, k=64, rs=buf, work=buf, size=need):
        return lib.q8k_fp4_weight_operand(fmt, buf, buf, rs, buf, buf, n, k, work, size, None)

    assert operand(fmt=0) == -2 and operand(n=24) == -1 and operand(n=0) == -1 and operand(k=48) == -1 and operand(rs=None) == -1
    assert operand(work=None) == -1 and operand(size=need - 4) == -3
    # an output of fp16 is for e4m3 operands without GELU
    assert lib.q8k_q8_mm(buf, buf, None, buf, buf, buf, f16, 1, 1, 8, 16, 64, 0, None, None) == -2
    assert lib.q8k_fp8_mm(buf, buf, None, buf, buf, buf, f16, 1, 1, 8, 16, 64, 1, None, None) == -2


def test_modules_need_positions_of_their_axes():
    from q8_kernels_b200.modules import AxialRotaryEmbedding, HeadNormRotary
    rotary = AxialRotaryEmbedding(64, (32, 32))
    q = torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16)
    for m in (rotary, HeadNormRotary(64, rotary)):
        for positions in (None, torch.zeros(4), torch.zeros(4, 3)):
            with pytest.raises(Q8KernelError, match="2 axes"):
                m(q, None, positions)


def test_cpu_tensors_are_refused():
    from q8_kernels_b200.functional import fp4, head_norm, rotary
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    freq, axes = axial_frequencies((32, 32))
    with pytest.raises(Q8KernelError):
        fp4.fp4_quantize(x)
    with pytest.raises(Q8KernelError):
        head_norm.head_norm(x.view(1, 4, 1, 64))
    with pytest.raises(Q8KernelError):
        rotary.apply_axial_rotary(x.view(1, 4, 1, 64), None, torch.zeros(4, 2), freq, axes)
