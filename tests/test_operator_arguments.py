"""Frequencies of the rotary embedding and the refusals of the entry points that need no GPU."""
import math

import pytest
import torch

from q8_kernels_b200 import Q8KernelError, _lib
from q8_kernels_b200.functional.rotary import rotary_frequencies


def test_plain_linear_and_ntk():
    f, a = rotary_frequencies(64)
    assert f.dtype == torch.float64 and f.shape == (32,) and a == 1.0
    for i in range(32):
        assert math.isclose(f[i].item(), 10000.0 ** (-2 * i / 64), rel_tol=1e-14)
    g, a = rotary_frequencies(64, scaling={"type": "linear", "factor": 4})
    assert torch.equal(g, f / 4) and a == 1.0
    g, a = rotary_frequencies(64, scaling={"type": "ntk", "factor": 8.0})
    assert g[0] == 1.0 and math.isclose(g[-1].item(), f[-1].item() / 8, rel_tol=1e-13) and a == 1.0


@pytest.mark.parametrize("r,base,n,factor", [(64, 10000.0, 4096, 32.0), (128, 500000.0, 8192, 8.0), (6, 10000.0, 4096, 2.0)])
def test_yarn(r, base, n, factor):
    f, _ = rotary_frequencies(r, base)
    g, a = rotary_frequencies(r, base, {"type": "yarn", "factor": factor, "original_length": n})
    assert math.isclose(a, 0.1 * math.log(factor) + 1.0)
    # whole turns within n positions of pair number i: n f / 2 pi; the ramp's ends are the pairs with 32 turns and with one
    low = max(math.floor(r * math.log(n / (32 * 2 * math.pi)) / (2 * math.log(base))), 0)
    high = min(math.ceil(r * math.log(n / (2 * math.pi)) / (2 * math.log(base))), r - 1)
    for i in range(r // 2):
        m = 0.0 if i <= low else 1.0 if i >= high else (i - low) / (high - low)
        assert math.isclose(g[i].item(), f[i].item() * ((1 - m) + m / factor), rel_tol=1e-13), i
    assert rotary_frequencies(r, base, {"type": "yarn", "factor": factor, "original_length": n, "amplitude": 1.0})[1] == 1.0


@pytest.mark.parametrize("args", [(0,), (7,), (-2,), (64, 1.0), (64, 1e4, {"type": "linear"}), (64, 1e4, {"type": "linear", "factor": 0.5}),
                                  (64, 1e4, {"type": "other", "factor": 2}), (64, 1e4, {"factor": 2}), (2, 1e4, {"type": "ntk", "factor": 2}),
                                  (64, 1e4, {"type": "yarn", "factor": 2}), (64, 1e4, {"type": "linear", "factor": 2, "beta_fast": 1}),
                                  (64, 1e4, {"type": "yarn", "factor": 2, "original_length": 4096, "beta_fast": 1, "beta_slow": 2})])
def test_refused_frequencies(args):
    with pytest.raises(Q8KernelError):
        rotary_frequencies(*args)


def test_refusals_of_the_c_entries():
    """Arguments are looked at before anything is launched."""
    import ctypes
    lib = _lib.lib
    buf = (torch.zeros(4096, dtype=torch.uint8).data_ptr() + 15) // 16 * 16
    bf, f32 = _lib.DT_BF16, _lib.DT_F32
    # layer norm: dim, type pair, null pointers, workspace
    assert lib.q8k_layer_norm(buf, bf, 0, None, None, buf, bf, None, None, 4, 0, 1e-5, None) == -1
    assert lib.q8k_layer_norm(buf, bf, 16385, None, None, buf, bf, None, None, 4, 16385, 1e-5, None) == -2
    assert lib.q8k_layer_norm(buf, bf, 64, None, None, buf, _lib.DT_F16, None, None, 4, 64, 1e-5, None) == -2
    assert lib.q8k_layer_norm(None, bf, 64, None, None, buf, bf, None, None, 4, 64, 1e-5, None) == -1
    assert lib.q8k_layer_norm(buf + 1, bf, 64, None, None, buf, bf, None, None, 4, 64, 1e-5, None) == -1
    assert lib.q8k_layer_norm(None, bf, 64, None, None, None, bf, None, None, 0, 64, 1e-5, None) == 0
    need = lib.q8k_layer_norm_backward_workspace_bytes(1000, 64)
    assert need > 0 and lib.q8k_layer_norm_backward_workspace_bytes(0, 64) == 0
    back = [buf, bf, 64, buf, bf, buf, buf, None, buf, buf, None, 1000, 64]
    assert lib.q8k_layer_norm_backward(*back, None, need, None) == -1
    assert lib.q8k_layer_norm_backward(*back, buf, need - 1, None) == -3
    # rotary: odd or too wide a part, type, null pointers; nothing to do
    s = (ctypes.c_int64 * 3)(64, 64, 64)

    def rotary(dtype=bf, q=buf, head=64, part=64, heads=1, batch=1, freq=buf):
        return lib.q8k_rotary(q, s, q, s, heads, None, None, None, None, 0, dtype, None, 0, 0, 0, freq, 1.0, batch, 1, head, part, 1, 0, None)

    assert rotary(part=63) == -1 and rotary(part=66) == -1 and rotary(part=0) == -1 and rotary(dtype=_lib.DT_E4M3) == -2
    assert rotary(q=None) == -1 and rotary(freq=None) == -1 and rotary(head=4098, part=64) == -2 and rotary(batch=-1) == -1
    assert rotary(heads=1 << 20) == -2
    assert rotary(batch=0) == 0 and rotary(heads=0) == 0
    # gated projection
    def mm(a=buf, pre=None, act=1, m=4, f=32, k=64):
        return lib.q8k_gated_mm(1, a, buf, None, buf, buf, buf, pre, act, m, f, k, None, None)

    assert mm(f=24) == -1 and mm(k=24) == -1 and mm(act=0) == -2 and mm(act=3) == -2 and mm(a=None) == -1 and mm(a=buf + 8) == -1
    assert mm(pre=buf + 4) == -1 and mm(m=-1) == -1 and mm(m=0) == 0
    assert lib.q8k_gated_backward_quant(buf, buf, buf, buf, 1, 4, 24, None) == -1
    assert lib.q8k_gated_backward_quant(buf, buf, buf, buf, 1, 4, 16400, None) == -2
    assert lib.q8k_gated_backward_quant(buf, None, buf, buf, 1, 4, 32, None) == -1
    assert lib.q8k_gated_backward_quant(buf, buf, buf, buf, 9, 4, 32, None) == -2
    need = lib.q8k_gated_weight_operand_workspace_bytes(32, 64)
    assert need > 0 and lib.q8k_gated_weight_operand_workspace_bytes(0, 64) == 0
    assert lib.q8k_gated_weight_operand(buf, _lib.DT_I8, buf, buf, buf, 32, 64, buf, need - 4, None) == -3
    assert lib.q8k_gated_weight_operand(buf, _lib.DT_I8, buf, buf, buf, 24, 64, buf, need, None) == -1
    assert lib.q8k_gated_weight_operand(buf, f32, buf, buf, buf, 32, 64, buf, need, None) == -2
    assert lib.q8k_gated_quant(buf, f32, 64, buf, _lib.DT_I8, buf, 4, 64, 0, None) == -2
    assert lib.q8k_gated_quant(buf, bf, 24, buf, _lib.DT_I8, buf, 4, 24, 0, None) == -1


def test_cpu_tensors_are_refused():
    from q8_kernels_b200.functional import gated, layer_norm, rotary
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(Q8KernelError):
        layer_norm.layer_norm(x)
    with pytest.raises(Q8KernelError):
        rotary.apply_rotary(x.view(1, 4, 1, 64), None, None, rotary_frequencies(64)[0])
    with pytest.raises(Q8KernelError):
        gated.q8_gated_linear(x, torch.zeros(64, 64, dtype=torch.int8), None, None, torch.zeros(64))


def test_native_path_looks_at_no_argument_of_a_call_with_a_wrong_number_of_them():
    from q8_kernels_b200 import _host
    for name, n in {"_layer_norm": 5, "_rotary": 6, "_gated_linear": 7}.items():
        for k in range(n + 3):
            if k != n:
                assert getattr(_host, name)(*[None] * k) is None
        assert getattr(_host, name)(*[torch.zeros(4, 64)] * n) is None


def test_gated_plan():
    """Rows of at most 128 take the 128-row tiles, many rows the pairs; tiles cover F and are of widths that the kernels take."""
    import ctypes
    lib = _lib.lib
    plan = (ctypes.c_int * 2)()

    def of(m, f, k):
        assert lib.q8k_gated_plan(m, f, k, plan) == 0
        return plan[0], plan[1]

    for m in (1, 8, 77, 128, 129, 256, 257, 1000, 6144, 100000):
        for f in (16, 48, 688, 1408, 5504, 8192, 10240, 16400, 40960):
            for k in (16, 512, 2048, 8192):
                pair, bn = of(m, f, k)
                assert (bn % 32 == 0 and 32 <= bn <= 128) if pair else (bn % 8 == 0 and 16 <= bn <= 128)
                assert not (m <= 128 and pair) and not (m >= 40000 and f >= 512 and not pair)
                if not pair and m > 128:                        # one round of tiles
                    assert -(-m // 128) * -(-f // bn) <= 148
    assert of(1, 8192, 2048) == (0, 56) and of(6144, 8192, 2048) == (1, 128)
    assert lib.q8k_gated_plan(0, 16, 16, plan) == -1 and lib.q8k_gated_plan(1, 16, 16, None) == -1
    # the call that does both steps: its refusals
    buf = (torch.zeros(4096, dtype=torch.uint8).data_ptr() + 255) // 256 * 256
    need = lib.q8k_gated_linear_workspace_bytes(4, 64)
    assert need >= 4 * 64 + 16 and lib.q8k_gated_linear_workspace_bytes(0, 64) == 0

    def linear(x=buf, xt=_lib.DT_BF16, wt=_lib.DT_I8, act=1, m=4, f=32, k=64, work=buf, size=need):
        return lib.q8k_gated_linear(x, xt, buf, wt, buf, None, buf, None, act, m, f, k, 1, work, size, None, None)

    assert linear(x=None) == -1 and linear(xt=_lib.DT_F16) == -2 and linear(wt=_lib.DT_BF16) == -2 and linear(act=7) == -2 and linear(f=24) == -1
    assert linear(k=40) == -1 and linear(work=None) == -1 and linear(work=buf + 16) == -1 and linear(size=need - 1) == -3 and linear(m=0) == 0


def test_whole_numbers_are_no_frequencies():
    from q8_kernels_b200.functional import rotary
    x = torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16)
    for freq in (torch.ones(32, dtype=torch.int64), torch.ones(32)):
        with pytest.raises(Q8KernelError, match="float64"):
            rotary.apply_rotary(x, None, None, freq)
