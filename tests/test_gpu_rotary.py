"""Rotary embedding from positions against complex products in 64 bits.

Tolerances count roundings: one to the output's type, and in fp32 (u = 2^-24) cosine and sine (2 u each, and amplitude's product) and the
two products and the sum: 8 u of |a| + |b|.  The fraction of a turn is rounded to fp32 (2^-25 of half a turn, 2^-23.3 radians); in
64 bits an angle of 2^31 is good to 2^-21, on both sides.
"""
import pytest
import torch

from helpers import bits

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24


def reference(x, positions, freq, amplitude, layout, sign=1.0):
    r = 2 * freq.numel()
    angle = positions.double().unsqueeze(-1) * freq
    rot = torch.polar(torch.full_like(angle, amplitude), sign * angle).unsqueeze(-2)
    x = x.double()
    out = x.clone()
    a, b = (slice(0, r, 2), slice(1, r, 2)) if layout == "interleaved" else (slice(0, r // 2), slice(r // 2, r))
    z = torch.complex(x[..., a], x[..., b]) * rot
    out[..., a], out[..., b] = z.real, z.imag
    size = torch.zeros_like(x)
    size[..., a] = size[..., b] = (x[..., a].abs() + x[..., b].abs()) * amplitude
    return out, size


def check(y, x, positions, freq, amplitude, layout, sign=1.0, far=1.0):
    ref, size = reference(x, positions, freq, amplitude, layout, sign)
    f = torch.finfo(x.dtype)
    assert y.dtype == x.dtype and y.shape == x.shape
    bad = (y.double() - ref).abs() > ref.abs() * (f.eps / 2) * 1.001 + f.tiny * f.eps + far * 8 * U * size
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {((y.double() - ref).abs()).max().item()}"
    assert torch.equal(bits(y[..., 2 * freq.numel():]), bits(x[..., 2 * freq.numel():]))


def frequencies(r, base=10000.0, scaling=None):
    from q8_kernels_b200.functional.rotary import rotary_frequencies
    f, a = rotary_frequencies(r, base, scaling)
    return f.cuda(), a


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("t", [BF16, F16, F32])
@pytest.mark.parametrize("d,r", [(64, 64), (64, 32), (96, 32), (80, 80), (128, 128), (128, 126), (256, 2), (2, 2), (65, 10), (192, 104), (512, 512)])
def test_layouts_types_and_sizes(layout, t, d, r):
    from q8_kernels_b200.functional.rotary import apply_rotary
    g = torch.Generator(device="cuda").manual_seed(d + r)
    freq, amp = frequencies(r, scaling={"type": "yarn", "factor": 4, "original_length": 2048})
    for b, s, hq, hk in ((1, 1, 1, 1), (2, 5, 3, 1), (3, 67, 8, 2)):
        q, k = (torch.randn(b, s, h, d, generator=g, device="cuda").to(t) for h in (hq, hk))
        pos = torch.randint(0, 5000, (b, s), generator=g, device="cuda")
        before = q.clone()
        y, z = apply_rotary(q, k, pos, freq, amp, layout)
        check(y, q, pos, freq, amp, layout)
        check(z, k, pos, freq, amp, layout)
        assert torch.equal(bits(before), bits(q))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d", [64, 72])
def test_strides_and_shapes(layout, d):
    from q8_kernels_b200.functional.rotary import apply_rotary
    freq, amp = frequencies(d - 8)
    qkv = torch.randn(2, 33, 6, d, device="cuda").to(BF16)
    pos = torch.arange(33, device="cuda").expand(2, 33) + 7
    heads_first = torch.randn(2, 4, 33, d, device="cuda").to(BF16).transpose(1, 2)
    offset = torch.randn(2, 33, 4, d + 3, device="cuda").to(BF16)[..., 1:d + 1]
    other_last = torch.randn(2, 33, d, 4, device="cuda").to(BF16).transpose(2, 3)
    for q in (qkv[:, :, :4], heads_first, offset, other_last, qkv[:, :, :1].expand(2, 33, 4, d), qkv[:1].expand(2, 33, 6, d)[:, ::1]):
        y, z = apply_rotary(q, qkv[:, :, 4:], pos, freq, amp, layout)
        check(y, q, pos, freq, amp, layout)
        check(z, qkv[:, :, 4:], pos, freq, amp, layout)
        assert y.is_contiguous()
    y, z = apply_rotary(qkv, None, pos, freq, amp, layout)
    assert z is None
    check(y, qkv, pos, freq, amp, layout)
    packed = qkv[0]                                            # [S,H,D]
    y, z = apply_rotary(packed[:, :4], packed[:, 4:], pos[0], freq, amp, layout)
    check(y, packed[:, :4], pos[0], freq, amp, layout)
    check(z, packed[:, 4:], pos[0], freq, amp, layout)
    for empty in (qkv[:0], qkv[:, :0], qkv[:, :, :0]):
        p = pos[:empty.shape[0], :empty.shape[1]]
        assert apply_rotary(empty, None, p, freq, amp, layout)[0].shape == empty.shape
    y, z = apply_rotary(qkv[:, :, :0], qkv[:, :, 4:], pos, freq, amp, layout)
    check(z, qkv[:, :, 4:], pos, freq, amp, layout)


def test_positions():
    from q8_kernels_b200.functional.rotary import apply_rotary
    freq, amp = frequencies(64)
    x = torch.randn(3, 50, 2, 64, device="cuda")
    near = torch.arange(50, device="cuda")
    for p in (near, near[None], near.int(), near.expand(3, 50), -near, torch.randint(0, 1 << 20, (3, 50), device="cuda"),
              torch.randint(0, 1 << 20, (50, 3), device="cuda").T, torch.arange(100, device="cuda")[::2], torch.zeros(3, 50, device="cuda").int()):
        check(apply_rotary(x, None, p, freq, amp)[0], x, p.expand(3, 50), freq, amp, "half")
    check(apply_rotary(x, None, None, freq, amp)[0], x, near.expand(3, 50), freq, amp, "half")
    far = torch.randint(1 << 30, (1 << 31) + 9, (3, 50), device="cuda")
    check(apply_rotary(x, None, far, freq, amp)[0], x, far, freq, amp, "half", far=4.0)


def test_long_offsets():
    """More than 2^31 elements between two batch entries' tokens."""
    from q8_kernels_b200.functional.rotary import apply_rotary
    store = torch.zeros(2 ** 31 + 4096, dtype=BF16, device="cuda")
    q = store.as_strided((2, 3, 2, 64), (2 ** 31, 128, 64, 1))
    q.copy_(torch.randn(2, 3, 2, 64, device="cuda"))
    freq, amp = frequencies(64)
    pos = torch.arange(3, device="cuda").expand(2, 3)
    check(apply_rotary(q, None, pos, freq, amp)[0], q, pos, freq, amp, "half")


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("t,d,r", [(BF16, 128, 128), (F16, 96, 32), (F32, 64, 62)])
def test_gradients(layout, t, d, r):
    from q8_kernels_b200.functional.rotary import apply_rotary
    freq, amp = frequencies(r, scaling={"type": "yarn", "factor": 16, "original_length": 512})
    qkv = torch.randn(2, 21, 9, d, device="cuda").to(t)
    q, k = qkv[:, :, :6].detach().requires_grad_(True), qkv[:, :, 6:8].detach().requires_grad_(True)
    pos = torch.randint(0, 9000, (2, 21), device="cuda")
    y, z = apply_rotary(q, k, pos, freq, amp, layout)
    gy, gz = torch.randn_like(y), torch.randn_like(z)
    dq, dk = torch.autograd.grad([y, z], [q, k], [gy, gz], retain_graph=True)
    check(dq, gy, pos, freq, amp, layout, sign=-1.0)
    check(dk, gz, pos, freq, amp, layout, sign=-1.0)
    # one output unused, a gradient that is not dense, one input without a gradient
    only = torch.autograd.grad(z, [k], gz.transpose(0, 1).contiguous().transpose(0, 1), retain_graph=True)[0]
    assert torch.equal(bits(only), bits(dk))
    assert torch.equal(bits(torch.autograd.grad(y, [q], gy)[0]), bits(dq))
    y, z = apply_rotary(q.detach(), k, pos, freq, amp, layout)
    assert torch.equal(bits(torch.autograd.grad([y.sum() + (z * gz).sum()], [k])[0]), bits(dk))
    # the map is linear: its difference along v is its value at v, and <g, R v> = <R'g, v>
    if t == F32:
        v = torch.randn_like(q)
        rv = apply_rotary(q.detach() + v, None, pos, freq, amp, layout)[0].double() - apply_rotary(q.detach() - v, None, pos, freq, amp, layout)[0]
        left, right = (gy.double() * rv).sum() / 2, (dq.double() * v.double()).sum()
        # 16 u of each product's size, added up as a random walk, with 8 for its tail
        assert abs(left - right) <= 8 * 16 * U * 2 * amp * v.numel() ** 0.5 * 4


def test_captured_other_stream_and_module():
    from q8_kernels_b200.modules import RotaryEmbedding
    m = RotaryEmbedding(64, 48, layout="interleaved", scaling={"type": "linear", "factor": 2.0}).cuda()
    assert m.state_dict() == {}
    q, k = torch.randn(4, 1, 8, 64, device="cuda").to(BF16), torch.randn(4, 1, 2, 64, device="cuda").to(BF16)
    pos = torch.tensor([[5], [70000], [0], [31]], device="cuda")
    eager = m(q, k, pos)
    cast = m.to(BF16)                                          # the frequencies stay 64-bit
    assert cast.frequencies.dtype == torch.float64
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = cast(q, k, pos)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m(q, k, pos)
    pos += 3
    graph.replay()
    fresh = m(q, k, pos)
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(eager, other))
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(out, fresh))
    check(fresh[0], q, pos, m.frequencies, 1.0, "interleaved")


def test_refusals():
    from q8_kernels_b200 import Q8KernelError
    from q8_kernels_b200.functional.rotary import apply_rotary
    freq, _ = frequencies(64)
    q = torch.zeros(2, 5, 3, 64, device="cuda", dtype=BF16)
    pos = torch.zeros(2, 5, device="cuda", dtype=torch.int64)
    for bad in (lambda: apply_rotary(q, q.half(), pos, freq), lambda: apply_rotary(q, q[:, :4], pos, freq), lambda: apply_rotary(q, q[..., :32], pos, freq),
                lambda: apply_rotary(q, None, pos.float(), freq), lambda: apply_rotary(q, None, pos[:, :4], freq), lambda: apply_rotary(q, None, pos.T, freq),
                lambda: apply_rotary(q, None, pos, freq.float()), lambda: apply_rotary(q[..., :62], None, pos, freq), lambda: apply_rotary(q, None, pos, freq, 1.0, "pairs"),
                lambda: apply_rotary(q.double(), None, pos, freq), lambda: apply_rotary(q, None, pos.cpu(), freq), lambda: apply_rotary(q, None, pos, freq[:0]),
                lambda: apply_rotary(q[0, 0], None, pos, freq), lambda: apply_rotary(q.cpu(), None, pos.cpu(), freq.cpu())):
        with pytest.raises(Q8KernelError):
            bad()
