"""Rotation by positions with several axes against complex products in 64 bits.

Tolerances count roundings as for one axis: one to the output's type, and in fp32 (u = 2^-24) 8 u of (|a| + |b|) amplitude for cosine and sine,
their products and the sum; the fraction of a turn is rounded to fp32 before (2^-25 of half a turn, 2^-23.3 radians, within the 8 u).
"""
import pytest
import torch

from helpers import bits

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24


def turned(x, positions, freq, axes, amplitude, layout, sign=1.0):
    """In 64 bits, and the size of what was added up."""
    r = 2 * freq.numel()
    p = positions.double()[..., axes.long().clamp(0, positions.shape[-1] - 1)]
    rot = torch.polar(torch.full_like(p, amplitude), sign * p * freq).unsqueeze(-2)
    x = x.double()
    out, size = x.clone(), torch.zeros_like(x)
    a, b = (slice(0, r, 2), slice(1, r, 2)) if layout == "interleaved" else (slice(0, r // 2), slice(r // 2, r))
    z = torch.complex(x[..., a], x[..., b]) * rot
    out[..., a], out[..., b] = z.real, z.imag
    size[..., a] = size[..., b] = (x[..., a].abs() + x[..., b].abs()) * amplitude
    return out, size


def check(y, x, positions, freq, axes, amplitude, layout, sign=1.0):
    ref, size = turned(x, positions, freq, axes, amplitude, layout, sign)
    f = torch.finfo(x.dtype)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    bad = (y.double() - ref).abs() > ref.abs() * (f.eps / 2) * 1.001 + f.tiny * f.eps + 8 * U * size
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {((y.double() - ref).abs()).max().item()}"
    assert torch.equal(bits(y[..., 2 * freq.numel():]), bits(x[..., 2 * freq.numel():]))


def angles(sections, base=10000.0, spectrum="own"):
    from q8_kernels_b200.functional.rotary import axial_frequencies
    f, a = axial_frequencies(sections, base, spectrum)
    return f.cuda(), a.cuda()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("t", [BF16, F16, F32])
@pytest.mark.parametrize("d,sections", [(64, (16, 24, 24)), (72, (36, 36)), (128, (32, 48, 48)), (80, (8, 12, 12)), (96, (2, 2, 2, 2)), (65, (4, 6)), (6, (2, 2, 2)),
                                        (256, (64,)), (512, (128, 384))])
def test_layouts_types_and_sizes(layout, t, d, sections):
    from q8_kernels_b200.functional.rotary import apply_axial_rotary
    g = torch.Generator(device="cuda").manual_seed(d)
    freq, axes = angles(sections, spectrum="shared" if d % 3 else "own")
    for b, s, hq, hk in ((1, 1, 1, 1), (2, 5, 3, 1), (3, 67, 8, 2)):
        q, k = (torch.randn(b, s, h, d, generator=g, device="cuda").to(t) for h in (hq, hk))
        pos = torch.randint(-50, 5000, (b, s, len(sections)), generator=g, device="cuda")
        before = q.clone()
        y, z = apply_axial_rotary(q, k, pos, freq, axes, 1.25, layout)
        check(y, q, pos, freq, axes, 1.25, layout)
        check(z, k, pos, freq, axes, 1.25, layout)
        assert torch.equal(bits(before), bits(q))


def test_positions_and_axes():
    from q8_kernels_b200.functional.rotary import apply_axial_rotary, apply_rotary, grid_positions
    freq, axes = angles((16, 24, 24))
    x = torch.randn(2, 60, 3, 64, device="cuda")
    grid = grid_positions(3, 4, 5, device="cuda")
    assert grid.shape == (60, 3) and grid[23].tolist() == [1, 0, 3]
    far = torch.randint(0, 1 << 20, (2, 60, 3), device="cuda")
    for p in (grid, grid[None], grid.int(), grid.expand(2, 60, 3), grid.float() * 0.04 + 0.5, grid.double() / 3, far, far.flip(0), far.double() + 0.25,
              torch.randint(0, 99, (3, 60, 2), device="cuda").permute(2, 1, 0), torch.randint(0, 99, (2, 120, 6), device="cuda")[:, ::2, ::2]):
        check(apply_axial_rotary(x, None, p, freq, axes)[0], x, p.expand(2, 60, 3), freq, axes, 1.0, "interleaved")
    # equal positions on all axes are one axis; any order of the pairs; an axis that there is not
    near = torch.arange(60, device="cuda")
    one = apply_rotary(x, None, near, freq, 1.0, "interleaved")[0]
    assert torch.equal(apply_axial_rotary(x, None, near[:, None].expand(60, 3), freq, axes)[0], one)
    mixed = torch.arange(32, device="cuda", dtype=torch.int32) % 3
    check(apply_axial_rotary(x, None, grid, freq, mixed)[0], x, grid.expand(2, 60, 3), freq, mixed, 1.0, "interleaved")
    for beyond in (3, 1 << 30, -1):
        last = torch.full((32,), beyond, dtype=torch.int32, device="cuda")
        assert torch.equal(apply_axial_rotary(x, None, grid, freq, last)[0], apply_axial_rotary(x, None, grid, freq, torch.full_like(last, 2))[0])
    # a position that is no number spoils its own token's pairs of that axis only
    bad = grid.float().clone()
    bad[7, 1] = float("nan")
    bad[8, 0] = float("inf")
    y = apply_axial_rotary(x, None, bad, freq, axes)[0]
    nan = torch.isnan(y)
    assert nan[:, 7, :, 16:40].all() and nan[:, 8, :, :16].all() and int(nan.sum()) == 2 * 3 * (24 + 16)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_strides_empty_and_long_offsets(layout):
    from q8_kernels_b200.functional.rotary import apply_axial_rotary
    freq, axes = angles((16, 24, 24))
    qkv = torch.randn(2, 33, 6, 72, device="cuda").to(BF16)
    pos = torch.randint(0, 999, (2, 33, 3), device="cuda")
    for q in (qkv[:, :, :4], qkv.transpose(1, 2).contiguous().transpose(1, 2), torch.randn(2, 33, 4, 75, device="cuda").to(BF16)[..., 1:73],
              torch.randn(2, 33, 72, 4, device="cuda").to(BF16).transpose(2, 3), qkv[:, :, :1].expand(2, 33, 4, 72)):
        y, z = apply_axial_rotary(q, qkv[:, :, 4:], pos, freq, axes, 1.0, layout)
        check(y, q, pos, freq, axes, 1.0, layout)
        check(z, qkv[:, :, 4:], pos, freq, axes, 1.0, layout)
    y, z = apply_axial_rotary(qkv[0], None, pos[0], freq, axes, 1.0, layout)         # [S,H,D]
    assert z is None
    check(y, qkv[0], pos[0], freq, axes, 1.0, layout)
    for empty in (qkv[:0], qkv[:, :0], qkv[:, :, :0]):
        assert apply_axial_rotary(empty, None, pos[:empty.shape[0], :empty.shape[1]], freq, axes, 1.0, layout)[0].shape == empty.shape
    store = torch.zeros(2 ** 31 + 4096, dtype=BF16, device="cuda")
    q = store.as_strided((2, 3, 2, 64), (2 ** 31, 128, 64, 1))
    q.copy_(torch.randn(2, 3, 2, 64, device="cuda"))
    check(apply_axial_rotary(q, None, pos[:, :3], freq, axes, 1.0, layout)[0], q, pos[:, :3], freq, axes, 1.0, layout)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("t,d", [(BF16, 64), (F16, 80), (F32, 70)])
def test_gradients(layout, t, d):
    from q8_kernels_b200.functional.rotary import apply_axial_rotary
    freq, axes = angles((16, 24, 24))
    qkv = torch.randn(2, 21, 9, d, device="cuda").to(t)
    q, k = qkv[:, :, :6].detach().requires_grad_(True), qkv[:, :, 6:8].detach().requires_grad_(True)
    pos = torch.rand(2, 21, 3, device="cuda", dtype=torch.float64) * 500
    y, z = apply_axial_rotary(q, k, pos, freq, axes, 1.5, layout)
    gy, gz = torch.randn_like(y), torch.randn_like(z)
    dq, dk = torch.autograd.grad([y, z], [q, k], [gy, gz], retain_graph=True)
    check(dq, gy, pos, freq, axes, 1.5, layout, sign=-1.0)
    check(dk, gz, pos, freq, axes, 1.5, layout, sign=-1.0)
    only = torch.autograd.grad(z, [k], gz.transpose(0, 1).contiguous().transpose(0, 1), retain_graph=True)[0]     # not dense, q unused
    assert torch.equal(bits(only), bits(dk))
    broadcast = torch.autograd.grad(y.sum(), [q])[0]                                  # a gradient of stride 0
    check(broadcast, torch.ones_like(y), pos, freq, axes, 1.5, layout, sign=-1.0)
    # differences: the map is linear, <g, R v> = <R' g, v>
    if t == F32:
        v = torch.randn_like(q)
        rv = apply_axial_rotary(q.detach() + v, None, pos, freq, axes, 1.5, layout)[0].double() - apply_axial_rotary(q.detach() - v, None, pos, freq, axes, 1.5, layout)[0]
        left, right = (gy.double() * rv).sum() / 2, (dq.double() * v.double()).sum()
        # 16 u of each product's size, added up as a random walk, with 8 for its tail
        assert abs(left - right) <= 8 * 16 * U * 2 * 1.5 * v.numel() ** 0.5 * 4


def test_module_captured_and_on_another_stream():
    from q8_kernels_b200.modules import AxialRotaryEmbedding
    m = AxialRotaryEmbedding(64, (16, 24, 24), base=(1000.0, 10000.0, 10000.0)).cuda()
    assert m.state_dict() == {}
    q, k = torch.randn(4, 6, 8, 64, device="cuda").to(BF16), torch.randn(4, 6, 2, 64, device="cuda").to(BF16)
    pos = torch.randint(0, 70000, (4, 6, 3), device="cuda")
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
    check(fresh[0], q, pos, m.frequencies, m.axes, 1.0, "interleaved")


def test_refusals():
    from q8_kernels_b200 import Q8KernelError
    from q8_kernels_b200.functional.rotary import apply_axial_rotary
    from q8_kernels_b200.modules import AxialRotaryEmbedding
    freq, axes = angles((16, 24, 24))
    q = torch.zeros(2, 5, 3, 64, device="cuda", dtype=BF16)
    pos = torch.zeros(2, 5, 3, device="cuda", dtype=torch.int64)
    m = AxialRotaryEmbedding(64, (16, 24, 24)).cuda()
    for bad in (lambda: apply_axial_rotary(q, q.half(), pos, freq, axes), lambda: apply_axial_rotary(q, q[:, :4], pos, freq, axes),
                lambda: apply_axial_rotary(q, None, pos.half(), freq, axes), lambda: apply_axial_rotary(q, None, pos[:, :4], freq, axes),
                lambda: apply_axial_rotary(q, None, pos[..., 0], freq, axes), lambda: apply_axial_rotary(q, None, pos[..., :0], freq, axes),
                lambda: apply_axial_rotary(q, None, None, freq, axes), lambda: apply_axial_rotary(q, None, pos, freq.float(), axes),
                lambda: apply_axial_rotary(q, None, pos, freq, axes.long()), lambda: apply_axial_rotary(q, None, pos, freq, axes[:-1]),
                lambda: apply_axial_rotary(q, None, pos, freq, axes.cpu()), lambda: apply_axial_rotary(q, None, pos.cpu(), freq, axes),
                lambda: apply_axial_rotary(q[..., :62], None, pos, freq, axes), lambda: apply_axial_rotary(q, None, pos, freq, axes, 1.0, "pairs"),
                lambda: apply_axial_rotary(q.double(), None, pos, freq, axes), lambda: apply_axial_rotary(q, None, pos, freq[:0], axes[:0]),
                lambda: apply_axial_rotary(q, None, pos, freq, None), lambda: m(q, None, pos[..., :2]), lambda: m(q[..., :32], None, pos)):
        with pytest.raises(Q8KernelError):
            bad()
