"""Norm of every head with the rotation in the same pass, against the formulas in 64 bits and differences of them.

Tolerances in fp32 roundings (u = 2^-24).  Forward: the sum of squares adds 16 values a lane and 5 times over lanes (21 u, half of it in its
root), mean and eps 1 u, rsqrt 4 u, two products 2 u, the rotation 8 u of (|a| + |b|): below 32 u of that size.  Backward: the rotation of the
gradient 8 u and its product with the weight 1 u, the sum of u x 21 u and twice the 15 u of rstd, the final products 5 u: below 64 u of
rstd (|u| + |x| rstd^2 mean(|u x|)), |u| the size of the rotated gradient times the weight.  The weights' gradients add up rows: of the sizes
here at most 200 one after the other in a thread, a CTA and over CTAs, with 26 u for a term: 256 u of the sum of sizes.  And half a step
of the output's type.
"""
import pytest
import torch

from helpers import bits

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24


def rotation(x, positions, freq, axes, amplitude, layout, sign=1.0):
    """x in 64 bits turned, and the size of what was added up for each channel."""
    if freq is None:
        return x, x.abs()
    r = 2 * freq.numel()
    p = positions.double()
    p = p.unsqueeze(-1) if axes is None else p[..., axes.long()]
    rot = torch.polar(torch.full_like(p * freq, amplitude), sign * p * freq).unsqueeze(-2)
    out, size = x.clone(), x.abs().clone()
    a, b = (slice(0, r, 2), slice(1, r, 2)) if layout == "interleaved" else (slice(0, r // 2), slice(r // 2, r))
    z = torch.complex(x[..., a], x[..., b]) * rot
    out[..., a], out[..., b] = z.real, z.imag
    size[..., a] = size[..., b] = (x[..., a].abs() + x[..., b].abs()) * amplitude
    return out, size


def forward(x, w, eps, angle):
    x = x.double()
    z = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    return rotation(z if w is None else z * w.double(), *angle)


def near(y, ref, slack):
    f = torch.finfo(y.dtype)
    bad = (y.double() - ref).abs() > ref.abs() * (f.eps / 2) * 1.001 + f.tiny * f.eps + slack * 1.01
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {((y.double() - ref).abs() - ref.abs() * f.eps / 2).max().item()}"


def check(y, x, w, eps, angle):
    ref, size = forward(x, w, eps, angle)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    near(y, ref, 32 * U * size)


def check_grads(dx, dw, x, w, g, eps, angle):
    x, g = x.detach().double(), g.double()
    rstd = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    t, size = rotation(g, *angle, -1.0) if angle[1] is not None else (g, g.abs())
    ww = torch.ones(x.shape[-1], device=x.device, dtype=torch.float64) if w is None else w.detach().double()
    u, us = t * ww, size * ww.abs()
    near(dx, rstd * (u - x * rstd ** 2 * (u * x).mean(-1, keepdim=True)), 64 * U * rstd * (us + x.abs() * rstd ** 2 * (us * x.abs()).mean(-1, keepdim=True)))
    if dw is not None:
        dims = tuple(range(x.dim() - 1))
        assert dw.dtype == F32 and dw.shape == (x.shape[-1],)
        near(dw, (t * x * rstd).sum(dims), 256 * U * (size * x.abs() * rstd).sum(dims))


def angles(kind, r, b, s, layout, g=None):
    """(positions, frequencies, axes, amplitude, layout) of no rotation, one axis or three."""
    from q8_kernels_b200.functional.rotary import axial_frequencies, rotary_frequencies
    if kind == "none":
        return None, None, None, 1.0, layout
    if kind == "one":
        f, amp = rotary_frequencies(r, 10000.0, {"type": "yarn", "factor": 4, "original_length": 512})
        return torch.randint(0, 5000, (b, s), device="cuda"), f.cuda(), None, amp, layout
    first = max(2, r // 8 * 2)
    second = max(2, (r - first) // 4 * 2)
    f, a = axial_frequencies((first, second, r - first - second))
    return torch.rand(b, s, 3, device="cuda", dtype=F32) * 300, f.cuda(), a.cuda(), 1.0, layout


@pytest.mark.parametrize("kind", ["none", "one", "axes"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("t", [BF16, F16, F32])
@pytest.mark.parametrize("d,r", [(64, 64), (128, 128), (72, 72), (80, 32), (96, 96), (128, 50), (256, 256), (192, 104), (65, 10), (512, 512), (6, 6), (509, 508), (36, 20)])
def test_layouts_types_and_sizes(kind, layout, t, d, r):
    from q8_kernels_b200.functional.head_norm import head_norm
    g = torch.Generator(device="cuda").manual_seed(d + r)
    for b, s, hq, hk in ((1, 1, 1, 1), (2, 5, 3, 1), (2, 67, 12, 2)):
        q, k = ((torch.randn(b, s, h, d, generator=g, device="cuda") * torch.exp(2 * torch.randn(b, s, h, 1, generator=g, device="cuda"))).to(t)
                .requires_grad_(True) for h in (hq, hk))
        wq, wk = ((1 + 0.3 * torch.randn(d, generator=g, device="cuda")).requires_grad_(True) for _ in range(2))
        if s == 5:
            wq = None
        angle = angles(kind, r, b, s, layout)
        with torch.no_grad():
            plain = head_norm(q, k, wq, wk, 1e-6, *angle[:4], layout)
        y, z = head_norm(q, k, wq, wk, 1e-6, *angle[:4], layout)
        assert torch.equal(bits(plain[0]), bits(y)) and torch.equal(bits(plain[1]), bits(z))
        check(y.detach(), q.detach(), wq, 1e-6, angle)
        check(z.detach(), k.detach(), wk, 1e-6, angle)
        gy, gz = torch.randn(y.shape, generator=g, device="cuda").to(t), torch.randn(z.shape, generator=g, device="cuda").to(t)
        leaves = [q, k, wk] + ([wq] if wq is not None else [])
        dq, dk, dwk, *dwq = torch.autograd.grad([y, z], leaves, [gy, gz])
        check_grads(dq, dwq[0] if dwq else None, q, wq, gy, 1e-6, angle)
        check_grads(dk, dwk, k, wk, gz, 1e-6, angle)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d", [64, 72])
def test_strides_shapes_and_parts(layout, d):
    from q8_kernels_b200.functional.head_norm import head_norm
    angle = angles("axes", d - 8, 2, 33, layout)
    w = 1 + 0.1 * torch.randn(d, device="cuda")
    qkv = torch.randn(2, 33, 6, d, device="cuda").to(BF16)
    k = qkv[:, :, 4:]
    for q in (qkv[:, :, :4], qkv.transpose(1, 2).contiguous().transpose(1, 2), torch.randn(2, 33, 4, d + 3, device="cuda").to(BF16)[..., 1:d + 1],
              torch.randn(2, 33, d, 4, device="cuda").to(BF16).transpose(2, 3), qkv[:, :, :1].expand(2, 33, 4, d), qkv[:1].expand(2, 33, 6, d)):
        leaf = q.detach().requires_grad_(True)
        assert leaf.stride() == q.stride()
        y, z = head_norm(leaf, k, w, None, 1e-5, *angle[:4], layout)
        check(y.detach(), q, w, 1e-5, angle)
        check(z, k, None, 1e-5, angle)
        gy = torch.randn(2, 4 if q.shape[2] == 4 else 6, 33, d, device="cuda").to(BF16).transpose(1, 2)          # a strided gradient
        dq, = torch.autograd.grad(y, [leaf], gy)
        check_grads(dq, None, q, w, gy, 1e-5, angle)
    y, z = head_norm(qkv, None, w, None, 1e-5, *angle[:4], layout)
    assert z is None
    check(y, qkv, w, 1e-5, angle)
    one = (angle[0][0], *angle[1:])                            # [S,H,D]
    y, z = head_norm(qkv[0, :, :4], qkv[0, :, 4:], w, w, 1e-5, *one[:4], layout)
    check(y, qkv[0, :, :4], w, 1e-5, one)
    check(z, qkv[0, :, 4:], w, 1e-5, one)
    for empty in (qkv[:0], qkv[:, :0], qkv[:, :, :0]):
        p = angle[0][:empty.shape[0], :empty.shape[1]]
        leaf, lw = empty.detach().requires_grad_(True), w.clone().requires_grad_(True)
        y = head_norm(leaf, None, lw, None, 1e-5, p, *angle[1:4], layout)[0]
        dx, dw = torch.autograd.grad(y, [leaf, lw], torch.zeros_like(y))
        assert y.shape == empty.shape and dx.shape == empty.shape and torch.equal(dw, torch.zeros(d, device="cuda"))
    y, z = head_norm(qkv[:, :, :0], qkv[:, :, 4:], w, w, 1e-5, *angle[:4], layout)
    check(z, qkv[:, :, 4:], w, 1e-5, angle)


def test_long_offsets_and_many_tokens():
    """More than 2^31 elements between two batch entries' tokens; more tokens than the backward pass has CTAs for at a time."""
    from q8_kernels_b200.functional.head_norm import head_norm
    store = torch.zeros(2 ** 31 + 4096, dtype=BF16, device="cuda")
    q = store.as_strided((2, 3, 2, 64), (2 ** 31, 128, 64, 1))
    q.copy_(torch.randn(2, 3, 2, 64, device="cuda"))
    angle = angles("one", 64, 2, 3, "half")
    w = 1 + 0.1 * torch.randn(64, device="cuda")
    leaf = q.detach().requires_grad_(True)
    y = head_norm(leaf, None, w, None, 1e-6, *angle[:4])[0]
    check(y.detach(), q, w, 1e-6, angle)
    gy = torch.randn_like(y)
    check_grads(torch.autograd.grad(y, [leaf], gy)[0], None, q, w, gy, 1e-6, angle)
    del store, q, leaf, y
    x, w = torch.randn(1, 20011, 3, 128, device="cuda").to(BF16).requires_grad_(True), w.repeat(2).requires_grad_(True)
    angle = angles("axes", 96, 1, 20011, "interleaved")
    y = head_norm(x, None, w, None, 1e-6, *angle[:4], "interleaved")[0]
    gy = torch.randn_like(y)
    dx, dw = torch.autograd.grad(y, [x, w], gy, retain_graph=True)
    check_grads(dx, dw, x, w, gy, 1e-6, angle)
    again = torch.autograd.grad(y, [x, w], gy)
    assert torch.equal(bits(again[0]), bits(dx)) and torch.equal(bits(again[1]), bits(dw))


@pytest.mark.parametrize("kind", ["one", "axes"])
def test_differences(kind):
    """<gradient, v> against the central difference of the 64-bit formula along v: its error is 1e-8 of the third derivative's size, which is
    below 100 times the output's, and the kernel's is bounded by its elements' roundings."""
    from q8_kernels_b200.functional.head_norm import head_norm
    angle = angles(kind, 48, 2, 9, "half")
    x = torch.randn(2, 9, 3, 64, device="cuda").requires_grad_(True)
    w = (1 + 0.2 * torch.randn(64, device="cuda")).requires_grad_(True)
    y = head_norm(x, None, w, None, 1e-6, *angle[:4])[0]
    g = torch.randn_like(y)
    dx, dw = torch.autograd.grad(y, [x, w], g)
    vx, vw, h = torch.randn_like(x).double(), torch.randn_like(w).double(), 1e-4

    def f(sx, sw):
        return (forward(x.detach().double() + sx * h * vx, w.detach().double() + sw * h * vw, 1e-6, angle)[0] * g.double()).sum()

    size = g.abs().double().sum()
    assert abs((f(1, 0) - f(-1, 0)) / (2 * h) - (dx.double() * vx).sum()) <= (100e-8 + 200 * U * 4) * size
    assert abs((f(0, 1) - f(0, -1)) / (2 * h) - (dw.double() * vw).sum()) <= (100e-8 + 256 * U * 4) * size


def test_parts_of_the_gradient():
    from q8_kernels_b200.functional.head_norm import head_norm
    angle = angles("one", 64, 2, 21, "half")
    qkv = torch.randn(2, 21, 8, 64, device="cuda").to(BF16)
    q, k = qkv[:, :, :6].detach().requires_grad_(True), qkv[:, :, 6:].detach().requires_grad_(True)
    wq, wk = (torch.ones(64, device="cuda", requires_grad=True) for _ in range(2))
    y, z = head_norm(q, k, wq, wk, 1e-6, *angle[:4])
    gy, gz = torch.randn_like(y), torch.randn_like(z)
    full = torch.autograd.grad([y, z], [q, k, wq, wk], [gy, gz], retain_graph=True)
    assert torch.equal(bits(torch.autograd.grad(z, [k], gz, retain_graph=True)[0]), bits(full[1]))
    # (the order of the weights' sums is that of the call's shape: two calls with other heads agree within the bound, not in bits)
    check_grads(full[1], torch.autograd.grad(z, [wk], gz, retain_graph=True)[0], k, wk, gz, 1e-6, angle)
    unused = torch.autograd.grad(z, [q, k, wq, wk], gz, allow_unused=True, retain_graph=True)
    assert unused[0] is None and unused[2] is None and torch.equal(bits(unused[1]), bits(full[1]))
    check_grads(full[0], torch.autograd.grad([y, z], [wq], [gy, gz])[0], q, wq, gy, 1e-6, angle)
    y, z = head_norm(q.detach(), k, wq.detach(), wk.detach(), 1e-6, *angle[:4])       # one input has a gradient
    assert torch.equal(bits(torch.autograd.grad(z, [k], gz)[0]), bits(full[1]))
    # one weight for both: the gradients add up
    shared = torch.ones(64, device="cuda", requires_grad=True)
    y, z = head_norm(q, k, shared, shared, 1e-6, *angle[:4])
    assert torch.equal(torch.autograd.grad([y, z], [shared], [gy, gz])[0], full[2] + full[3])
    with pytest.raises(RuntimeError):
        y, z = head_norm(q, k, shared, None, 1e-6, *angle[:4])
        torch.autograd.grad(torch.autograd.grad(y, [q], gy.requires_grad_(True), create_graph=True)[0].float().sum(), [gy])


def test_values_that_are_not_finite():
    """A head with NaN or an infinity is spoilt, its neighbours are not; a head of zeros stays zeros, the largest values of a type do not."""
    from q8_kernels_b200.functional.head_norm import head_norm
    angle = angles("one", 32, 1, 4, "half")
    x = torch.randn(1, 4, 3, 64, device="cuda")
    x[0, 1, 1, 5], x[0, 2, 0, 60] = float("nan"), float("inf")
    x[0, 3, 2] = 0
    y = head_norm(x, None, None, None, 1e-6, *angle[:4])[0]
    spoilt = torch.isnan(y).any(-1)[0]
    assert spoilt.nonzero().tolist() == [[1, 1], [2, 0]]
    assert not y[0, 3, 2].any()
    for t in (BF16, F16):                                      # squares beyond the type, within fp32
        big = torch.full((1, 4, 1, 64), 6e4, device="cuda").to(t)
        check(head_norm(big, None, None, None, 1e-6, *angle[:4])[0], big, None, 1e-6, angle)


def test_module_captured_and_on_another_stream():
    from q8_kernels_b200.modules import AxialRotaryEmbedding, HeadNormRotary, RotaryEmbedding
    m = HeadNormRotary(64, AxialRotaryEmbedding(64, (16, 24, 24))).cuda()
    assert set(m.state_dict()) == {"q_weight", "k_weight"}
    m.q_weight.data.add_(0.1 * torch.randn(64, device="cuda"))
    q, k = torch.randn(2, 12, 8, 64, device="cuda").to(BF16), torch.randn(2, 12, 2, 64, device="cuda").to(BF16)
    pos = torch.randint(0, 700, (2, 12, 3), device="cuda")
    with torch.no_grad():
        eager = m(q, k, pos)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            other = m(q, k, pos)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m(q, k, pos)
        pos += 3
        q.mul_(2)
        graph.replay()
        fresh = m(q, k, pos)
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(eager, other))
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(out, fresh))
    check(fresh[0], q, m.q_weight.detach(), 1e-6, (pos, m.rotary.frequencies, m.rotary.axes, 1.0, "interleaved"))
    cast = HeadNormRotary(64, RotaryEmbedding(64)).cuda().to(BF16)                    # weights of 16 bits are widened
    y, _ = cast(q, None, pos[..., 0])
    check(y.detach(), q, None, 1e-6, (pos[..., 0], cast.rotary.frequencies, None, 1.0, "half"))
    plain = HeadNormRotary(64, elementwise_affine=False)
    assert not list(plain.parameters())
    check(plain(q)[0], q, None, 1e-6, (None, None, None, 1.0, "half"))


def test_captured_backward():
    """Forward and backward in one graph, replayed on other contents, beside the eager passes of other leaves."""
    from q8_kernels_b200.functional.head_norm import head_norm
    angle = angles("axes", 64, 2, 40, "interleaved")
    x, w = torch.randn(2, 40, 4, 64, device="cuda").to(BF16), torch.rand(64, device="cuda") + 0.5
    g = torch.randn(2, 40, 4, 64, device="cuda").to(BF16)

    def step(x, w):
        x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        y = head_norm(x, None, w, None, 1e-6, *angle[:4], "interleaved")[0]
        return (y.detach(), *torch.autograd.grad(y, [x, w], g))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(x, w)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, w)
    x.copy_(torch.randn_like(x))
    graph.replay()
    for a, b in zip(out, step(x, w)):
        assert torch.equal(bits(a), bits(b))


def test_refusals():
    from q8_kernels_b200 import Q8KernelError
    from q8_kernels_b200.functional.head_norm import head_norm
    from q8_kernels_b200.modules import AxialRotaryEmbedding, HeadNormRotary, RotaryEmbedding
    pos, freq, axes, _, _ = angles("axes", 64, 2, 5, "half")
    q = torch.zeros(2, 5, 3, 64, device="cuda", dtype=BF16)
    w = torch.ones(64, device="cuda")
    for bad in (lambda: head_norm(q, q.half()), lambda: head_norm(q, q[:, :4]), lambda: head_norm(q, None, w[:32]), lambda: head_norm(q, None, w.half()),
                lambda: head_norm(q, None, w.cpu()), lambda: head_norm(q, None, None, None, -1.0), lambda: head_norm(q, None, None, None, float("nan")),
                lambda: head_norm(q, None, None, None, 1e-6, pos), lambda: head_norm(q, None, None, None, 1e-6, pos, freq),
                lambda: head_norm(q, None, None, None, 1e-6, None, freq, axes), lambda: head_norm(q, None, None, None, 1e-6, None, None, axes),
                lambda: head_norm(q, None, None, None, 1e-6, pos[:, :4], freq, axes), lambda: head_norm(q, None, None, None, 1e-6, None, freq[:0]),
                lambda: head_norm(q[..., :32], None, None, None, 1e-6, pos, freq, axes), lambda: head_norm(q.double()), lambda: head_norm(q.cpu()),
                lambda: head_norm(q[0, 0]), lambda: head_norm(torch.zeros(1, 2, 3, 520, device="cuda")), lambda: head_norm(q, layout="pairs"),
                lambda: HeadNormRotary(64, RotaryEmbedding(32)), lambda: HeadNormRotary(64, torch.nn.Identity()), lambda: HeadNormRotary(32).cuda()(q),
                lambda: HeadNormRotary(64).cuda()(q, None, pos), lambda: HeadNormRotary(64, AxialRotaryEmbedding(64, (32, 32))).cuda()(q, None, pos)):
        with pytest.raises(Q8KernelError):
            bad()
