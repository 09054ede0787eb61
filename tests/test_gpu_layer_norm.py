"""Layer norm against its formula in 64 bits: types, odd sizes, strides, which gradients, capture.

Tolerances count roundings.  One to the output's type: eps / 2 of the value (and half a step of the subnormals).  In fp32, with
u = 2^-24: a sum of n values in threads of at most 32 values, then a tree, is off by at most (32 + 16) u times the sum of the
magnitudes; the rest of a formula adds some ten roundings.  64 u times the magnitudes that enter covers both.
"""
import pytest
import torch

from helpers import bits

pytestmark = pytest.mark.gpu
BF16, F16, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
U = 2.0 ** -24
SHAPES = [(1, 1), (1, 2), (3, 7), (5, 16), (9, 250), (6, 256), (3, 257), (7, 1024), (2, 1031), (5, 1537), (130, 2048), (700, 48), (2, 4095),
          (3, 8192), (2, 10239), (3, 16384), (2, 16383)]


def step(t, ref):
    f = torch.finfo(t)
    return ref.abs() * (f.eps / 2) + f.tiny * f.eps


def rows(r, d, t, seed=0, offset=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(r, d, generator=g, device="cuda") + offset * torch.randn(r, 1, generator=g, device="cuda")
    return x.to(t), 1 + 0.2 * torch.randn(d, generator=g, device="cuda"), 0.2 * torch.randn(d, generator=g, device="cuda"), \
        torch.randn(r, d, generator=g, device="cuda").to(t)


def check_forward(y, x, w, b, eps):
    x, w, b = x.double(), (torch.ones(1, device="cuda") if w is None else w).double(), (torch.zeros(1, device="cuda") if b is None else b).double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    ref = (x - mean) * rstd * w + b
    # the mean's error moves every z, the variance's scales it
    err = 64 * U * (rstd * (x.abs() + x.abs().mean(-1, keepdim=True)) * w.abs() + b.abs())
    assert y.shape == ref.shape
    bad = (y.double() - ref).abs() > step(y.dtype, ref) * 1.001 + err
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}"
    return mean, rstd


def check_backward(got, x, w, g, eps):
    x, g = x.double(), g.double()
    w = torch.ones(x.shape[-1], dtype=torch.float64, device="cuda") if w is None else w.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    z, gw = (x - mean) * rstd, g * w
    dx = rstd * (gw - gw.mean(-1, keepdim=True) - z * (gw * z).mean(-1, keepdim=True))
    # what z is off by, and with it the products
    dz = 64 * U * rstd * (x.abs() + x.abs().mean(-1, keepdim=True))
    m = (gw.abs() * (z.abs() + dz)).mean(-1, keepdim=True)
    err = rstd * (64 * U * (gw.abs() + gw.abs().mean(-1, keepdim=True) + z.abs() * m)
                  + dz * m + z.abs() * (gw.abs() * dz).mean(-1, keepdim=True))
    if got[0] is not None:
        bad = (got[0].double() - dx).abs() > step(got[0].dtype, dx) * 1.001 + err
        assert not bad.any(), f"dx: {int(bad.sum())} of {bad.numel()}"
    r = x.shape[0]
    # a column's sum: at most r / groups values one after the other, then the groups; r + 64 roundings at the very most
    n = min(r, 400) + 64
    for name, a, ref, mag in (("dw", got[1], (g * z).sum(0), (g.abs() * (z.abs() * n * U + dz)).sum(0)), ("db", got[2], g.sum(0), g.abs().sum(0) * n * U)):
        if a is not None:
            assert a.dtype == F32 and ((a.double() - ref).abs() <= mag + 1e-30).all(), name


@pytest.mark.parametrize("r,d", SHAPES)
@pytest.mark.parametrize("t,out", [(BF16, None), (F16, None), (F32, None), (F32, BF16), (F32, F16), (BF16, E4M3)])
def test_forward(r, d, t, out):
    from q8_kernels_b200.functional.layer_norm import layer_norm
    x, w, b, _ = rows(r, d, t, seed=r + d, offset=3.0)
    for ww, bb in ((w, b), (w, None), (None, None)):
        y = layer_norm(x, ww, bb, 1e-5, out)
        assert y.dtype == (out or t)
        check_forward(y, x, ww, bb, 1e-5)


@pytest.mark.parametrize("r,d", SHAPES)
@pytest.mark.parametrize("t,out", [(BF16, None), (F16, None), (F32, None), (F32, BF16), (F32, F16)])
def test_backward(r, d, t, out):
    from q8_kernels_b200.functional.layer_norm import layer_norm
    x, w, b, g = rows(r, d, t, seed=r + 3 * d)
    for v in (x, w, b):
        v.requires_grad_(True)
    g = g.to(out or t)
    y = layer_norm(x, w, b, 1e-5, out)
    got = torch.autograd.grad(y, [x, w, b], g)
    assert got[0].dtype == t and got[0].shape == x.shape
    check_backward(got, x.detach(), w.detach(), g, 1e-5)


@pytest.mark.parametrize("need", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (1, 0, 1), (0, 1, 1)])
@pytest.mark.parametrize("d", [512, 517])
def test_which_gradients(need, d):
    from q8_kernels_b200.functional.layer_norm import layer_norm
    x, w, b, g = rows(33, d, BF16, seed=4)
    leaves = [v.requires_grad_(bool(n)) for v, n in zip((x, w, b), need)]
    y = layer_norm(*leaves, 1e-6)
    wanted = [v for v in leaves if v.requires_grad]
    it = iter(torch.autograd.grad(y, wanted, g))
    check_backward([next(it) if n else None for n in need], x.detach(), w.detach(), g, 1e-6)


def test_without_weight_and_with_weight_only():
    from q8_kernels_b200.functional.layer_norm import layer_norm
    x, w, _, g = rows(17, 768, F32, seed=8)
    x.requires_grad_(True)
    check_backward([torch.autograd.grad(layer_norm(x), [x], g)[0], None, None], x.detach(), None, g, 1e-5)
    w.requires_grad_(True)
    dx, dw = torch.autograd.grad(layer_norm(x, w), [x, w], g)
    check_backward([dx, dw, None], x.detach(), w.detach(), g, 1e-5)


@pytest.mark.parametrize("t", [BF16, F32])
def test_strides(t):
    from q8_kernels_b200.functional.layer_norm import layer_norm
    big, w, b, g = rows(24, 1100, t, seed=5)
    views = [big[:, 3:1027], big[:, 8:1032], big[::2, :1024], big[:, :1024].reshape(2, 3, 4, 1024).transpose(0, 2), big[:1024, :24].T[:, :24],
             big[0, :1024].expand(6, 1024), big[5, 1:600]]
    for x in views:
        d = x.shape[-1]
        leaf = x.detach().requires_grad_(True)                  # keeps the strides
        y = layer_norm(leaf, w[:d], b[:d])
        flat = leaf.detach().reshape(-1, d)
        check_forward(y.detach().reshape(-1, d), flat, w[:d], b[:d], 1e-5)
        gr = torch.randn(y.shape, device="cuda").to(t)
        dx = torch.autograd.grad(y, [leaf], gr)[0]
        assert dx.shape == leaf.shape
        check_backward([dx.reshape(-1, d), None, None], flat, w[:d], gr.reshape(-1, d), 1e-5)
    # a gradient that is not dense, and a broadcast one
    x = big[:, :1024].detach().requires_grad_(True)
    y = layer_norm(x, w[:1024], b[:1024])
    wide = torch.randn(24, 2048, device="cuda").to(t)
    check_backward([torch.autograd.grad(y, [x], wide[:, ::2], retain_graph=True)[0], None, None], x.detach(), w[:1024], wide[:, ::2], 1e-5)
    one = torch.ones((), device="cuda", dtype=t).expand(24, 1024)
    check_backward([torch.autograd.grad(y, [x], one)[0], None, None], x.detach(), w[:1024], one, 1e-5)


def test_far_mean_and_empty_rows():
    from q8_kernels_b200.functional.layer_norm import layer_norm
    x, w, b, _ = rows(6, 2048, F32, seed=6)
    x = x * 0.01 + 1000.0                                      # E[x^2] - mean^2 would have no digit left
    check_forward(layer_norm(x, w, b), x, w, b, 1e-5)
    c = torch.full((3, 640), 7.0, device="cuda", dtype=BF16)    # no spread: z = 0
    assert torch.equal(layer_norm(c, w[:640].contiguous(), b[:640].contiguous()), b[:640].to(BF16).expand(3, 640))
    e = torch.empty(0, 640, device="cuda", dtype=BF16, requires_grad=True)
    ww = w[:640].clone().requires_grad_(True)
    y = layer_norm(e, ww, None)
    dx, dw = torch.autograd.grad(y, [e, ww], torch.empty_like(y))
    assert y.shape == (0, 640) and dx.shape == (0, 640) and torch.equal(dw, torch.zeros_like(dw))


def test_not_finite_rows_stay_alone():
    from q8_kernels_b200.functional.layer_norm import layer_norm
    x, w, b, g = rows(8, 1000, BF16, seed=7)
    x[2, 5], x[4, 9] = float("nan"), float("inf")
    y = layer_norm(x, w, b)
    assert y[2].isnan().all() and y[4].isnan().any()
    keep = [0, 1, 3, 5, 6, 7]
    check_forward(y[keep], x[keep], w, b, 1e-5)


def test_same_bits_every_time():
    from q8_kernels_b200.native import layer_norm, layer_norm_backward
    for r, d in ((5000, 256), (3001, 1537), (4096, 2048)):
        x, w, b, g = rows(r, d, BF16, seed=9)
        _, m, s = layer_norm(x, w, b, 1e-5, None, True)
        first = layer_norm_backward(x, m, s, g, w, True, True, True)
        for _ in range(3):
            again = layer_norm_backward(x, m, s, g, w, True, True, True)
            assert all(torch.equal(bits(p), bits(q)) for p, q in zip(first, again))


@pytest.mark.parametrize("d", [768, 2048, 1537])
def test_gradients_against_differences(d):
    """Along a random direction v of unit length: (L(x + h v) - L(x - h v)) / 2h of the fp32 kernel, L = sum(y g).  L is rounded by at most 64 u
    sum|y g| on each side, and the third derivative along a unit direction is below 30 times the gradient's scale (|g| rstd^3)."""
    from q8_kernels_b200.functional.layer_norm import layer_norm
    x, w, b, g = rows(4, d, F32, seed=d)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(*leaves), leaves, g)
    with torch.no_grad():
        for i, grad in enumerate(grads):
            v = torch.randn_like(leaves[i])
            v /= v.norm()
            h = 0.05

            def loss(s):
                args = [t.detach() for t in leaves]
                args[i] = args[i] + s * v
                return (layer_norm(*args).double() * g.double()).sum()

            got = (grad.double() * v.double()).sum()
            diff = (loss(h) - loss(-h)) / (2 * h)
            size = (layer_norm(x, w, b).double() * g.double()).abs().sum()
            # rounding of both sides as random walk: sqrt(n) of the mean rounding, with 16 for the tail
            rounding = 16 * 64 * U * size / (4 * d) ** 0.5 / h
            truncation = 30 * h * h * g.double().norm() / d ** 0.5
            assert abs(got - diff) <= rounding + truncation, (i, got.item(), diff.item())


def test_captured_and_on_another_stream():
    from q8_kernels_b200.functional.layer_norm import layer_norm
    x, w, b, g = rows(300, 1024, BF16, seed=11)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def step_():
        y = layer_norm(*leaves)
        return (y.detach(),) + torch.autograd.grad(y, leaves, g)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            on_stream = step_()
    torch.cuda.current_stream().wait_stream(s)
    eager = step_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step_()
    with torch.no_grad():
        x.copy_(torch.randn_like(x))
    graph.replay()
    fresh = step_()
    torch.cuda.synchronize()
    assert all(torch.equal(bits(p), bits(q)) for p, q in zip(on_stream, eager))
    assert all(torch.equal(bits(p), bits(q)) for p, q in zip(out, fresh))


def test_module():
    from q8_kernels_b200.modules import LayerNorm
    m = LayerNorm(512, eps=1e-6).cuda()
    assert set(m.state_dict()) == {"weight", "bias"}
    x, w, b, g = rows(40, 512, BF16, seed=12)
    m.weight.data, m.bias.data = w, b
    x.requires_grad_(True)
    y = m(x.view(4, 10, 512))
    assert y.shape == (4, 10, 512)
    check_forward(y.detach().view(40, 512), x.detach(), w, b, 1e-6)
    y.backward(g.view(4, 10, 512))
    check_backward([x.grad, m.weight.grad, m.bias.grad], x.detach(), w, g, 1e-6)
    assert list(LayerNorm(64, elementwise_affine=False).parameters()) == [] and LayerNorm(64, bias=False).bias is None
    assert m(x, out_dtype=E4M3).dtype == E4M3


def test_refusals():
    from q8_kernels_b200 import Q8KernelError
    from q8_kernels_b200.functional.layer_norm import layer_norm
    x, w, b, _ = rows(4, 64, BF16)
    for bad in (lambda: layer_norm(x, w.to(BF16), b), lambda: layer_norm(x, w[:63], b), lambda: layer_norm(x, w, b, 1e-5, F16),
                lambda: layer_norm(x.to(torch.int8), w, b), lambda: layer_norm(x.cpu(), w, b), lambda: layer_norm(x, w.cpu(), b),
                lambda: layer_norm(torch.zeros(2, 16400, device="cuda")), lambda: layer_norm(x[:, :0]), lambda: layer_norm(x, w.view(1, 64), b)):
        with pytest.raises(Q8KernelError):
            bad()


@pytest.mark.parametrize("r,d", [(20000, 40), (20000, 500), (12000, 760), (12000, 777), (12000, 1000), (8000, 1500), (8000, 1537), (6000, 2040),
                                 (4000, 3000), (4000, 4000), (1500, 5000), (1500, 5001), (1200, 8000), (1200, 10240)])
@pytest.mark.parametrize("t", [BF16, F32])
def test_more_rows_than_the_ring_holds(r, d, t):
    """Every group of threads comes by each slot of its ring again."""
    from q8_kernels_b200 import native
    x, w, b, g = rows(r, d, t, seed=r + d, offset=2.0)
    y, mean, rstd = native.layer_norm(x, w, b, 1e-5, None, True)
    check_forward(y, x, w, b, 1e-5)
    g = g.to(t)
    check_backward(native.layer_norm_backward(x, mean, rstd, g, w, True, True, True), x, w, g, 1e-5)
    dx = native.layer_norm_backward(x, mean, rstd, g, w, True, False, False)[0]
    check_backward([dx, None, None], x, w, g, 1e-5)
