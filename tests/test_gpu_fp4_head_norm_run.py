"""4-bit linears, head norms and rotations together, as a video transformer's attention block runs them: eager, captured, on two streams, with their
gradients; their native calls against the Python bodies; derivatives they refuse.

Tolerances.  A norm with rotation is held against the formula in 64 bits at the inputs it got: sums of up to 64 squares, factors and the rotation
are off by at most 80 fp32 steps of what is added up, then one rounding to bf16.  A gradient through two 4-bit linears: each rounds both factors of
a product to e4m3, by at most 2^-4 of themselves, so its gradient is off by at most 2^-3 + 2^-8 of the sizes it adds up; as its errors are
independent of each other that is a share of the norms, not of the sums of sizes, with 2 to spare.  bf16 between the parts adds 2^-9 each.
"""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from helpers import bits

pytestmark = pytest.mark.gpu
BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
E4M3 = torch.float8_e4m3fn


class Block(torch.nn.Module):
    """x -> projection -> norm and rotation of queries and keys -> attention -> projection."""

    def __init__(self, dim, heads, fmt):
        from q8_kernels_b200.modules import AxialRotaryEmbedding, FP4Linear, HeadNormRotary
        super().__init__()
        full = [torch.nn.Linear(dim, n, device="cuda", dtype=BF16) for n in (3 * dim, dim)]
        self.heads = heads
        self.qkv, self.out = (FP4Linear.from_linear(f, fmt) for f in full)
        self.norm = HeadNormRotary(64, AxialRotaryEmbedding(64, (16, 24, 24), device="cuda"), device="cuda")
        with torch.no_grad():
            for w in self.norm.parameters():
                w.add_(0.1 * torch.randn(64, device="cuda"))

    def project(self, x, positions):
        q, k, v = self.qkv(x).view(*x.shape[:2], 3, self.heads, 64).unbind(2)
        return (q, k, v, *self.norm(q, k, positions))

    def forward(self, x, positions):
        from q8_kernels_b200.functional.flash_attention import flash_attn_func
        _, _, v, q, k = self.project(x, positions)
        y = flash_attn_func(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), out_dtype=BF16, token_major_out=True)
        return self.out(y.transpose(1, 2).reshape(x.shape))


def norm_rotation(x, w, positions, rotary, eps=1e-6):
    """In 64 bits, and the size of what was added up."""
    x = x.double()
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    turn = positions.double()[..., rotary.axes.long()] * rotary.frequencies
    z = torch.polar(torch.ones_like(turn), turn).unsqueeze(-2) * torch.view_as_complex(y.unflatten(-1, (-1, 2)).contiguous())
    size = y.abs().unflatten(-1, (-1, 2)).sum(-1, keepdim=True).expand(*y.shape[:-1], -1, 2).flatten(-2)
    return torch.view_as_real(z).flatten(-2), size


def grid(b, t, h, w):
    from q8_kernels_b200.functional.rotary import grid_positions
    p = grid_positions(t, h, w, device="cuda")
    return p if b is None else p.expand(b, -1, -1).contiguous()


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("b,size,heads", [(1, (1, 1, 1), 2), (2, (3, 5, 7), 4), (1, (4, 16, 16), 6)])
def test_block(fmt, b, size, heads):
    from q8_kernels_b200 import check_status
    from q8_kernels_b200.functional.fp4 import fp4_dequantize, fp4_quantize
    torch.manual_seed(5)
    block = Block(64 * heads, heads, fmt)
    pos = grid(b, *size)
    x = torch.randn(b, pos.shape[1], 64 * heads, device="cuda").to(BF16)
    with torch.no_grad():
        y = block(x, pos)
        q, k, v, qn, kn = block.project(x, pos)
        # the projection against the de-quantised operands
        weight = fp4_dequantize(block.qkv.weight.data, block.qkv.weight_scales, F32).double()
        values = fp4_dequantize(*fp4_quantize(x, fmt), F32).double()
        ref = values @ weight.T + block.qkv.bias.double()
        size_of = values.abs() @ weight.abs().T + block.qkv.bias.abs().double()
        got = torch.stack([q, k, v], 2).flatten(2).double()
        assert ((got - ref).abs() <= ref.abs() * 2.0 ** -8 * 1.01 + (64 * heads // 64 + 40) * 2.0 ** -23 * size_of).all()
        for t, n, w in ((q, qn, block.norm.q_weight), (k, kn, block.norm.k_weight)):
            ref, size_of = norm_rotation(t, w, pos, block.norm.rotary)
            assert ((n.double() - ref).abs() <= ref.abs() * 2.0 ** -8 * 1.01 + 80 * 2.0 ** -24 * size_of + 1e-38).all()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            other = block(x, pos)
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(bits(other), bits(y)) and torch.isfinite(y).all()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = block(x, pos)
        x.copy_(torch.randn_like(x))
        pos.add_(2)
        graph.replay()
        assert torch.equal(bits(out), bits(block(x, pos)))
    check_status()


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_gradients_through_the_block(fmt):
    """The framework's attention has no gradient; a plain product of queries and keys stands in its place."""
    from q8_kernels_b200 import check_status
    from q8_kernels_b200.functional.fp4 import fp4_dequantize
    torch.manual_seed(6)
    heads, dim = 4, 256
    block = Block(dim, heads, fmt)
    pos = grid(2, 2, 4, 5)
    x = torch.randn(2, 40, dim, device="cuda").to(BF16).requires_grad_(True)
    g = torch.randn(2, 40, dim, device="cuda").to(BF16)

    def mixed(q, k, v):
        return (torch.einsum("bshd,bthd->bhst", q, k) / 8).softmax(-1).to(v.dtype) @ v.transpose(1, 2)

    q, k, v, qn, kn = block.project(x, pos)
    y = block.out(mixed(qn.float(), kn.float(), v.float()).transpose(1, 2).reshape(x.shape).to(BF16))
    got = torch.autograd.grad(y, [x, block.norm.q_weight, block.norm.k_weight], g)
    check_status()
    # the same chain in 64 bits at the same projections
    w_in, w_out = (fp4_dequantize(m.weight.data, m.weight_scales, F32).double() for m in (block.qkv, block.out))
    p = torch.stack([q, k, v], 2).detach().double().requires_grad_(True)
    wq, wk = (w.detach().double().requires_grad_(True) for w in block.norm.parameters())
    a, b = norm_rotation(p[:, :, 0], wq, pos, block.norm.rotary)[0], norm_rotation(p[:, :, 1], wk, pos, block.norm.rotary)[0]
    mid = mixed(a, b, p[:, :, 2]).transpose(1, 2).reshape(x.shape)
    dp, dq, dk = torch.autograd.grad(mid, [p, wq, wk], g.double() @ w_out)
    ref = (dp.flatten(2) @ w_in, dq, dk)
    one = 2.0 ** -3 + 2.0 ** -8                                # of one 4-bit linear's gradient
    for r, h, linears in zip(ref, got, (2, 1, 1)):
        assert h.shape == r.shape and (h.double() - r).norm() <= 2 * linears * one * r.norm(), ((h.double() - r).norm() / r.norm()).item()


def step_of(kind):
    """A step (leaves -> outputs and gradients), contents for its inputs."""
    from q8_kernels_b200.functional import fp4, rotary
    if kind == "fp4":
        w, ws = fp4.fp4_quantize((torch.randn(256, 512, device="cuda") / 20).to(BF16))
        x, g = torch.randn(70, 512, device="cuda").to(BF16), torch.randn(70, 256, device="cuda").to(BF16)

        def call(leaf):
            return fp4.fp4_linear(leaf, w, None, None, ws)
    else:
        freq, axes = (t.cuda() for t in rotary.axial_frequencies((16, 24, 24)))
        x, g = torch.randn(2, 35, 4, 64, device="cuda").to(BF16), torch.randn(2, 35, 4, 64, device="cuda").to(BF16)
        pos = torch.randint(0, 50, (2, 35, 3), device="cuda")

        def call(leaf):
            return rotary.apply_axial_rotary(leaf, None, pos, freq, axes)[0]

    def step():
        leaf = x.detach().requires_grad_(True)
        y = call(leaf)
        return y.detach(), torch.autograd.grad(y, [leaf], g)[0]

    return step, x, g


@pytest.mark.parametrize("kind", ["fp4", "axial"])
def test_captured_passes_in_turn(kind):
    """Two graphs with a pool in common, forward and backward pass in each, replayed in turn on other contents, beside eager passes."""
    (one, x1, _), (two, x2, _) = step_of(kind), step_of(kind)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        one(), two()
    torch.cuda.current_stream().wait_stream(s)
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        out1 = one()
    with torch.cuda.graph(second, pool=first.pool()):
        out2 = two()
    for _ in range(2):
        x1.copy_(torch.randn_like(x1))
        x2.copy_(torch.randn_like(x2))
        first.replay()
        got1 = [t.clone() for t in out1]
        second.replay()
        got2 = [t.clone() for t in out2]
        for got, step in ((got1, one), (got2, two)):
            assert all(torch.equal(bits(a), bits(b)) for a, b in zip(got, step()))


def test_two_streams_at_once():
    from q8_kernels_b200 import check_status
    block = Block(256, 4, "nvfp4")
    pos = grid(None, 4, 8, 8)
    xs = [torch.randn(2, 256, 256, device="cuda").to(BF16) for _ in range(2)]
    with torch.no_grad():
        alone = [block(x, pos) for x in xs]
        streams = [torch.cuda.Stream() for _ in xs]
        outs = [[], []]
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        for _ in range(20):
            for i, s in enumerate(streams):
                with torch.cuda.stream(s):
                    outs[i].append(block(xs[i], pos))
        torch.cuda.synchronize()
    for ref, out in zip(alone, outs):
        assert all(torch.equal(bits(y), bits(ref)) for y in out)
    check_status()


# ------------------------------------------------------------------------------------------ native calls and Python bodies

def calls():
    """(call, its leaves) of the differentiable ones."""
    from q8_kernels_b200.functional import fp4, head_norm, rotary
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(2, 30, 4, 64, generator=g, device="cuda").to(BF16)
    k = torch.randn(2, 30, 2, 64, generator=g, device="cuda").to(BF16)
    w = 1 + 0.1 * torch.randn(64, generator=g, device="cuda")
    freq, axes = (t.cuda() for t in rotary.axial_frequencies((16, 24, 24)))
    pos = torch.randint(0, 90, (2, 30, 3), generator=g, device="cuda")
    a = torch.randn(2, 30, 256, generator=g, device="cuda")
    w4, s4 = fp4.fp4_quantize((torch.randn(96, 256, generator=g, device="cuda") / 16).to(BF16))
    m4, t4 = fp4.fp4_quantize((torch.randn(96, 256, generator=g, device="cuda") / 16).to(BF16), "mxfp4")
    bias = torch.randn(96, generator=g, device="cuda")
    return [(lambda q, k: torch.cat(rotary.apply_axial_rotary(q, k, pos, freq, axes, 1.25), 2), (x, k)),
            (lambda q: rotary.apply_axial_rotary(q, None, pos[0].float() / 3, freq, axes, 1.0, "half")[0], (x.half(),)),
            (lambda q, k, w, v: torch.cat(head_norm.head_norm(q, k, w, v, 1e-6, pos, freq, axes), 2), (x, k, w, w + 0.5)),
            (lambda q, w: head_norm.head_norm(q, None, w, None, 1e-5, pos[0, :, 0], freq, layout="interleaved")[0], (x, w)),
            (lambda q: head_norm.head_norm(q)[0], (x.float(),)),
            (lambda a: fp4.fp4_linear(a, w4, bias, None, s4), (a.to(BF16),)),
            (lambda a: fp4.fp4_linear(a, m4, None, None, t4, out_dtype=F16), (a.to(BF16),))]


NAMES = ("_axial_rotary", "_head_norm", "_fp4_linear")


@pytest.mark.parametrize("i", range(7))
def test_native_and_python_body(i):
    from q8_kernels_b200 import _host
    call, tensors = calls()[i]
    seen = []

    def run(native):
        leaves = [t.clone().requires_grad_(True) for t in tensors]
        kept = {n: getattr(_host, n) for n in NAMES}
        for n in NAMES:
            def watch(*a, fn=kept[n]):
                out = fn(*a) if native else None
                seen.append(out is not None)
                return out
            setattr(_host, n, watch)
        try:
            y = call(*leaves)
            with torch.no_grad():
                plain = call(*leaves)
        finally:
            for n in NAMES:
                setattr(_host, n, kept[n])
        grad = torch.randn(y.shape, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(y.dtype)
        return y.detach(), plain, *torch.autograd.grad(y, leaves, grad)

    a, b = run(True), run(False)
    assert seen == [True, True, False, False]
    for p, q in zip(a, b):
        assert p.dtype == q.dtype and torch.equal(bits(p), bits(q))
    assert torch.equal(bits(a[0]), bits(a[1]))


@pytest.mark.parametrize("i", range(7))
def test_once_differentiable(i):
    call, tensors = calls()[i]
    leaves = [t.clone().requires_grad_(True) for t in tensors]
    y = call(*leaves)
    grads = torch.autograd.grad(y, leaves, torch.ones_like(y).requires_grad_(True), create_graph=True)
    assert all(torch.isfinite(d.float()).all() for d in grads)
    with pytest.raises(RuntimeError, match="twice|once"):
        grads[0].float().sum().backward()


@pytest.mark.parametrize("i", range(7))
@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("leaf", [False, True])
def test_tangents_are_refused(i, strided, leaf):
    from q8_kernels_b200 import Q8KernelError
    call, tensors = calls()[i]
    if strided:
        tensors = tuple(torch.stack([t, t], -1)[..., 0] if t.dim() > 1 else t for t in tensors)
    with fwd.dual_level():
        call(*tensors)
        for j, t in enumerate(tensors):
            t = t.clone().requires_grad_(True) if leaf else t
            with pytest.raises(Q8KernelError, match="forward-mode"):
                call(*tensors[:j], fwd.make_dual(t, torch.ones_like(t)), *tensors[j + 1:])
    call(*tensors)


def test_what_is_left_to_python():
    from q8_kernels_b200 import _host
    from q8_kernels_b200.functional import fp4, rotary
    x = torch.zeros(2, 6, 2, 64, device="cuda", dtype=BF16)
    pos = torch.zeros(6, 3, device="cuda")
    freq, axes = (t.cuda() for t in rotary.axial_frequencies((16, 24, 24)))
    w = torch.ones(64, device="cuda")
    axial, norm, linear = _host._axial_rotary, _host._head_norm, _host._fp4_linear
    assert axial(x, None, pos, freq, axes, 1.0, True) is not None and norm(x, None, w, None, 1e-6, pos, freq, axes, 1.0, True) is not None
    for a in ((x[..., ::2], None, pos, freq[:16], axes[:16], 1.0, True), (x, x.half(), pos, freq, axes, 1.0, True), (x, None, pos[:5], freq, axes, 1.0, True),
              (x, None, pos.half(), freq, axes, 1.0, True), (x, None, pos, freq.float(), axes, 1.0, True), (x, None, pos, freq, axes[:5], 1.0, True),
              (x, None, pos, freq, axes.long(), 1.0, True), (x.cpu(), None, pos, freq, axes, 1.0, True), (x, None, pos, freq, axes, 1, True)):
        assert axial(*a) is None
        assert norm(a[0], a[1], None, None, 1e-6, *a[2:]) is None
    assert norm(x, None, w[:32], None, 1e-6, None, None, None, 1.0, True) is None and norm(x, None, w.half(), None, 1e-6, None, None, None, 1.0, True) is None
    assert norm(x, None, w, None, -1.0, None, None, None, 1.0, True) is None and norm(x, None, w, None, 1e-6, pos, None, None, 1.0, True) is None
    a = torch.zeros(3, 64, device="cuda", dtype=BF16)
    q, (bs, rs) = fp4.fp4_quantize(torch.ones(32, 64, device="cuda", dtype=BF16))
    assert linear(a, q, None, bs, rs, False, None) is not None and linear(a, q, None, bs.view(torch.uint8), rs.view(torch.int32), False, None) is not None
    for args in ((a.float(), q, None, bs, rs, False, None), (a, q, None, bs, None, False, None), (a, q[:24], None, bs, rs[:24], False, None),
                 (a, q, rs[:16], bs, rs, False, None), (a, q, None, bs[:, :2], rs, False, None), (a, q, None, bs, rs, False, F32),
                 (a[:, :32], q, None, bs, rs, False, None), (a.cpu(), q, None, bs, rs, False, None)):
        assert linear(*args) is None
    assert linear(a.clone().requires_grad_(True), q, None, bs, rs, True, None) is None
    for fn, n in ((axial, 7), (norm, 10), (linear, 7)):
        for bad in (0, n - 1, n + 1):
            assert fn(*[None] * bad) is None


def test_gradient_of_many_output_channels_is_refused():
    from q8_kernels_b200 import Q8KernelError
    from q8_kernels_b200.functional.fp4 import fp4_linear, fp4_quantize
    w, ws = fp4_quantize(torch.ones(32784, 32, device="cuda", dtype=BF16))
    x = torch.ones(2, 32, device="cuda", dtype=BF16, requires_grad=True)
    with pytest.raises(Q8KernelError, match="32768"):
        fp4_linear(x, w, None, None, ws)
    with torch.no_grad():
        assert (fp4_linear(x, w, None, None, ws) == 32).all()


@pytest.mark.parametrize("m,n,k", [(1, 16, 32), (5, 48, 2048), (200, 1024, 512), (3000, 2064, 544)])
def test_fp8_products_in_fp16(m, n, k):
    """Products of e4m3 are exact in fp32; k of them add up with at most 2^-23 of their sizes for each addition of a block of 32."""
    from q8_kernels_b200 import check_status, native
    a, sa = native.tokenwise_quant(torch.randn(m, k, device="cuda").to(BF16), E4M3)
    b, sb = native.tokenwise_quant(torch.randn(n, k, device="cuda").to(BF16), E4M3)
    y = native.fp8_mm(a, b, sa, sb, False, F16)
    check_status()
    wa, wb = a.double() * sa.double().view(-1, 1), b.double() * sb.double().view(-1, 1)
    ref, slack = wa @ wb.T, (k // 32 + 8) * 2.0 ** -23 * (wa.abs() @ wb.abs().T)
    assert y.dtype == F16 and ((y.double() - ref).abs() <= slack + (ref.abs() + slack) * 2.0 ** -11 * 1.001 + 2.0 ** -24).all()


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_a_row_has_its_bits_in_every_call(fmt):
    """One row alone, in small tiles of any width and in tiles of pairs: each element is one accumulator's sum in ascending K."""
    from q8_kernels_b200 import check_status
    from q8_kernels_b200.functional.fp4 import fp4_linear, fp4_quantize
    w, ws = fp4_quantize((torch.randn(2080, 1056, device="cuda") / 32).to(BF16), fmt)
    x, bias = torch.randn(4000, 1056, device="cuda").to(BF16), torch.randn(2080, device="cuda")
    y = fp4_linear(x, w, bias, None, ws)
    for rows in ((0, 1), (130, 230), (700, 1000), (40, 1900)):
        assert torch.equal(bits(fp4_linear(x[rows[0]:rows[1]], w, bias, None, ws)), bits(y[rows[0]:rows[1]]))
    few, fews = fp4_quantize(torch.zeros(48, 1056, device="cuda", dtype=BF16), fmt)
    assert (fp4_linear(x, few, bias[:48].contiguous(), None, fews) == bias[:48].to(BF16)).all()
    check_status()


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("n,k", [(16, 32), (48, 96), (272, 2016), (2048, 2048), (9600, 544), (20480, 288), (64, 8192), (32, 8224)])
def test_few_rows(fmt, t, n, k):
    """Up to eight rows, which the product quantises itself where K and N allow: the bits of quantizer and product, rows that are not finite, tiny
    and zero rows among them."""
    from q8_kernels_b200 import check_status
    from q8_kernels_b200.functional.fp4 import fp4_linear, fp4_quantize
    w, ws = fp4_quantize((torch.randn(n, k, device="cuda") / 16).to(t), fmt)
    bias = torch.randn(n, device="cuda")
    x = torch.randn(9, k, device="cuda").to(t)
    x[2] *= 1e-3
    x[3] = 0
    x[4, k // 2] = float("nan")
    x[5, k - 1] = float("inf")
    x[6] = torch.finfo(t).tiny
    for m in range(1, 10):
        for gelu in (False, True):
            rows = x[9 - m:].contiguous()
            y = fp4_linear(rows, w, bias, None, ws, gelu)
            q, s = fp4_quantize(rows, fmt)
            ref = fp4_linear(q, w, bias, s, ws, gelu, t)
            assert torch.equal(torch.isnan(y), torch.isnan(ref)) and torch.equal(bits(y.nan_to_num()), bits(ref.nan_to_num()))
    check_status()


@pytest.mark.parametrize("m,n", [(1, 64), (40, 64), (3000, 2048)])
def test_a_launch_after_a_failed_one_stores_nothing(m, n):
    """On a status word that is not zero the output stays as it was, in every kernel of the products; the word stays, too."""
    from q8_kernels_b200 import _lib
    from q8_kernels_b200.functional.fp4 import fp4_quantize
    w, (wb, wr) = fp4_quantize(torch.randn(n, 256, device="cuda").to(BF16))
    x, out = torch.randn(m, 256, device="cuda").to(BF16), torch.full((m, n), 7.0, device="cuda", dtype=BF16)
    status = torch.tensor([257], dtype=torch.int32, device="cuda")
    work = torch.empty(max(1, _lib.lib.q8k_fp4_linear_workspace_bytes(2, m, n, 256)), dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream

    def call():
        rc = _lib.lib.q8k_fp4_linear(2, x.data_ptr(), _lib.DT_BF16, w.data_ptr(), wb.data_ptr(), wr.data_ptr(), None, out.data_ptr(), _lib.DT_BF16, m, n, 256, 0,
                                     work.data_ptr(), work.numel(), status.data_ptr(), stream)
        assert rc == 0, _lib.lib.q8k_last_error_detail()

    call()
    assert (out == 7).all() and status.item() == 257
    status.zero_()
    call()
    assert (out != 7).any() and status.item() == 0


@pytest.mark.parametrize("i", range(7))
def test_gradients_of_any_strides(i):
    """One number for all outputs, a gradient with its channels far apart, one that is a part of another, one at an odd address.

    The 4-bit linear's has the bits of the dense one.  The others' kernels come in forms by the width of their accesses, which round a c - b s and
    their sums in another order.  With G = max |g| and W = max |w| a rotation's sum has two terms of up to 1.25 G, so two forms differ by
    2 * 4 u * 2.5 G before they round to the output's type, each by half a step.  Norms: t has two terms of G, |u| <= 2 G W, normed values are
    at most 8 and their mean square is 1, so rstd u and x rstd^3 mean(u x) add up at most 9 * 2 G W rstd, over sums of 64: 2 * 80 u of that.
    dw adds up N terms of 2 G times normed values: 2 * (N + 80) u * 2 G * N."""
    call, tensors = calls()[i]
    leaves = [t.clone().requires_grad_(True) for t in tensors]

    def grads(g):
        return torch.autograd.grad(call(*leaves), leaves, g)

    y = call(*leaves)
    dense = torch.randn(y.shape, device="cuda").to(y.dtype)
    wide = torch.zeros(*y.shape[:-1], y.shape[-1] + 6, device="cuda", dtype=y.dtype)
    wide[..., 3:-3] = dense
    odd = torch.zeros(y.numel() + 1, device="cuda", dtype=y.dtype)[1:].view(y.shape).copy_(dense)
    one = torch.full((), 0.5, device="cuda", dtype=y.dtype)
    rstd = tensors[0].float().square().mean(-1).rsqrt().max().item() if i in (2, 3, 4) else 0.0
    u = 2.0 ** -24
    for g, same in ((one.expand(y.shape), one.expand(y.shape).contiguous()), (dense.transpose(-1, -2).contiguous().transpose(-1, -2), dense),
                    (wide[..., 3:-3], dense), (odd, dense)):
        top = same.float().abs().max().item()
        for a, b in zip(grads(g), grads(same)):
            if a.dim() == 1:
                n = tensors[0].numel() // 64
                slack, step = 2 * (n + 80) * u * 2 * top * n, 0.0
            else:
                weight = max((t.abs().max().item() for t in tensors if t.dim() == 1), default=1.0)
                slack = 20 * u * top if i < 2 else 2 * 80 * u * 18 * top * weight * rstd if i < 5 else 0.0
                step = torch.finfo(a.dtype).eps
            if i >= 5:
                assert torch.equal(bits(a), bits(b))
            else:
                assert ((a.double() - b.double()).abs() <= slack + step * (b.double().abs() + slack)).all(), (a.double() - b.double()).abs().max().item()


def test_tokens_captured():
    """A few rows in a graph, replayed on other contents, and two threads at once on streams of their own."""
    import threading
    from q8_kernels_b200.modules import FP4Linear
    m = FP4Linear.from_linear(torch.nn.Linear(1024, 2048, device="cuda", dtype=BF16), "nvfp4")
    x = torch.randn(3, 1024, device="cuda").to(BF16)
    with torch.no_grad():
        m(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m(x, fuse_gelu=True)
        x.copy_(torch.randn_like(x))
        graph.replay()
        assert torch.equal(bits(out), bits(m(x, fuse_gelu=True)))
        refs, got = [m(x * k) for k in (1, 2)], [[], []]
        torch.cuda.synchronize()

        def work(k):
            s = torch.cuda.Stream()
            with torch.no_grad(), torch.cuda.stream(s):
                for _ in range(200):
                    got[k].append(m(x * (k + 1)))
            s.synchronize()

        threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    for ref, outs in zip(refs, got):
        assert len(outs) == 200 and all(torch.equal(bits(y), bits(ref)) for y in outs)
