"""4-bit values with block scales: the quantizer bit by bit against its definition, products against those in 64 bits.

Tolerances.  The quantizer's scales and values are defined operation by operation in fp32: no tolerance.  Products: values and scales are exact
in the tensor core, whose fp32 sum of K products is off by at most K u of the sum of their sizes (u = 2^-23 where it truncates); it adds
blocks of 64 at a time, so K / 64 + 8 additions count.  Scaling, bias and GELU add a few fp32 roundings, and the output's type half a
step (`torch.finfo(t).eps / 2`).  The tanh of the fused GELU is good to 2^-10.9 (absolute), that is |y| 2^-11.9 of the output.
"""
import pytest
import torch

from helpers import bits

pytestmark = pytest.mark.gpu
BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
BLOCK = {"mxfp4": 32, "nvfp4": 16}
FORMATS = ["mxfp4", "nvfp4"]
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def unpacked(values):
    """uint8 [rows, K/2] -> the 4-bit values in 64 bits."""
    codes = torch.stack([values & 15, values >> 4], -1).flatten(-2).long()
    v = GRID.to(values.device).double()[codes & 7]
    return torch.where(codes >= 8, -v, v)


def scale_table(block, rows, k, fmt):
    """The tiles of block scales as [rows, K / block] bytes."""
    b = block.view(torch.uint8)
    t = b.view(b.shape[0], b.shape[1], 32, 4, 4)                # [row tile, tile, r % 32, r / 32, block]
    return t.permute(0, 3, 2, 1, 4).reshape(b.shape[0] * 128, -1)[:rows, :k // BLOCK[fmt]]


def wide(values, block, row, fmt):
    """What they stand for, in 64 bits."""
    rows, k = values.shape[0], 2 * values.shape[1]
    s = scale_table(block, rows, k, fmt)
    s = s.contiguous().view(E4M3).double() if fmt == "nvfp4" else torch.where(s == 255, torch.nan, torch.exp2(s.double() - 127))
    v = unpacked(values) * s.repeat_interleave(BLOCK[fmt], 1)
    return v if row is None else v * row.double().unsqueeze(1)


def nearest(y):
    """Codes of the 4-bit values nearest to y (64 bits), halves to the even code."""
    away = (y.abs().unsqueeze(-1) - GRID.to(y.device).double()).abs()
    even_first = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7], device=y.device)
    code = even_first[away[..., even_first].argmin(-1)]
    return code | ((torch.signbit(y)).long() << 3)


def definition(x, fmt):
    """Codes [rows, K], scale bytes [rows, K / block] and row scales by the definition, each fp32 operation rounded on its own."""
    x = x.float().cpu()
    rows, k = x.shape
    v = x.view(rows, -1, BLOCK[fmt])
    a = v.abs().amax(2)
    if fmt == "mxfp4":
        e = ((a.view(torch.int32) >> 23) - 2).clamp(min=0)
        e = torch.where(torch.isfinite(a), e, torch.full_like(e, 255))
        y = v.double() / torch.exp2(e.double() - 127).unsqueeze(2)
        return nearest(y).view(rows, k), e.to(torch.uint8), None
    top = a.amax(1, keepdim=True)
    big = torch.finfo(F32).max
    r = top / torch.full_like(top, 2688.0)
    s = (a * torch.where(top > 0, (torch.full_like(top, 448.0) / top).clamp(max=big), torch.zeros_like(top))).to(E4M3)
    unit = s.float() * r
    f = torch.where(s.float() > 0, (torch.ones_like(unit) / unit).clamp(max=big), torch.zeros_like(unit))
    s = s.view(torch.uint8)
    s = torch.where(s & 127 == 127, torch.full_like(s, 127), s)                     # NaN has no sign
    return nearest((v * f.unsqueeze(2)).double()).view(rows, k), s, r.view(rows)


def sample(rows, k, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=g) * torch.exp(2 * torch.randn(rows, 1, generator=g))
    x *= torch.exp(torch.randn(rows, k // 16, generator=g)).repeat_interleave(16, 1)
    return x.to(dtype)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,k", [(1, 32), (3, 64), (5, 96), (1, 2048), (7, 2016), (130, 288), (129, 4096), (3, 8192), (2, 10240), (257, 512), (1, 65536), (1100, 2048), (1025, 4096), (1030, 20000),
                                    (1024, 34016), (4097, 32), (4100, 512), (4222, 544), (4130, 1120), (4096, 1536), (4127, 2048)])
def test_quantizer_bits(fmt, dtype, rows, k):
    from q8_kernels_b200 import native
    x = sample(rows, k, dtype, rows + k)
    if rows > 2:
        x[1] = 0
        x[2, :k // 2] = 0
        x[0, :8] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -6.0])      # the ties of a block with scale 1
    codes, scales, r = definition(x, fmt)
    values, block, row = native.fp4_quant(x.cuda(), fmt)
    got = torch.stack([values & 15, values >> 4], -1).flatten(-2).cpu().long()
    same = (got == codes) | ((got & 7 == 0) & (codes & 7 == 0))                    # the sign of a zero stands for nothing
    assert torch.equal(scale_table(block, rows, k, fmt).cpu(), scales)
    # (values beyond fp16 are infinite: nothing is said of the values of a block whose scale is NaN)
    same |= (scales == (255 if fmt == "mxfp4" else 127)).repeat_interleave(BLOCK[fmt], 1)
    assert same.all(), int((~same).sum())
    assert (row is None) if fmt == "mxfp4" else torch.equal(bits(row.cpu()), bits(r))
    # the scales that fill up a tile are zero
    full = block.view(torch.uint8).view(*block.shape[:2], 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(block.shape[0] * 128, -1)
    assert not full[rows:].any() and not full[:, k // BLOCK[fmt]:].any()
    for t in (BF16, F16, F32):
        y = native.fp4_dequant(values, block, row, t)
        ref = wide(values, block, None, fmt).float()
        ref = ref if row is None else ref * row.unsqueeze(1)
        assert y.dtype == t and ((bits(y) == bits(ref.to(t))) | (torch.isnan(y) & torch.isnan(ref))).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("gelu,bias,out", [(False, True, BF16), (True, True, F16), (False, False, F16), (True, False, BF16)])
@pytest.mark.parametrize("m,n,k", [(1, 16, 32), (3, 48, 96), (8, 128, 256), (77, 272, 2048), (128, 96, 64), (129, 2048, 544), (300, 560, 1024), (1, 8192, 2048),
                                   (16, 4096, 4096), (1000, 1408, 512), (2002, 5504, 288), (700, 4096, 8192), (3000, 256, 512), (60000, 512, 64),
                                   (20100, 528, 2048), (1300, 2064, 2080), (1, 20480, 544), (100, 18960, 96), (129, 10256, 160),
                                   (19000, 16, 288), (200, 4144, 1056)])
def test_products(fmt, gelu, bias, out, m, n, k):
    from q8_kernels_b200 import check_status, native
    a, b = sample(m, k, BF16, 1).cuda(), sample(n, k, BF16, 2).cuda()
    qa, qb = native.fp4_quant(a, fmt), native.fp4_quant(b, fmt)
    c = torch.randn(n, device="cuda") if bias else None
    y = native.fp4_mm(qa[0], qb[0], c, qa[1:], qb[1:], gelu, out)
    check_status()
    assert y.dtype == out and y.shape == (m, n)
    wa, wb = wide(*qa, fmt), wide(*qb, fmt)
    ref = wa @ wb.T
    size = wa.abs() @ wb.abs().T
    slack = (k // 64 + 8) * 2.0 ** -23 * size
    if bias:
        ref, slack = ref + c.double(), slack + 2.0 ** -22 * c.double().abs()
    if gelu:
        slack = 1.13 * slack + 2.0 ** -11.9 * ref.abs() + 2.0 ** -22 * ref.abs()    # |gelu'| < 1.13
        ref = torch.nn.functional.gelu(ref, approximate="tanh")
    f = torch.finfo(out)
    ref = ref.clamp(-2 * f.max, 2 * f.max)
    bad = (y.double() - ref).abs() > slack + (ref.abs() + slack) * f.eps / 2 * 1.001 + f.tiny * f.eps
    bad &= ~(torch.isinf(y) & (ref.abs() >= f.max) & (torch.signbit(y) == torch.signbit(ref)))
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {((y.double() - ref).abs() / size.clamp(min=1e-30)).max().item()}"


# ------------------------------------------------------------------------------------------ the linear

def rows_e4m3(x):
    """Rows of fp32 values as e4m3 with the factor 448 / absmax, and 1 / factor."""
    amax = x.abs().amax(1, keepdim=True)
    f = torch.full_like(amax, 448.0) / amax
    return (x * torch.where(amax > 0, f, torch.zeros_like(f))).to(E4M3), torch.ones_like(f) / f


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("n,k", [(16, 32), (48, 96), (272, 2048), (2048, 544), (5504, 288), (1408, 4096)])
def test_weight_operand(fmt, n, k):
    """Bit by bit: value * block scale * row scale in fp32, the column's factor 448 / absmax, rounded to e4m3."""
    from q8_kernels_b200 import native
    w = sample(n, k, BF16, 3)
    w[:, 5] = 0
    q = native.fp4_quant(w.cuda(), fmt)
    got, scales = native.fp4_weight_operand(q[0], q[1:])
    full = wide(*q[:2], None, fmt).float()
    full = full if q[2] is None else full * q[2].unsqueeze(1)
    ref, rs = rows_e4m3(full.T.contiguous().cpu())
    assert got.shape == (k, n) and torch.equal(got.cpu().view(torch.uint8) & 127, ref.view(torch.uint8) & 127)
    assert torch.equal(got.cpu().float(), ref.float()) and torch.equal(bits(scales.cpu()), bits(rs[:, 0]))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("shape,n", [((5, 96), 48), ((2, 31, 512), 272), ((1, 2048), 2048), ((3, 1, 7, 64), 16), ((700, 1024), 1408)])
def test_linear_and_gradient(fmt, t, shape, n):
    from q8_kernels_b200 import check_status, native
    from q8_kernels_b200.functional.fp4 import fp4_linear, fp4_quantize
    k = shape[-1]
    x = sample(torch.Size(shape[:-1]).numel(), k, t, 4).cuda().clamp(-1e3, 1e3).view(shape).requires_grad_(True)
    w, ws = fp4_quantize((sample(n, k, BF16, 5) * 0.02).to(t).cuda(), fmt)
    bias = torch.randn(n, device="cuda")
    y = fp4_linear(x, w, bias, None, ws)
    with torch.no_grad():
        assert torch.equal(bits(fp4_linear(x, w, bias, None, ws)), bits(y))
    assert y.dtype == t and y.shape == shape[:-1] + (n,)
    qx = fp4_quantize(x, fmt)
    assert torch.equal(bits(fp4_linear(qx[0], w, bias, qx[1], ws, out_dtype=t)), bits(y))
    # the gradient: e4m3 rows of the output's gradient times the e4m3 weight operand.  Values are products of e4m3 values, exact in fp32; the
    # sum of n adds up in fp32 (n / 32 + 8 additions of blocks, 2^-23 each), two scale products, one rounding
    g = torch.randn(y.shape, device="cuda").to(t)
    dx, = torch.autograd.grad(y, [x], g)
    check_status()
    g8, gs = rows_e4m3(g.reshape(-1, n).float())
    w8, wsc = native.fp4_weight_operand(w, ws)
    a, b = g8.double() * gs.double(), w8.double() * wsc.double().unsqueeze(1)
    ref, size = a @ b.T, a.abs() @ b.abs().T
    f = torch.finfo(t)
    assert dx.dtype == t and dx.shape == x.shape
    slack = (n // 32 + 12) * 2.0 ** -23 * size
    bad = (dx.reshape(-1, k).double() - ref).abs() > slack + (ref.abs() + slack) * f.eps / 2 * 1.001 + f.tiny * f.eps
    assert not bad.any(), int(bad.sum())
    # and against the de-quantised weight in 64 bits, by differences along v: e4m3 values on both sides are off by at most 2^-4 of themselves
    # (independent: the error of the sum is a random walk, 8 times its size)
    wide_w = wide(w, ws[0].view(torch.uint8) if fmt == "mxfp4" else ws[0], ws[1], fmt)
    v = torch.randn(shape, device="cuda", dtype=F64)
    left = (g.double().reshape(-1, n) * (v.reshape(-1, k) @ wide_w.T)).sum()
    terms = (g.double().reshape(-1, n).square() @ (wide_w.square())) * v.reshape(-1, k).square()
    assert abs(left - (dx.double() * v).sum()) <= 8 * 2.0 ** -3 * terms.sum().sqrt() + f.eps * (ref.abs() * v.reshape(-1, k).abs()).sum()


def test_linear_with_gelu_and_gradient():
    """With a gradient the GELU is a kernel on the product rounded to bf16: the output is gelu(bf16(product)), the gradient passes gelu'."""
    from q8_kernels_b200 import native
    from q8_kernels_b200.functional.fp4 import fp4_linear, fp4_quantize
    for t in (BF16, F16):
        x = torch.randn(40, 512, device="cuda").to(t).requires_grad_(True)
        w, ws = fp4_quantize((torch.randn(256, 512, device="cuda") * 0.05).to(t))
        bias = torch.randn(256, device="cuda")
        y = fp4_linear(x, w, bias, None, ws, True)
        pre = fp4_linear(x.detach(), w, bias, None, ws, out_dtype=BF16)
        assert torch.equal(bits(y), bits(native.gelu_forward(pre, BF16).to(t)))
        g = torch.randn(40, 256, device="cuda").to(t)
        dx, = torch.autograd.grad(y, [x], g)
        x2 = x.detach().requires_grad_(True)
        ref, = torch.autograd.grad(fp4_linear(x2, w, bias, None, ws), [x2], native.gelu_backward(pre, g.to(BF16), BF16).to(t))
        assert dx.dtype == t and ((dx.float() - ref.float()).norm() <= 2.0 ** -7 * ref.float().norm())


@pytest.mark.parametrize("fmt", FORMATS)
def test_rows_that_are_not_finite_and_tiny_ones(fmt):
    """NaN and infinities spoil their own row's products and no other row's; rows of zeros give the bias; rows down to the smallest values of
    the type give no NaN."""
    from q8_kernels_b200.functional.fp4 import fp4_linear, fp4_quantize
    w, ws = fp4_quantize(torch.randn(160, 512, device="cuda").to(BF16), fmt)
    bias = torch.randn(160, device="cuda")
    for m in (12, 300):
        x = torch.randn(m, 512, device="cuda").to(BF16)
        x[1, 7], x[3, 500], x[4, 0] = float("nan"), float("inf"), -float("inf")
        x[6] = 0
        x[7] = 9.2e-41
        x[8] = 1e-37
        x[8, 3] = 1e-30
        x[9] = 3e38
        y = fp4_linear(x, w, bias, None, ws)
        bad = torch.isnan(y).any(1)
        assert torch.isnan(y[[1, 3, 4]]).all() and bad.nonzero().flatten().tolist() == [1, 3, 4]
        assert torch.equal(y[6], bias.to(BF16)) and torch.equal(y[7], bias.to(BF16))
        clean = x.clone()
        clean[[1, 3, 4]] = 0
        rest = [i for i in range(m) if i not in (1, 3, 4)]
        assert torch.equal(bits(fp4_linear(clean, w, bias, None, ws)[rest]), bits(y[rest]))
    # a NaN in the weight spoils its output channel
    wn = torch.randn(160, 512, device="cuda").to(BF16)
    wn[17, 100] = float("nan")
    w, ws = fp4_quantize(wn, fmt)
    y = fp4_linear(torch.randn(5, 512, device="cuda").to(BF16), w, bias, None, ws)
    assert torch.isnan(y).all(0).nonzero().flatten().tolist() == [17] and int(torch.isnan(y).sum()) == 5


def test_strided_offset_and_empty_inputs():
    from q8_kernels_b200.functional.fp4 import fp4_dequantize, fp4_linear, fp4_quantize
    w, ws = fp4_quantize(torch.randn(64, 128, device="cuda").to(BF16))
    x = torch.randn(9, 128, device="cuda").to(BF16)
    y = fp4_linear(x, w, None, None, ws)
    off = torch.zeros(9 * 128 + 1, device="cuda", dtype=BF16)[1:].view(9, 128).copy_(x)
    wide_rows = torch.zeros(9, 300, device="cuda", dtype=BF16)
    wide_rows[:, 3:131] = x
    for other in (off, wide_rows[:, 3:131], x.T.contiguous().T, torch.stack([x, x], 1)[:, 0]):
        assert torch.equal(bits(fp4_linear(other, w, None, None, ws)), bits(y))
        q, s = fp4_quantize(other)
        assert torch.equal(bits(fp4_linear(q, w, None, s, ws)), bits(y))
    for shape in ((0, 128), (2, 0, 128)):
        e = torch.zeros(shape, device="cuda", dtype=BF16, requires_grad=True)
        out = fp4_linear(e, w, None, None, ws)
        assert out.shape == shape[:-1] + (64,) and torch.autograd.grad(out.sum(), [e])[0].shape == shape
        q, s = fp4_quantize(e)
        assert fp4_dequantize(q, s).shape == shape and fp4_linear(q, w, None, s, ws).shape == out.shape


def test_module_checkpoint_cast_capture_and_streams():
    from q8_kernels_b200 import check_status
    from q8_kernels_b200.modules import FP4Linear
    for fmt in FORMATS:
        full = torch.nn.Linear(512, 208, device="cuda", dtype=BF16)
        m = FP4Linear.from_linear(full, fmt)
        x = torch.randn(3, 50, 512, device="cuda").to(BF16)
        y = m(x)
        assert y.shape == (3, 50, 208) and not any(p.requires_grad for p in m.parameters())
        # 4-bit steps of the values on both sides: at most a sixth, 10 % rms of an element in its block
        ref = full(x)
        assert ((y - ref).float().norm() / ref.float().norm()).item() < 0.2
        other = FP4Linear(512, 208, format=fmt).cuda()
        other.load_state_dict(m.state_dict())
        assert torch.equal(bits(other(x)), bits(y))
        assert torch.equal(bits(FP4Linear.from_linear(full, fmt).to(F16).to(BF16)(x.float().to(BF16))), bits(y)) or m.bias is not None
        cast = FP4Linear.from_linear(torch.nn.Linear(512, 208, bias=False, device="cuda", dtype=BF16), fmt)
        before = cast(x)
        assert torch.equal(bits(cast.to(torch.float64).to(F16)(x)), bits(before))     # a cast of the model leaves the scales alone
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            on_other = m(x)
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(bits(on_other), bits(y))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m(x, fuse_gelu=True)
        x.copy_(torch.randn_like(x))
        graph.replay()
        assert torch.equal(bits(out), bits(m(x, fuse_gelu=True)))
    check_status()


def test_refusals():
    from q8_kernels_b200 import Q8KernelError, native
    from q8_kernels_b200.functional.fp4 import fp4_dequantize, fp4_linear, fp4_quantize
    from q8_kernels_b200.modules import FP4Linear
    x = torch.randn(6, 128, device="cuda").to(BF16)
    w, ws = fp4_quantize(torch.randn(64, 128, device="cuda").to(BF16))
    wm, wms = fp4_quantize(torch.randn(64, 128, device="cuda").to(BF16), "mxfp4")
    odd, odds = fp4_quantize(torch.randn(24, 128, device="cuda").to(BF16))
    for bad in (lambda: fp4_quantize(x[:, :80]), lambda: fp4_quantize(x.float()), lambda: fp4_quantize(x, "fp4"), lambda: fp4_quantize(x.cpu()),
                lambda: fp4_quantize(x[:, :0]), lambda: fp4_dequantize(w, ws, torch.int8), lambda: fp4_dequantize(w, (ws[0], None)),
                lambda: fp4_dequantize(wm, (wms[0], ws[1])), lambda: fp4_dequantize(w[:32], ws), lambda: fp4_dequantize(w, (ws[0], ws[1].half())),
                lambda: fp4_linear(x, w), lambda: fp4_linear(x, w, None, None, ws[0]), lambda: fp4_linear(x[:, :64], w, None, None, ws),
                lambda: fp4_linear(x.float(), w, None, None, ws), lambda: fp4_linear(x, w, torch.zeros(63, device="cuda"), None, ws),
                lambda: fp4_linear(x, w, torch.zeros(64, device="cuda", dtype=BF16), None, ws), lambda: fp4_linear(x, odd, None, None, odds),
                lambda: fp4_linear(x, w, None, None, ws, out_dtype=torch.float32), lambda: fp4_linear(x, w.cpu(), None, None, ws),
                lambda: fp4_linear(*fp4_quantize(x, "mxfp4")[:1], w, None, fp4_quantize(x, "mxfp4")[1], ws), lambda: fp4_linear(x, w[0], None, None, ws),
                lambda: native.fp4_weight_operand(odd, odds), lambda: FP4Linear(128, 24), lambda: FP4Linear(100, 32), lambda: FP4Linear(128, 32, format="e2m1"),
                lambda: FP4Linear.from_linear(torch.nn.Linear(128, 32, device="cuda"))):
        with pytest.raises(Q8KernelError):
            bad()
