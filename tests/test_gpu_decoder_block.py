"""Layer norm, rotary positions and the gated feed-forward together with the package's linears and attention: a pre-norm block of 64-wide
heads as an encoder or decoder has it, forward and backward."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


class Block(torch.nn.Module):
    def __init__(self, dim=512, inner=1024, linear="int8"):
        super().__init__()
        from q8_kernels_b200.modules import GatedFeedForward, LayerNorm, RotaryEmbedding
        from q8_kernels_b200.modules.linear import make_linear
        self.heads = dim // 64
        self.norm1, self.norm2 = LayerNorm(dim), LayerNorm(dim)
        self.qkv, self.out = make_linear(linear, dim, 3 * dim), make_linear(linear, dim, dim)
        self.rotary = RotaryEmbedding(64, 32, scaling={"type": "yarn", "factor": 8.0, "original_length": 128})
        self.ff = GatedFeedForward(dim, inner, "silu", linear=linear)

    def forward(self, x, positions, lens=None):
        from q8_kernels_b200.functional.flash_attention import flash_attn_func
        b, s, d = x.shape
        q, k, v = self.qkv(self.norm1(x), out_dtype=BF16).view(b, s, 3, self.heads, 64).unbind(2)
        q, k = self.rotary(q, k, positions)
        o = flash_attn_func(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), batch_mask=lens, apply_qk_hadamard=True, out_dtype=BF16,
                            token_major_out=True)
        x = x + self.out(o.transpose(1, 2).reshape(b, s, d), out_dtype=BF16).view(b, s, d)
        return x + self.ff(self.norm2(x)).view(b, s, d)


def filled(block, seed=0):
    """Weights N(0, 1 / fan-in) on their 8-bit grids; also those weights in 64 bits, un-rotated."""
    from q8_kernels_b200 import native
    g = torch.Generator(device="cuda").manual_seed(seed)
    block.cuda()
    wide = {}
    for name, m in block.named_modules():
        if hasattr(m, "scales"):
            n, k = m.weight.shape
            w = (torch.randn(n, k, generator=g, device="cuda") * k ** -0.5).to(BF16)
            p = k if getattr(m, "use_hadamard", True) else 0     # a rotated weight, or as it is
            m.weight.data, m.scales.data = native.hadamard_quant(w, k ** -0.5, m.weight.dtype) if p else native.tokenwise_quant(w, m.weight.dtype)
            m.bias.data = 0.1 * torch.randn(n, generator=g, device="cuda")
            wide[name] = (m.weight.double() * m.scales.double().unsqueeze(1), m.bias.double(), p)
    for m in (block.norm1, block.norm2):
        m.weight.data = 1 + 0.1 * torch.randn(m.dim, generator=g, device="cuda")
        m.bias.data = 0.1 * torch.randn(m.dim, generator=g, device="cuda")
    return wide


def rotated(x, p):
    if not p:
        return x
    d = x.shape[-1]
    h = torch.ones(1, 1, dtype=torch.float64, device=x.device)
    while h.shape[0] < p:
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    return x @ h[:d, :d] * d ** -0.5


def plain(block, wide, x, positions, lens):
    """The block's formulas in 64 bits, with the 8-bit weights but no other rounding."""
    def lin(name, t):
        w, b, p = wide[name]
        return rotated(t, p) @ w.T + b

    def norm(m, t):
        return torch.nn.functional.layer_norm(t, (m.dim,), m.weight.double(), m.bias.double(), m.eps)

    b, s, d = x.shape
    q, k, v = lin("qkv", norm(block.norm1, x)).view(b, s, 3, block.heads, 64).unbind(2)
    angle = (positions.double().unsqueeze(-1) * block.rotary.frequencies).unsqueeze(2)
    c, n = angle.cos() * block.rotary.amplitude, angle.sin() * block.rotary.amplitude

    def turn(t):
        return torch.cat([t[..., :16] * c - t[..., 16:32] * n, t[..., 16:32] * c + t[..., :16] * n, t[..., 32:]], -1)

    scores = torch.einsum("bqhd,bkhd->bhqk", turn(q), turn(k)) / 8
    mask = torch.arange(s, device="cuda") >= lens.view(b, 1, 1, 1)
    o = torch.einsum("bhqk,bkhd->bqhd", torch.softmax(scores.masked_fill(mask, float("-inf")), -1), v).reshape(b, s, d)
    x = x + lin("out", o)
    gate, up = lin("ff.gate_up", norm(block.norm2, x)).chunk(2, -1)
    return x + lin("ff.proj_down", torch.nn.functional.silu(gate) * up)


@pytest.mark.parametrize("linear", ["int8", "fp8"])
def test_block(linear):
    """Rounding errors of a normalised row, each relative to its tensor: int8 rows of rotated, i.e. normal, values have steps of 4 sigma / 127,
    1 % rms; e4m3 rows at most 2^-4, 2.6 % rms; q, k, v and the probabilities e4m3.  Eight of them one after the other, added up
    as squares, in a sum with the residual: 8 % with e4m3 everywhere."""
    block = Block(inner=1024 if linear == "int8" else 1360, linear=linear)
    wide = filled(block)
    x = torch.randn(2, 77, 512, device="cuda").to(BF16)
    positions = torch.stack([torch.arange(77, device="cuda"), torch.arange(77, device="cuda") + 900])
    lens = torch.tensor([77, 40], device="cuda", dtype=torch.int32)
    with torch.no_grad():
        y = block(x, positions, lens)
        ref = plain(block, wide, x.double(), positions, lens)
    assert ((y.double() - ref).norm() / ref.norm()).item() <= 0.08
    # captured and replayed with other contents
    with torch.no_grad():
        from q8_kernels_b200 import check_status
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = block(x, positions, lens)
        x.copy_(torch.randn_like(x))
        positions += 5
        lens.fill_(11)
        graph.replay()
        assert torch.equal(out.view(torch.int16), block(x, positions, lens).view(torch.int16))
        check_status()


def test_feed_forward_gradients():
    """x + ff(norm(x)): gradients of x and of the norm's weight and bias against those of the formulas in 64 bits.  The gradient passes
    two products whose operands are e4m3 (2.6 % rms each: 5 % for four), and the forward's activations int8 grids (1 %)."""
    block = Block()
    wide = filled(block, 3)
    x = torch.randn(3, 50, 512, device="cuda").to(BF16).requires_grad_(True)
    g = torch.randn(3, 50, 512, device="cuda").to(BF16)
    leaves = [x, block.norm2.weight, block.norm2.bias]
    y = x + block.ff(block.norm2(x)).view_as(x)
    got = torch.autograd.grad(y, leaves, g)
    xd, w, b = (t.detach().double().requires_grad_(True) for t in leaves)

    def lin(name, t):
        ww, bb, p = wide[name]
        return rotated(t, p) @ ww.T + bb

    gate, up = lin("ff.gate_up", torch.nn.functional.layer_norm(xd, (512,), w, b, 1e-5)).chunk(2, -1)
    ref = torch.autograd.grad(xd + lin("ff.proj_down", torch.nn.functional.silu(gate) * up), [xd, w, b], g.double())
    for a, r in zip(got, ref):
        assert ((a.double() - r).norm() / r.norm()).item() <= 0.1
