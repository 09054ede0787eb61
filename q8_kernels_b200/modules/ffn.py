"""FeedForward (reference: q8_kernels/modules/ffn.py:10-17)."""
import torch
import torch.nn as nn

from .activations import GELU, GatedLinear
from .linear import FP8Linear, Q8Linear, make_linear


class FeedForward(nn.Module):
    def __init__(self, dim: int, mult: int = 4, bias: bool = True, linear: str = "int8"):
        super().__init__()
        self.inner_dim = dim * mult
        self.act = GELU(dim, self.inner_dim, bias=bias, linear=linear)
        self.proj_down = make_linear(linear, self.inner_dim, dim, bias=bias)

    def forward(self, x, out_dtype=None):
        return self.proj_down(self.act(x, out_dtype=out_dtype), out_dtype=out_dtype)


class GatedFeedForward(nn.Module):
    """``proj_down(act(gate(x)) * up(x))``, gate and up projection, activation and product in one kernel.  ``inner_dim`` columns between the
    projections, a multiple of 16.  ``linear="int8"`` rotates both activations, so both widths have to be powers of two; "fp8" rotates
    the first if its width is one, and not the second, where FP8Linear has no gradient with a rotation.  Trains as its linears do: the
    activation has a gradient.  The output has x's leading dims, whatever they are (the linears alone return [1, M, N] for [M, K]).
    No counterpart in the reference."""

    def __init__(self, dim: int, inner_dim: int, act: str = "silu", bias: bool = True, linear: str = "int8"):
        super().__init__()
        self.inner_dim = inner_dim
        if linear == "int8" and (dim & (dim - 1) or inner_dim & (inner_dim - 1)):
            raise ValueError(f"int8 linears rotate their activations: {dim} and {inner_dim} have to be powers of two")
        self.gate_up = GatedLinear(dim, inner_dim, act, bias=bias, linear=linear, use_hadamard=dim & (dim - 1) == 0)
        self.proj_down = Q8Linear(inner_dim, dim, bias) if linear == "int8" else FP8Linear(inner_dim, dim, bias)

    def forward(self, x, out_dtype=torch.bfloat16):
        h = self.gate_up(x)
        dim = self.proj_down.out_features
        if h.numel() == 0 and h.requires_grad:               # the linears' backward pass does not take a tensor without rows
            return h[..., :1].expand(*h.shape[:-1], dim).to(h.dtype if out_dtype is None else out_dtype)
        if h.dim() not in (2, 3):
            h = h.reshape(-1, self.inner_dim)
        return self.proj_down(h, out_dtype=out_dtype).reshape(*x.shape[:-1], dim)

    @classmethod
    def from_linears(cls, gate: nn.Linear, up: nn.Linear, down: nn.Linear, act: str = "silu", linear: str = "int8"):
        """Quantises the three 16-bit projections of a checkpoint."""
        layer = cls(gate.in_features, gate.out_features, act, gate.bias is not None, linear)
        layer.gate_up = GatedLinear.from_linears(gate, up, act, linear, layer.gate_up.use_hadamard)
        layer.proj_down = Q8Linear.from_linear(down) if linear == "int8" else FP8Linear.from_linear(down)
        return layer
