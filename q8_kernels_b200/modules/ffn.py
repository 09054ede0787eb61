"""FeedForward (reference: q8_kernels/modules/ffn.py:10-17)."""
import torch
import torch.nn as nn

from .activations import GELU, GatedLinear
from .linear import make_linear


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
    projections, a multiple of 16.  Trains as its linears do: the activation has a gradient.  No counterpart in the reference."""

    def __init__(self, dim: int, inner_dim: int, act: str = "silu", bias: bool = True, linear: str = "int8"):
        super().__init__()
        self.inner_dim = inner_dim
        self.gate_up = GatedLinear(dim, inner_dim, act, bias=bias, linear=linear)
        self.proj_down = make_linear(linear, inner_dim, dim, bias=bias)

    def forward(self, x, out_dtype=torch.bfloat16):
        return self.proj_down(self.gate_up(x), out_dtype=out_dtype)
