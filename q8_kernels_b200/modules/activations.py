"""GELU projection (reference: q8_kernels/modules/activations.py:9-16): a
quantised linear whose GEMM epilogue applies tanh-GELU (``linear="fp8"`` builds it
from FP8Linear instead of Q8Linear)."""
import torch
import torch.nn as nn

from .. import functional as Q8F
from .linear import FP8Linear, Q8Linear, make_linear


class GELU(nn.Module):
    def __init__(self, dim_in: int, dim_out: int, approximate: str = "none", bias: bool = True, linear: str = "int8"):
        super().__init__()
        self.proj = make_linear(linear, dim_in, dim_out, bias=bias)

    def forward(self, hidden_states, out_dtype=None):
        return self.proj(hidden_states, fuse_gelu=True, out_dtype=out_dtype)


class GatedLinear(nn.Module):
    """``act(gate(x)) * up(x)`` from one 8-bit weight [2 * dim_out, dim_in], the gate's rows first: parameters and state-dict keys of a
    Q8Linear / FP8Linear of that size.  ``linear``: "int8", or "fp8" with ``use_hadamard`` as in FP8Linear.  No counterpart in the reference."""

    def __init__(self, dim_in: int, dim_out: int, act: str = "silu", bias: bool = True, linear: str = "int8", use_hadamard: bool = True,
                 device=None):
        super().__init__()
        if act not in ("silu", "gelu_tanh"):
            raise ValueError(f"activation {act!r} is not 'silu' or 'gelu_tanh'")
        if linear not in ("int8", "fp8"):
            raise ValueError(f"linear kind {linear!r} is not 'int8' or 'fp8'")
        self.dim_in, self.dim_out, self.act, self.linear, self.use_hadamard = dim_in, dim_out, act, linear, use_hadamard
        dtype = torch.int8 if linear == "int8" else torch.float8_e4m3fn
        self.weight = nn.Parameter(torch.empty(2 * dim_out, dim_in, device=device, dtype=dtype), requires_grad=False)
        if bias:
            self.bias = nn.Parameter(torch.empty(2 * dim_out, device=device, dtype=torch.float), requires_grad=False)
        else:
            self.register_parameter("bias", None)
        self.register_buffer("scales", torch.empty(2 * dim_out, device=device, dtype=torch.float))

    def forward(self, x, x_scales=None):
        bias = self.bias.data if self.bias is not None else None
        if self.linear == "int8":
            return Q8F.gated.q8_gated_linear(x, self.weight.data, bias, x_scales, self.scales, self.act)
        return Q8F.gated.fp8_gated_linear(x, self.weight.data, bias, x_scales, self.scales, self.act, self.use_hadamard)

    @classmethod
    def from_linears(cls, gate: nn.Linear, up: nn.Linear, act: str = "silu", linear: str = "int8", use_hadamard: bool = True):
        """Quantises the two 16-bit projections of a checkpoint, as Q8Linear / FP8Linear.from_linear do.  With the rotation (int8 always)
        their input must have a power of two of channels: only that many the Hadamard matrix leaves the products as they are."""
        if (linear == "int8" or use_hadamard) and gate.in_features & (gate.in_features - 1):
            raise ValueError(f"{gate.in_features} input channels are no power of two, which the rotation needs: use linear='fp8' with "
                             "use_hadamard=False")
        if gate.weight.shape != up.weight.shape or (gate.bias is None) != (up.bias is None):
            raise ValueError("the gate and the up projection must have the same shape and both a bias or none")
        layer = cls(gate.in_features, gate.out_features, act, gate.bias is not None, linear, use_hadamard, gate.weight.device)
        halves = [Q8Linear.from_linear(m) if linear == "int8" else FP8Linear.from_linear(m, use_hadamard=use_hadamard) for m in (gate, up)]
        for name in ("weight", "scales", "bias"):
            if getattr(layer, name) is not None:
                getattr(layer, name).data = torch.cat([getattr(h, name).data for h in halves], dim=0)
        return layer
