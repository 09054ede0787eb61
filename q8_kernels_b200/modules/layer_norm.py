"""LayerNorm module beside RMSNorm (no counterpart in the reference)."""
import torch
import torch.nn as nn

from .. import functional as Q8F


class LayerNorm(nn.Module):
    """``weight`` and ``bias`` are fp32 and trainable; ``elementwise_affine=False`` has neither, ``bias=False`` no bias.  In a model that is
    cast to 16 bits they are rounded with it, and widened again in each call."""

    def __init__(self, dim: int, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True, device=None):
        super().__init__()
        self.dim = dim
        self.eps = eps
        for name, value in (("weight", torch.ones), ("bias", torch.zeros)):
            if elementwise_affine and (bias or name == "weight"):
                setattr(self, name, nn.Parameter(value(dim, dtype=torch.float, device=device)))
            else:
                self.register_parameter(name, None)

    def forward(self, x, out_dtype=None):
        weight, bias = self.weight, self.bias
        if weight is not None and weight.dtype != torch.float:
            weight = weight.float()
        if bias is not None and bias.dtype != torch.float:
            bias = bias.float()
        return Q8F.layer_norm.layer_norm(x, weight, bias, self.eps, out_dtype)
