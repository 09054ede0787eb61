"""Layer norm with the gradients of input, weight and bias (no counterpart in the reference, whose blocks have RMS norm only)."""
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from .. import _host
from ..native import E4M3, layer_norm_backward, refuse_tangents
from ..native import layer_norm as _layer_norm


class LayerNormFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, out_type):
        y, mean, rstd = _layer_norm(x, weight, bias, eps, out_type, True)
        ctx.save_for_backward(x, mean, rstd, weight)
        ctx.has_bias = bias is not None
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, mean, rstd, weight = ctx.saved_tensors
        need = ctx.needs_input_grad
        if grad.dtype == E4M3:
            grad = grad.to(torch.bfloat16)                   # exact
        dx, dw, db = layer_norm_backward(x, mean, rstd, grad, weight, need[0], need[1], need[2] and ctx.has_bias)
        return dx, dw, db, None, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
               out_type: Optional[torch.dtype] = None) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dim of x (bf16, fp16 or fp32; any leading dims and strides), with fp32
    ``weight`` and ``bias`` of that dim, at most 16384.  ``out_type``: x's type (default), e4m3 for bf16, or bf16 / fp16 for fp32.
    Statistics and sums are fp32; the gradients of weight and bias are fp32 and have the same bits in every run."""
    fast = _host._layer_norm(x, weight, bias, eps, out_type)
    if fast is not None:
        return fast
    refuse_tangents("layer_norm", x, weight, bias)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return LayerNormFunc.apply(x, weight, bias, eps, out_type)
    return _layer_norm(x, weight, bias, eps, out_type, False)[0]
