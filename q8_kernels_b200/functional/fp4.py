"""Linear layers on microscaled 4-bit values (no counterpart in the reference, whose linears are 8-bit).

Values are e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) in blocks along a row that share a scale:

* ``"mxfp4"``  blocks of 32, the scale a power of two (e8m0)
* ``"nvfp4"``  blocks of 16, the scale e4m3, and one fp32 scale a row

The tensor cores multiply them with their scales at four times the bf16 rate.  ``native.fp4_quant`` has the layout.  As in the 8-bit linears,
activations are quantised per call, weights are frozen, and the activation is what has a gradient: the output's gradient is
quantised per token and the de-quantised weight per input channel to e4m3, and the FP8 GEMM multiplies them.  (A gradient of 4 bits would lose
an eighth of each value; the product of e4m3 takes twice the time.)  There are no forward-mode derivatives.

With a gradient, a fused GELU becomes a kernel of its own on the product rounded to bf16, which the backward pass takes again, because
the GELU kernels are those of the 8-bit linears, which read and write bf16 and e4m3.  So such a call has two roundings to bf16 where the call
without a gradient has one to the output's type, and other bits: 2002 x 2048 -> 8192 is off by some 2^-7 of an element at most in the place of
2^-8 with bf16 and 2^-10.9 with fp16.  Who trains in fp16 and needs its 11 bits leaves ``fuse_gelu`` off and takes the GELU of the fp16 output.
"""
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from .. import native
from .linear import is_16bit

FORMATS = tuple(native.FP4_FORMATS)
Scales = Tuple[torch.Tensor, Optional[torch.Tensor]]


def fp4_quantize(x: torch.Tensor, format: str = "nvfp4") -> Tuple[torch.Tensor, Scales]:
    """x [...,K] (bf16 or fp16, K a multiple of 32) as ``(values, (block scales, row scales))``: uint8 [...,K/2], two values a byte, block scales
    in tiles, e4m3 ("nvfp4") or e8m0 ("mxfp4"), row scales fp32 [...] ("nvfp4") or None.  No gradient."""
    values, block, row = native.fp4_quant(x.detach(), format)
    return values, (block, row)


def fp4_dequantize(values: torch.Tensor, scales: Scales, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """What ``values`` with ``scales`` stand for, [...,K] in bf16, fp16 or fp32."""
    native.fp4_format("fp4_dequantize", values, scales)
    return native.fp4_dequant(values, *scales, out_dtype)


class FP4LinearFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, a, b, bias, block, row, fuse_gelu, out_dtype):
        # (bf16 with GELU: see the module's docstring)
        y = native.fp4_linear(a, b, (block, row), bias, False, torch.bfloat16 if fuse_gelu else out_dtype)
        ctx.save_for_backward(b, block, row, y if fuse_gelu else None)
        ctx.dtype = a.dtype
        return native.gelu_forward(y, torch.bfloat16).to(out_dtype) if fuse_gelu else y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        b, block, row, y = ctx.saved_tensors
        n, k = b.shape[0], 2 * b.shape[1]
        if grad.numel() == 0:                                # no rows: fp8_mm refuses the null pointers of empty tensors
            return (grad.new_empty(*grad.shape[:-1], k, dtype=ctx.dtype),) + (None,) * 6
        if y is not None:
            grad = native.gelu_backward(y, grad.to(torch.bfloat16), torch.bfloat16)
        g8, gs = native.fp4_backward_quant(grad.reshape(-1, n))
        w8, ws = native.fp4_weight_operand(b, (block, row))
        dx = native.fp8_mm(g8, w8, gs, ws, False, ctx.dtype)
        return dx.reshape(*grad.shape[:-1], k), None, None, None, None, None, None


def fp4_linear(a: torch.Tensor, b: torch.Tensor, bias: Optional[torch.Tensor] = None, scale_a: Optional[Scales] = None,
               scale_b: Optional[Scales] = None, fuse_gelu: bool = False, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``act(a b^T + bias)`` with a 4-bit weight ``b`` uint8 [N,K/2] and its scales ``scale_b`` as ``fp4_quantize`` returns them, N a multiple of
    16.  ``a``: bf16 or fp16 [...,K], quantised in the weight's format first, or 4-bit values with ``scale_a``.  ``bias`` fp32 [N] or None; act is
    tanh-GELU with ``fuse_gelu``.  Returns [...,N] in ``out_dtype``, bf16 or fp16, by default a's type (bf16 for 4-bit a).
    Differentiable in an un-quantised ``a``, with N up to 32768."""
    if scale_b is None:
        raise native.Q8KernelError("fp4_linear: the weight must be 4-bit values with their scales")
    if scale_a is None and isinstance(scale_b, (tuple, list)) and len(scale_b) == 2 and isinstance(scale_b[0], torch.Tensor) \
            and scale_b[0].dtype != torch.uint8 and (scale_b[1] is None or scale_b[1].dtype == torch.float32):
        # (_host takes the bits that FP4Linear holds, too)
        fast = native._host._fp4_linear(a, b, bias, scale_b[0], scale_b[1], bool(fuse_gelu), out_dtype)
        if fast is not None:
            return fast
    out_dtype = (a.dtype if is_16bit(a) else torch.bfloat16) if out_dtype is None else out_dtype
    if not is_16bit(out_dtype):
        raise native.Q8KernelError(f"fp4_linear: output type {out_dtype} is not bfloat16 or float16")
    if scale_a is not None:
        native.refuse_tangents("fp4_linear", bias)
        return native.fp4_mm(a, b, bias, scale_a, scale_b, fuse_gelu, out_dtype)
    native.fp4_linear_check("fp4_linear", a, b, scale_b, bias)
    native.refuse_tangents("fp4_linear", a, bias, scale_b[1])
    if torch.is_grad_enabled() and a.requires_grad:
        if b.shape[0] > 32768:                                 # what quantises the gradient holds a row of it in a CTA
            raise native.Q8KernelError(f"fp4_linear: the gradient of {b.shape[0]} output channels: at most 32768 are supported")
        return FP4LinearFunc.apply(a, b, bias, *scale_b, bool(fuse_gelu), out_dtype)
    return native.fp4_linear(a, b, scale_b, bias, fuse_gelu, out_dtype)
