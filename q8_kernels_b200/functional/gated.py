"""Gated 8-bit linears: gate and up projection, activation and product in one kernel (no counterpart in the reference, whose feed-forward
has one projection with GELU).

The weight ``b`` [2F, K] holds the gate's rows first and the up projection's behind them, with one scale per row.  Activations are
quantised as ``q8_linear`` and ``fp8_linear`` do it, but for the last bit of a row's factor (see native.gated_quant); where the bits of those
are wanted, quantise with them and pass ``scale_a``.  As there, weights are frozen and the activation is what has a gradient: the
gradient of [gate | up] is quantised per token and the de-quantised weight per input channel to e4m3, the FP8 GEMM
multiplies them, and the result is rotated back where the forward pass rotated.  Both the product and the rotated result are rounded to
bf16, as in q8_linear's backward pass: the transform takes 16-bit rows, and half a bf16 step is far below the e4m3 steps before it (a step of
2002 x 2048 x 5504 is 0.0024 from 64 bits, the formulas in fp32 with that product unrounded 0.0024 to 0.0026).  fp16 activations are rounded
to bf16 first.

A row with NaN gives NaN throughout, in int8 too; rows of values down to the smallest ones give no NaN.  There are no forward-mode derivatives.
"""
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from .. import native
from .fast_hadamard import hadamard_transform
from .linear import E4M3, is_16bit


def _quantised(a, int8, rotate):
    if a.dtype == torch.float16:
        a = a.to(torch.bfloat16)
    return native.gated_quant(a, rotate, torch.int8 if int8 else E4M3)


class GatedLinearFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, a, b, bias, scale_b, act, int8, rotate):
        q, qs = _quantised(a, int8, rotate)
        out, pre = native.gated_mm(q, b, bias, qs, scale_b, act, True)
        ctx.save_for_backward(pre, b, scale_b)
        ctx.act, ctx.rotate, ctx.dtype = act, rotate, a.dtype
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        pre, b, scale_b = ctx.saved_tensors
        if grad.numel() == 0:                                # no rows: fp8_mm refuses the null pointers of empty tensors
            return (grad.new_empty(*grad.shape[:-1], b.shape[1], dtype=ctx.dtype),) + (None,) * 6
        g8, gs = native.gated_backward_quant(grad.to(torch.bfloat16), pre, ctx.act)
        w8, ws = native.gated_weight_operand(b, scale_b)
        k = b.shape[1]
        dx = native.fp8_mm(g8.reshape(-1, g8.shape[-1]), w8, gs.reshape(-1), ws, False, torch.bfloat16).reshape(*grad.shape[:-1], k)
        if ctx.rotate:
            dx = hadamard_transform(dx)
        return dx.to(ctx.dtype), None, None, None, None, None, None


def _gated(op, a, b, bias, scale_a, scale_b, act, int8, rotate):
    if scale_a is None:
        fast = native._host._gated_linear(a, b, bias, scale_b, native.ACTIVATIONS.get(act, 0), int8, rotate)
        if fast is not None:
            return fast
    native.refuse_tangents(op, a, bias, scale_a, scale_b)
    weight_type = torch.int8 if int8 else E4M3
    if b.dtype != weight_type or scale_b is None:
        raise native.Q8KernelError(f"{op}: the weight must be {weight_type} with its scales")
    if scale_a is not None:
        if a.dtype != weight_type:
            raise native.Q8KernelError(f"{op}: an activation with scales must be {weight_type}, not {a.dtype}")
        return native.gated_mm(a, b, bias, scale_a, scale_b, act, False)[0]
    if not (is_16bit(a) or (int8 and a.dtype == E4M3)):
        raise native.Q8KernelError(f"{op}: an activation of type {a.dtype} needs scales" if a.dtype == weight_type
                                   else f"{op}: activation type {a.dtype} is not supported")
    if torch.is_grad_enabled() and a.requires_grad:
        native.gated_check(a, b, bias, None, scale_b, act, op, training=True)
        return GatedLinearFunc.apply(a, b, bias, scale_b, act, int8, rotate)
    native.gated_check(a, b, bias, None, scale_b, act, op)
    q, qs = _quantised(a, int8, rotate)
    return native.gated_mm(q, b, bias, qs, scale_b, act, False)[0]


def q8_gated_linear(a: torch.Tensor, b: torch.Tensor, bias: Optional[torch.Tensor] = None, scale_a: Optional[torch.Tensor] = None,
                    scale_b: Optional[torch.Tensor] = None, act: str = "silu") -> torch.Tensor:
    """``act(a Wg^T + bg) * (a Wu^T + bu)`` in bf16, with ``b`` = [Wg; Wu] int8 [2F,K], ``scale_b`` fp32 [2F] and ``bias`` fp32 [2F] or None.
    ``a`` [...,K]: bf16, fp16 or e4m3, rotated (Hadamard, 1/sqrt(K)) and quantised per token first, or int8 with ``scale_a``.
    ``act``: "silu" or "gelu_tanh".  F and K are multiples of 16.  Differentiable in an un-quantised ``a`` (F up to 16384)."""
    return _gated("q8_gated_linear", a, b, bias, scale_a, scale_b, act, True, True)


def fp8_gated_linear(a: torch.Tensor, b: torch.Tensor, bias: Optional[torch.Tensor] = None, scale_a: Optional[torch.Tensor] = None,
                     scale_b: Optional[torch.Tensor] = None, act: str = "silu", use_hadamard: bool = False) -> torch.Tensor:
    """``q8_gated_linear`` with an e4m3 weight: ``a`` is bf16 or fp16, quantised per token to e4m3 (with ``use_hadamard`` after the rotation),
    or e4m3 with ``scale_a``."""
    return _gated("fp8_gated_linear", a, b, bias, scale_a, scale_b, act, False, bool(use_hadamard))
