"""Norms of queries and keys for each head, with the rotation by position in the same pass (no counterpart in the reference, which norms whole rows
and rotates them by tables: see rms_norm.py, rope.py).

``y = R(p) (x / sqrt(mean(x^2) + eps) * weight)`` over the channels of a head, in fp32 and rounded once; squares are fp32's, so |x| has to be below
1e19, and without eps above 1e-19.  The gradients are those of the formula.  All sums, those of the weights' gradients over tokens and heads
among them, are taken in an order that sizes, strides, alignment of the tensors and the number of SMs fix: equal calls give equal bits, the same values at
other strides or an odd address may differ in the last fp32 bits.  There are no forward-mode derivatives.
"""
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from .. import native
from .rotary import LAYOUTS


class HeadNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, eps, positions, frequencies, axes, amplitude, half):
        ctx.save_for_backward(q, k, q_weight, k_weight, positions, frequencies, axes)
        ctx.eps, ctx.amplitude, ctx.half = eps, amplitude, half
        ctx.set_materialize_grads(False)
        return native.head_norm(q, k, q_weight, k_weight, eps, positions, frequencies, axes, amplitude, half)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_q, grad_k):
        q, k, q_weight, k_weight, positions, frequencies, axes = ctx.saved_tensors
        need = ctx.needs_input_grad
        grads = [g if need[i] or need[2 + i] else None for i, g in enumerate((grad_q, grad_k))]
        if all(g is None for g in grads):
            return (None,) * 10
        d = native.head_norm_backward(q, k, q_weight, k_weight, *grads, ctx.eps, positions, frequencies, axes, ctx.amplitude, ctx.half, need[2:4])
        return (*(g if n else None for g, n in zip(d, need)), None, None, None, None, None, None)


def head_norm(q: torch.Tensor, k: Optional[torch.Tensor] = None, q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
              eps: float = 1e-6, positions: Optional[torch.Tensor] = None, frequencies: Optional[torch.Tensor] = None,
              axes: Optional[torch.Tensor] = None, amplitude: float = 1.0, layout: str = "half"):
    """RMS norm of every head of ``q`` [B,S,Hq,D] and ``k`` [B,S,Hk,D] (or None; both also [S,H,D]) with fp32 weights [D] (or None), then the
    rotation of ``apply_rotary``, or with ``axes`` of ``apply_axial_rotary``; none without ``frequencies``.  bf16, fp16 or fp32, any strides, D up
    to 512; returns new dense tensors ``(q', k')``.  Differentiable in q, k and the weights."""
    if layout not in LAYOUTS:
        raise native.Q8KernelError(f"head_norm: layout {layout!r} is not one of {', '.join(LAYOUTS)}")
    if not eps >= 0.0:
        raise native.Q8KernelError(f"head_norm: eps {eps} must not be negative")
    if frequencies is not None and frequencies.dtype != torch.float64:           # (_host takes int64 as the bits that the modules hold)
        raise native.Q8KernelError(f"head_norm: frequencies must be float64 [rotary_dim / 2], not {frequencies.dtype}")
    eps, amplitude, half = float(eps), float(amplitude), layout == "half"
    fast = native._host._head_norm(q, k, q_weight, k_weight, eps, positions, frequencies, axes, amplitude, half)
    if fast is not None:
        return fast
    native.refuse_tangents("head_norm", q, k, q_weight, k_weight, positions, frequencies)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
        return HeadNorm.apply(q, k, q_weight, k_weight, eps, positions, frequencies, axes, amplitude, half)
    return native.head_norm(q, k, q_weight, k_weight, eps, positions, frequencies, axes, amplitude, half)
