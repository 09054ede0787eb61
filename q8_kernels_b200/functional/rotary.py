"""Rotary embedding from positions: half and interleaved layouts, part of a head, scaled for long contexts, queries and keys in one launch
(no counterpart in the reference, which rotates whole rows of interleaved pairs by fp32 tables: see rope.py)."""
import math
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from .. import _host
from ..native import Q8KernelError, refuse_tangents
from ..native import rotary as _rotary

LAYOUTS = ("half", "interleaved")


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[dict] = None) -> Tuple[torch.Tensor, float]:
    """Radians per position of each of the ``rotary_dim / 2`` pairs, ``base ** (-2i / rotary_dim)``, as a float64 CPU tensor, and the
    factor on cosine and sine.  ``scaling`` stretches them over a longer context:

    * ``{"type": "linear", "factor": f}``  positions divided by f
    * ``{"type": "ntk", "factor": f}``     base times ``f ** (rotary_dim / (rotary_dim - 2))``: the slowest pair is slowed down by f, the
      fastest not at all
    * ``{"type": "yarn", "factor": f, "original_length": n}``  pairs that turn more than ``beta_fast`` (32) times within n positions
      keep their frequency, those that turn less than ``beta_slow`` (1) times are slowed down by f, a linear ramp over the pairs
      between; cosine and sine times ``amplitude`` (``0.1 ln f + 1``)
    """
    if not isinstance(rotary_dim, int) or rotary_dim < 2 or rotary_dim % 2:
        raise Q8KernelError(f"rotary_frequencies: rotary_dim {rotary_dim} must be a positive even number")
    if not base > 1.0:
        raise Q8KernelError(f"rotary_frequencies: base {base} must be greater than 1")
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    if scaling is None:
        return base ** (-2.0 * i / rotary_dim), 1.0
    known = {"linear": {"factor"}, "ntk": {"factor"},
             "yarn": {"factor", "original_length", "beta_fast", "beta_slow", "amplitude"}}
    kind = scaling.get("type")
    if kind not in known:
        raise Q8KernelError(f"rotary_frequencies: scaling type {kind!r} is not one of {', '.join(known)}")
    unknown = set(scaling) - known[kind] - {"type"}
    if unknown:
        raise Q8KernelError(f"rotary_frequencies: {kind} scaling has no {', '.join(sorted(unknown))}")
    factor = scaling.get("factor")
    if not isinstance(factor, (int, float)) or not factor >= 1.0:
        raise Q8KernelError(f"rotary_frequencies: factor {factor} must be at least 1")
    if kind == "linear":
        return base ** (-2.0 * i / rotary_dim) / factor, 1.0
    if kind == "ntk":
        if rotary_dim == 2:
            raise Q8KernelError("rotary_frequencies: ntk scaling needs a rotary_dim of 4 or more")
        return (base * factor ** (rotary_dim / (rotary_dim - 2.0))) ** (-2.0 * i / rotary_dim), 1.0
    length, fast, slow = scaling.get("original_length"), scaling.get("beta_fast", 32.0), scaling.get("beta_slow", 1.0)
    if not isinstance(length, (int, float)) or not length > 0 or not fast > slow > 0:
        raise Q8KernelError("rotary_frequencies: yarn scaling needs original_length > 0 and beta_fast > beta_slow > 0")

    def pair(turns):                                         # number of the pair that turns so often within `length` positions
        return rotary_dim * math.log(length / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

    low, high = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), rotary_dim - 1)
    ramp = ((i - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
    freq = base ** (-2.0 * i / rotary_dim)
    return freq * (1.0 - ramp) + freq / factor * ramp, float(scaling.get("amplitude", 0.1 * math.log(factor) + 1.0))


class Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, frequencies, amplitude, half):
        ctx.save_for_backward(positions, frequencies)
        ctx.amplitude, ctx.half = amplitude, half
        ctx.set_materialize_grads(False)
        return _rotary(q, k, positions, frequencies, amplitude, half, False)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_q, grad_k):
        positions, frequencies = ctx.saved_tensors
        need_q, need_k = ctx.needs_input_grad[:2]
        grads = [g if need else None for g, need in ((grad_q, need_q), (grad_k, need_k))]
        if any(g is not None for g in grads):
            grads = _rotary(grads[0], grads[1], positions, frequencies, ctx.amplitude, ctx.half, True)
        return (*grads, None, None, None, None)


def apply_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: Optional[torch.Tensor], frequencies: torch.Tensor,
                 amplitude: float = 1.0, layout: str = "half"):
    """Turns the first ``2 * len(frequencies)`` channels of every head of ``q`` [B,S,Hq,D] and ``k`` [B,S,Hk,D] (or None; both also [S,H,D])
    by ``position * frequency`` and scales them by ``amplitude``; the other channels are copied.  bf16, fp16 or fp32, any strides;
    returns new dense tensors ``(q', k')``.  ``positions``: int32 or int64 [S], [1,S] or [B,S], any size and sign, or None for 0, 1, ...;
    ``frequencies``: float64 on the device (``rotary_frequencies``).  ``layout``: channel i is paired with i + rotary_dim / 2 ("half") or
    2i with 2i + 1 ("interleaved").  Differentiable in q and k."""
    if layout not in LAYOUTS:
        raise Q8KernelError(f"apply_rotary: layout {layout!r} is not one of {', '.join(LAYOUTS)}")
    if frequencies.dtype != torch.float64:                       # (_host takes int64 as the bits that RotaryEmbedding holds)
        raise Q8KernelError(f"apply_rotary: frequencies must be float64 [rotary_dim / 2], not {frequencies.dtype}")
    amplitude, half = float(amplitude), layout == "half"
    fast = _host._rotary(q, k, positions, frequencies, amplitude, half)
    if fast is not None:
        return fast
    refuse_tangents("apply_rotary", q, k, frequencies)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return Rotary.apply(q, k, positions, frequencies, amplitude, half)
    return _rotary(q, k, positions, frequencies, amplitude, half, False)
