"""RotaryEmbedding and AxialRotaryEmbedding: queries and keys turned by their positions, HeadNormRotary: normed before (no counterparts in the
reference)."""
from typing import Optional, Sequence, Union

import torch
import torch.nn as nn

from .. import _host
from .. import functional as Q8F
from ..native import Q8KernelError


class RotaryEmbedding(nn.Module):
    """Rotates the first ``rotary_dim`` (all, if None) channels of every head; ``layout`` and ``scaling`` as in functional.rotary.
    ``forward(q, k, positions)`` takes [B,S,H,D] or [S,H,D] and returns the rotated pair."""

    def __init__(self, head_dim: int, rotary_dim: Optional[int] = None, base: float = 10000.0, layout: str = "half",
                 scaling: Optional[dict] = None, device=None):
        super().__init__()
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if layout not in Q8F.rotary.LAYOUTS:
            raise Q8KernelError(f"RotaryEmbedding: layout {layout!r} is not one of {', '.join(Q8F.rotary.LAYOUTS)}")
        frequencies, self.amplitude = Q8F.rotary.rotary_frequencies(rotary_dim, base, scaling)
        if rotary_dim > head_dim:
            raise Q8KernelError(f"RotaryEmbedding: rotary_dim {rotary_dim} exceeds the head dim {head_dim}")
        self.head_dim, self.rotary_dim, self.layout, self._half = head_dim, rotary_dim, layout, layout == "half"
        # held as the bits of the 64-bit values: a module that is cast to another floating type must not round them
        self.register_buffer("_frequency_bits", frequencies.view(torch.int64).to(device), persistent=False)

    @property
    def frequencies(self) -> torch.Tensor:
        return self._frequency_bits.view(torch.float64)

    def forward(self, q, k=None, positions=None):
        if q.shape[-1] != self.head_dim:
            raise Q8KernelError(f"RotaryEmbedding: heads of {q.shape[-1]} channels, {self.head_dim} expected")
        fast = _host._rotary(q, k, positions, self._frequency_bits, self.amplitude, self._half)
        if fast is not None:
            return fast
        return Q8F.rotary.apply_rotary(q, k, positions, self.frequencies, self.amplitude, self.layout)


class AxialRotaryEmbedding(nn.Module):
    """Rotates the first ``sum(sections)`` channels of every head by positions with an axis for each section (time, height, width); ``base``,
    ``spectrum`` and ``layout`` as in functional.rotary.  ``forward(q, k, positions)`` takes [B,S,H,D] or [S,H,D] and positions [S,A] or
    [B,S,A], whole or fractional, and returns the rotated pair."""

    def __init__(self, head_dim: int, sections: Sequence[int], base: Union[float, Sequence[float]] = 10000.0, layout: str = "interleaved",
                 spectrum: str = "own", device=None):
        super().__init__()
        if layout not in Q8F.rotary.LAYOUTS:
            raise Q8KernelError(f"AxialRotaryEmbedding: layout {layout!r} is not one of {', '.join(Q8F.rotary.LAYOUTS)}")
        frequencies, axes = Q8F.rotary.axial_frequencies(sections, base, spectrum)
        self.head_dim, self.sections, self.rotary_dim, self.layout = head_dim, tuple(sections), sum(sections), layout
        self.amplitude, self._half = 1.0, layout == "half"
        if self.rotary_dim > head_dim:
            raise Q8KernelError(f"AxialRotaryEmbedding: sections of {self.rotary_dim} channels exceed the head dim {head_dim}")
        # held as the bits of the 64-bit values: a module that is cast to another floating type must not round them
        self.register_buffer("_frequency_bits", frequencies.view(torch.int64).to(device), persistent=False)
        self.register_buffer("_axes", axes.to(device), persistent=False)

    @property
    def frequencies(self) -> torch.Tensor:
        return self._frequency_bits.view(torch.float64)

    @property
    def axes(self) -> torch.Tensor:
        return self._axes

    def forward(self, q, k, positions):
        if q.shape[-1] != self.head_dim:
            raise Q8KernelError(f"AxialRotaryEmbedding: heads of {q.shape[-1]} channels, {self.head_dim} expected")
        if positions is None or positions.dim() < 2 or positions.shape[-1] != len(self.sections):
            raise Q8KernelError(f"AxialRotaryEmbedding: positions {None if positions is None else tuple(positions.shape)} for {len(self.sections)} axes")
        fast = _host._axial_rotary(q, k, positions, self._frequency_bits, self._axes, self.amplitude, self._half)
        if fast is not None:
            return fast
        return Q8F.rotary.apply_axial_rotary(q, k, positions, self.frequencies, self._axes, self.amplitude, self.layout)


class HeadNormRotary(nn.Module):
    """RMS norm of every head of queries and keys and, with ``rotary`` (a RotaryEmbedding or AxialRotaryEmbedding), their rotation, in one pass.
    ``q_weight`` and ``k_weight`` are fp32 [head_dim] and trainable; ``elementwise_affine=False`` has neither.  In a model that is cast to 16
    bits they are rounded with it, and widened again in each call.  ``forward(q, k, positions)`` as that of ``rotary``; k may be None."""

    def __init__(self, head_dim: int, rotary: Optional[nn.Module] = None, eps: float = 1e-6, elementwise_affine: bool = True, device=None):
        super().__init__()
        if rotary is not None and (not isinstance(rotary, (RotaryEmbedding, AxialRotaryEmbedding)) or rotary.head_dim != head_dim):
            raise Q8KernelError(f"HeadNormRotary: {rotary} is no rotary embedding of heads of {head_dim} channels")
        self.head_dim, self.rotary, self.eps = head_dim, rotary, float(eps)
        for name in ("q_weight", "k_weight"):
            if elementwise_affine:
                setattr(self, name, nn.Parameter(torch.ones(head_dim, dtype=torch.float, device=device)))
            else:
                self.register_parameter(name, None)

    def forward(self, q, k=None, positions=None):
        if q.shape[-1] != self.head_dim:
            raise Q8KernelError(f"HeadNormRotary: heads of {q.shape[-1]} channels, {self.head_dim} expected")
        weights = [w if w is None or w.dtype == torch.float else w.float() for w in (self.q_weight, self.k_weight)]
        r = self.rotary
        if r is None:
            if positions is not None:
                raise Q8KernelError("HeadNormRotary: positions without a rotation")
            return Q8F.head_norm.head_norm(q, k, *weights, self.eps)
        axes = None
        if isinstance(r, AxialRotaryEmbedding):
            axes = r.axes
            if positions is None or positions.dim() < 2 or positions.shape[-1] != len(r.sections):
                raise Q8KernelError(f"HeadNormRotary: positions {None if positions is None else tuple(positions.shape)} for {len(r.sections)} axes")
        fast = _host._head_norm(q, k, *weights, self.eps, positions, r._frequency_bits, axes, r.amplitude, r._half)
        if fast is not None:
            return fast
        return Q8F.head_norm.head_norm(q, k, *weights, self.eps, positions, r.frequencies, axes, r.amplitude, r.layout)
