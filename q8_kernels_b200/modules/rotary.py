"""RotaryEmbedding: queries and keys turned by their positions (no counterpart in the reference)."""
from typing import Optional

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
