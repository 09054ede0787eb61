"""Drop-in for ``q8_kernels.functional`` (reference: q8_kernels/functional/__init__.py), and the ops beside it: ``fp4``, ``gated``,
``head_norm``, ``layer_norm``, ``rotary``."""
from . import fast_hadamard, flash_attention, fma, fp4, gated, head_norm, layer_norm, linear, quantizer, rms_norm, rope, rotary

__all__ = ["fast_hadamard", "flash_attention", "fma", "fp4", "gated", "head_norm", "layer_norm", "linear", "quantizer", "rms_norm", "rope", "rotary"]
