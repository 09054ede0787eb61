"""Drop-in for ``q8_kernels.modules`` (reference: q8_kernels/modules/), and the modules beside it: ``AxialRotaryEmbedding``,
``FP4Linear``, ``GatedLinear``, ``GatedFeedForward``, ``HeadNormRotary``, ``LayerNorm``, ``RotaryEmbedding``."""
from .activations import GELU, GatedLinear
from .attention import Attention
from .ffn import FeedForward, GatedFeedForward
from .layer_norm import LayerNorm
from .linear import FP4Linear, FP8Linear, Q8Linear, Q8LinearLora
from .rms_norm import RMSNorm
from .rotary import AxialRotaryEmbedding, HeadNormRotary, RotaryEmbedding

__all__ = ["Attention", "AxialRotaryEmbedding", "FeedForward", "FP4Linear", "FP8Linear", "GatedFeedForward", "GatedLinear", "GELU", "HeadNormRotary",
           "LayerNorm", "Q8Linear", "Q8LinearLora", "RMSNorm", "RotaryEmbedding"]
