"""Drop-in for ``q8_kernels.modules`` (reference: q8_kernels/modules/), and the modules beside it: ``GatedLinear``, ``GatedFeedForward``,
``LayerNorm``, ``RotaryEmbedding``."""
from .activations import GELU, GatedLinear
from .attention import Attention
from .ffn import FeedForward, GatedFeedForward
from .layer_norm import LayerNorm
from .linear import FP8Linear, Q8Linear, Q8LinearLora
from .rms_norm import RMSNorm
from .rotary import RotaryEmbedding

__all__ = ["Attention", "FeedForward", "FP8Linear", "GatedFeedForward", "GatedLinear", "GELU", "LayerNorm", "Q8Linear", "Q8LinearLora",
           "RMSNorm", "RotaryEmbedding"]
