"""oops_amd: MI355X-native pair-biased triangle attention (and the operators beside it) with the OOps API.

``from oops_amd import triangle_attention, pair_bias_attention, OOpsUnsupportedError``
is the drop-in for ``from oops import ...`` on the attention path.
"""

from ._errors import OOpsUnsupportedError
from .attention import (
    gate_attention_output,
    gated_pair_bias_attention,
    linear_attention,
    linear_attention_step,
    pair_bias_attention,
    triangle_attention,
)
from .linear import int8_linear
from .normalization import LayerNorm, RMSNorm, layer_norm, quantize_int8, rms_norm, rms_norm_int8
from .pair import triangle_multiplication

__all__ = [
    "LayerNorm",
    "OOpsUnsupportedError",
    "RMSNorm",
    "gate_attention_output",
    "gated_pair_bias_attention",
    "int8_linear",
    "layer_norm",
    "linear_attention",
    "linear_attention_step",
    "pair_bias_attention",
    "quantize_int8",
    "rms_norm",
    "rms_norm_int8",
    "triangle_attention",
    "triangle_multiplication",
]
