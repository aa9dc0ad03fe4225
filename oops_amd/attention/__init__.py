"""Attention operators (gfx950 HIP kernels): the reference's pair-biased attention, linear attention, and causal attention
with its 4-bit key/value cache."""

from .cache import cache_attention, cache_read, cache_write, quantized_cache
from .causal import causal_attention
from .gate import gate_attention_output, gated_pair_bias_attention
from .linear import linear_attention, linear_attention_step
from .pair_bias import pair_bias_attention
from .triangle import triangle_attention

__all__ = [
    "cache_attention",
    "cache_read",
    "cache_write",
    "causal_attention",
    "gate_attention_output",
    "gated_pair_bias_attention",
    "linear_attention",
    "linear_attention_step",
    "pair_bias_attention",
    "quantized_cache",
    "triangle_attention",
]
