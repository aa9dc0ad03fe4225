"""Attention operators (gfx950 HIP kernels): the reference's pair-biased attention, and linear attention."""

from .gate import gate_attention_output, gated_pair_bias_attention
from .linear import linear_attention, linear_attention_step
from .pair_bias import pair_bias_attention
from .triangle import triangle_attention

__all__ = [
    "gate_attention_output",
    "gated_pair_bias_attention",
    "linear_attention",
    "linear_attention_step",
    "pair_bias_attention",
    "triangle_attention",
]
