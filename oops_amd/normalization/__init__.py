"""Normalization operators (the reference's ``oops.normalization``, and the root-mean-square norm)."""

from .layer_norm import layer_norm
from .modules import LayerNorm, RMSNorm
from .rms_norm import quantize_int8, rms_norm, rms_norm_int8
from .rotary import rms_norm_rotary, rotary_table

__all__ = ["LayerNorm", "RMSNorm", "layer_norm", "quantize_int8", "rms_norm", "rms_norm_int8", "rms_norm_rotary", "rotary_table"]
