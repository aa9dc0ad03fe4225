"""Linear layers on the HIP matrix kernels."""

from .int8 import int8_linear

__all__ = ["int8_linear"]
