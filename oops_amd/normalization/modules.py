"""``LayerNorm`` and ``RMSNorm``: the ``torch.nn`` modules on the HIP row kernels.

Drop-in for the reference's module (oops/normalization/layer_norm/modules.py:31-70,
exported as ``oops.LayerNorm``): the constructor, parameters and state dict are
``torch.nn.LayerNorm``'s; a call goes through ``layer_norm`` and, when that
operator declines the input with ``OOpsUnsupportedError`` (CPU tensors, float64,
several normalized dimensions, widths above 8192, ...), through PyTorch's own
LayerNorm instead.  Call ``layer_norm`` directly where unsupported inputs should
raise.  ``RMSNorm`` does the same for ``torch.nn.RMSNorm`` and takes the residual
that ``rms_norm`` adds.
"""

from __future__ import annotations

import torch
from torch import Tensor, nn

from .._errors import OOpsUnsupportedError
from .layer_norm import layer_norm
from .rms_norm import rms_norm


class LayerNorm(nn.LayerNorm):
    """``torch.nn.LayerNorm`` whose served calls run ``oops_amd.layer_norm``."""

    def forward(self, input: Tensor) -> Tensor:
        try:
            return layer_norm(input, self.normalized_shape, self.weight, self.bias, self.eps)
        except OOpsUnsupportedError:
            return super().forward(input)


class RMSNorm(nn.RMSNorm):
    """``torch.nn.RMSNorm`` whose served calls run ``oops_amd.rms_norm``.  With a ``residual`` the call returns
    ``(y, input + residual)``."""

    def forward(self, input: Tensor, residual: Tensor | None = None):
        # (PyTorch's default is the eps of the type it computes in: float32's for every type that rms_norm takes)
        eps = torch.finfo(torch.float32).eps if self.eps is None else self.eps
        try:
            return rms_norm(input, self.normalized_shape, self.weight, eps, residual)
        except OOpsUnsupportedError:
            if residual is None:
                return super().forward(input)
            summed = input + residual
            return super().forward(summed), summed
