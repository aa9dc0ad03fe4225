"""``int8_linear``: a linear layer whose activations and weight are 8-bit integers with float32 scales.

    out[..., j] = input_scale[...] * weight_scale[j] * sum_k input[..., k] * weight[j, k] + bias[j]

The serving form of the projections around attention and its gated output stage: ``rms_norm_int8`` makes the
activations behind a norm, ``quantize_int8`` elsewhere, and the weight once, when a model is loaded.  The sums
are exact 32-bit integers on the int8 matrix units; scales and bias are applied in float32 (the conversion of a sum
above 2^24, the product with the token's scale and a fused product and addition round once each), then the result is
rounded to its type.  Kernels: csrc/int8_linear.hip.
The reference has no counterpart.
"""

from __future__ import annotations

import ctypes
import functools
from typing import Optional

import torch
from torch import Tensor

from .. import _lib
from .._errors import unsupported
from ..attention._runtime import (
    call_on,
    is_nested,
    needs_custom_op,
    on_one_device,
    require_no_forward_mode,
    require_same_device,
    wants_gradient,
)

_OPERATOR = "int8_linear"
_DTYPE_CODE = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
MAX_FEATURES = 131071  # 32-bit sums of products of -128 by -128


def int8_linear(
    input: Tensor,
    input_scale: Tensor,
    weight: Tensor,
    weight_scale: Tensor,
    bias: Optional[Tensor] = None,
    *,
    dtype: torch.dtype = torch.bfloat16,
) -> Tensor:
    r"""8-bit linear layer; inference only (no gradients).

    Args:
        input: CUDA int8 ``(..., K)`` activations, ``K`` up to 131071.
        input_scale: float32 ``(...)``, one scale a token (``input``'s leading shape).
        weight: int8 ``(N, K)``.
        weight_scale: float32 ``(N,)``, one scale an output channel.
        bias: optional ``(N,)``, float32 or ``dtype``.
        dtype: of the result, bfloat16 (default), float16 or float32.

    Returns ``(..., N)`` in ``dtype``.  Rows are read in place where the last dimension is contiguous; rows and
    pointers that are multiples of 16 bytes are the fast case.  ``quantize_int8`` and ``rms_norm_int8`` make rows of up
    to 16384 values; wider ones take the same formula in PyTorch, with x in float32: ``scale = x.abs().amax(-1) / 127``
    and ``torch.round(x / scale.clamp_min(1e-30)[..., None]).to(torch.int8)``.
    """

    if is_nested(input):
        raise unsupported(_OPERATOR, "takes dense tensors", hint="pass the packed values")
    require_no_forward_mode(_OPERATOR, input, input_scale, weight, weight_scale, bias)
    if not on_one_device(input.device, input_scale, weight, weight_scale, bias):
        require_same_device(_OPERATOR, input, input_scale, weight, weight_scale, bias)
    if input.dim() < 1 or weight.dim() != 2 or input.shape[-1] != weight.shape[1]:
        raise ValueError(f"{_OPERATOR} takes input (..., K) and weight (N, K), got {tuple(input.shape)} and "
                         f"{tuple(weight.shape)}")  # fmt: skip
    n, k = weight.shape
    if input_scale.shape != input.shape[:-1] or weight_scale.shape != (n,):
        raise ValueError(f"{_OPERATOR} takes one input scale a token {tuple(input.shape[:-1])} and one weight scale a "
                         f"channel ({n},), got {tuple(input_scale.shape)} and {tuple(weight_scale.shape)}")  # fmt: skip
    if bias is not None and bias.shape != (n,):
        raise ValueError(f"{_OPERATOR} bias must have shape ({n},), got {tuple(bias.shape)}")
    ok = (
        input.is_cuda
        and input.dtype == weight.dtype == torch.int8
        and input_scale.dtype == weight_scale.dtype == torch.float32
        and dtype in _DTYPE_CODE
        and (bias is None or bias.dtype in (dtype, torch.float32))
        and k <= MAX_FEATURES
        and n < 2**31
        and input.numel() // max(k, 1) < 2**31
    )
    if not ok:
        raise unsupported(
            _OPERATOR,
            "requires CUDA int8 operands with float32 scales, a bias in float32 or the result's dtype, and at most "
            "131071 input features",
            device=input.device,
            input_dtype=input.dtype,
            weight_dtype=weight.dtype,
            scale_dtypes=(input_scale.dtype, weight_scale.dtype),
            dtype=dtype,
            bias_dtype=None if bias is None else bias.dtype,
            features=k,
        )
    if wants_gradient(input_scale, weight_scale, bias):
        raise unsupported(_OPERATOR, "has no gradient", hint="call it under torch.no_grad() or on detached tensors")
    rows = input_scale.numel()
    x = _rows(input if input.dim() == 2 else input.reshape(rows, k))
    args = (x, _flat(input_scale), _rows(weight), _flat(weight_scale), None if bias is None else _flat(bias), dtype)
    out = int8_linear_forward(*args) if needs_custom_op(*args[:-1]) else _forward_impl(*args)
    return out if input.dim() == 2 else out.view(*input.shape[:-1], n)


def _rows(t: Tensor) -> Tensor:
    t = t.resolve_neg()
    if (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        t = t.contiguous()
    return t


def _flat(t: Tensor) -> Tensor:
    t = t.resolve_neg()
    return t.reshape(-1).contiguous() if t.dim() != 1 or not t.is_contiguous() else t


@functools.lru_cache(maxsize=1024)
def _geometry(lib, rows: int, n: int, k: int, x_row: int, w_row: int, out_dtype, bias_dtype) -> tuple:
    """The launch geometry and its workspace (cached: the library only reads it)."""

    geo = ctypes.pointer(_lib.Int8Geometry(rows, n, k, x_row, w_row, _DTYPE_CODE[out_dtype], _DTYPE_CODE[bias_dtype]))
    return geo, lib.oops_int8_linear_workspace_bytes(geo)


def _forward_impl(x: Tensor, x_scale: Tensor, weight: Tensor, weight_scale: Tensor, bias: Optional[Tensor],
                  dtype: torch.dtype) -> Tensor:  # fmt: skip
    lib = _lib.load()
    rows, k = x.shape
    n = weight.shape[0]
    geo, ws_bytes = _geometry(lib, rows, n, k, x.stride(0) if rows > 1 else k, weight.stride(0) if n > 1 else k, dtype,
                              dtype if bias is None else bias.dtype)  # fmt: skip
    device = x.device
    out = torch.empty((rows, n), dtype=dtype, device=device)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device) if ws_bytes else None
    rc = call_on(device.index, lib.oops_int8_linear, geo, x.data_ptr(), x_scale.data_ptr(), weight.data_ptr(),
                 weight_scale.data_ptr(), None if bias is None else bias.data_ptr(), out.data_ptr(),
                 None if ws is None else ws.data_ptr(), ws_bytes)
    _lib.check(rc, _OPERATOR)
    return out


@torch.library.custom_op("oops_amd::int8_linear", mutates_args=(), device_types="cuda")
def int8_linear_forward(x: Tensor, x_scale: Tensor, weight: Tensor, weight_scale: Tensor, bias: Optional[Tensor],
                        dtype: torch.dtype) -> Tensor:  # fmt: skip
    """Rows ``x`` (rows, K) and ``weight`` (N, K) with unit column strides."""

    return _forward_impl(x, x_scale, weight, weight_scale, bias, dtype)


@int8_linear_forward.register_fake
def _(x, x_scale, weight, weight_scale, bias, dtype):
    return x.new_empty(x.shape[0], weight.shape[0], dtype=dtype)
