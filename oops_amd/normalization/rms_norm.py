"""``rms_norm`` and its 8-bit form: the root-mean-square norm over the last dimension on the HIP row kernels.

    h = input + residual            (rounded to the input's dtype, returned as the new residual stream)
    y = h * (mean(h^2) + eps)^-1/2 * weight

The norm of language-model blocks, beside ``layer_norm`` and with its conventions: float16 / bfloat16 /
float32 activations, an optional weight in the activation dtype or float32, float32 statistics, rows read in
place where the last dimension is contiguous, nested inputs.  ``rms_norm_int8`` returns each row of y in 8 bits
with a float32 scale, what ``int8_linear`` reads; ``quantize_int8`` does that without the norm.  Kernels:
csrc/rms_norm.hip.  The reference has no counterpart.
"""

from __future__ import annotations

import ctypes
import functools
from typing import Iterable, Optional, Tuple, Union

import torch
from torch import Tensor

from .. import _lib
from .._errors import unsupported
from ..attention._runtime import (
    any_wrapped,
    call_on,
    is_nested,
    needs_custom_op,
    on_one_device,
    require_no_forward_mode,
    require_same_device,
    wants_gradient,
    without_second_derivative,
)
from .layer_norm import _ptr

_DTYPE_CODE = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
MAX_WIDTH = 16384


def rms_norm(
    input,
    normalized_shape: Union[int, Iterable[int]],
    weight: Optional[Tensor] = None,
    eps: float = 1e-6,
    residual=None,
):
    r"""Root-mean-square norm of the final feature dimension, after adding ``residual`` if one is given.

    Args:
        input: CUDA float16 / bfloat16 / float32 ``(..., C)`` tensor, or a nested tensor whose final feature
            axis is static and physically last.
        normalized_shape: ``C`` or ``(C,)`` with ``1 <= C <= 16384``.
        weight: optional ``(C,)`` in the activation dtype or float32.
        eps: added to the mean square before the reciprocal square root.
        residual: optional tensor of the input's shape and dtype (nested with the same packing for a nested
            input), added first; the sum is rounded to that dtype.

    Returns ``y``, or ``(y, summed)`` with a residual: ``summed`` is the new residual stream.  Both take part in
    autograd; second derivatives raise.
    """

    if is_nested(input):
        return _nested("rms_norm", input, residual, lambda x, r: rms_norm(x, normalized_shape, weight, eps, r))
    _check("rms_norm", input, normalized_shape, weight, residual)
    x, r = _rows(input), _rows(residual)
    w = None if weight is None else weight.resolve_neg().contiguous()
    grad = wants_gradient(input, weight, residual)
    if needs_custom_op(x, w, r):
        y, summed, _ = rms_norm_forward(x, w, r, float(eps), grad)
    elif grad:
        y, summed = _EagerRmsNorm.apply(x, w, r, float(eps))
    else:
        y, summed, _ = _forward_impl(x, w, r, float(eps), False)
    y = y if input.dim() == 2 else y.view(input.shape)
    if residual is None:
        return y
    return y, summed if input.dim() == 2 else summed.view(input.shape)


def rms_norm_int8(
    input,
    normalized_shape: Union[int, Iterable[int]],
    weight: Optional[Tensor] = None,
    eps: float = 1e-6,
    residual=None,
):
    r"""``rms_norm`` with an 8-bit output for ``int8_linear``; inference only (no gradients).

    Arguments as for ``rms_norm`` (no nested inputs).  Returns ``(values, scales)``, or
    ``(values, scales, summed)`` with a residual: int8 ``values`` of the input's shape in -127..127 and float32
    ``scales`` of its leading shape, with ``y = values * scales[..., None]`` to half a step.  ``y`` is quantized
    from its float32 values.  A row of zeros has scale 0; a row that holds an infinity or a NaN has zero values
    and the scale NaN, so what is computed from it is NaN.
    """

    operator = "rms_norm_int8"
    _check(operator, input, normalized_shape, weight, residual)
    _require_inference(operator, input, weight, residual)
    x, r = _rows(input), _rows(residual)
    w = None if weight is None else weight.resolve_neg().contiguous()
    call = rms_norm_int8_forward if needs_custom_op(x, w, r) else _int8_impl
    values, scales, summed = call(x, w, r, float(eps))
    if input.dim() != 2:
        values, scales = values.view(input.shape), scales.view(input.shape[:-1])
        summed = summed.view(input.shape) if residual is not None else summed
    return (values, scales) if residual is None else (values, scales, summed)


def quantize_int8(input: Tensor) -> Tuple[Tensor, Tensor]:
    r"""Each row of the last dimension in 8 bits: ``values = rint(input * 127 / max|row|)``, ``scales = max|row| / 127``.

    ``input``: CUDA float16 / bfloat16 / float32 ``(..., C)``, ``C`` in 1..16384: activations, or the weight
    ``(out_features, in_features)`` of an 8-bit linear layer (wider rows: see ``int8_linear``).  Returns int8 values and
    float32 scales as ``rms_norm_int8`` does; inference only.
    """

    operator = "quantize_int8"
    _check(operator, input, 0 if is_nested(input) or not input.dim() else input.shape[-1], None, None)
    _require_inference(operator, input)
    x = _rows(input)
    call = quantize_int8_forward if needs_custom_op(x) else _quantize_impl
    values, scales = call(x)
    return (values, scales) if input.dim() == 2 else (values.view(input.shape), scales.view(input.shape[:-1]))


# ----------------------------------------------------------------- checks


def _check(operator: str, input: Tensor, normalized_shape, weight: Optional[Tensor], residual: Optional[Tensor]) -> None:
    if is_nested(input):  # (rms_norm has taken its packed values)
        raise unsupported(operator, "takes dense tensors", hint="pass the packed values")
    if is_nested(residual):
        raise ValueError(f"{operator} residual must have the input's shape")
    require_no_forward_mode(operator, input, weight, residual)
    if not on_one_device(input.device, weight, residual):
        require_same_device(operator, input, weight, residual)
    shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(normalized_shape)
    if len(shape) != 1:
        raise unsupported(operator, "normalizes over the final dimension only", normalized_shape=shape)
    width = shape[0]
    if residual is not None and residual.shape != input.shape:
        raise ValueError(f"{operator} residual must have the input's shape")
    ok = (
        input.is_cuda
        and input.dtype in _DTYPE_CODE
        and input.dim() >= 1
        and input.shape[-1] == width
        and 0 < width <= MAX_WIDTH
        and input.numel() // width < 2**31
        and (residual is None or residual.dtype == input.dtype)
        and (weight is None or (tuple(weight.shape) == (width,) and weight.dtype in (input.dtype, torch.float32)))
    )
    if not ok:
        raise unsupported(
            operator,
            "requires a CUDA half/float32 activation of 1..16384 channels, a residual of its dtype and a matching "
            "weight in its dtype or float32",
            input_dtype=input.dtype,
            device=input.device,
            normalized_size=width,
            weight_dtype=None if weight is None else weight.dtype,
            residual_dtype=None if residual is None else residual.dtype,
        )


def _require_inference(operator: str, *tensors) -> None:
    if wants_gradient(*tensors):
        raise unsupported(operator, "has no gradient", hint="call it under torch.no_grad() or on detached tensors")


def _nested(operator: str, input, residual, call):
    """A packed ragged batch: the operator on its packed values (as ``layer_norm`` takes it)."""

    if input.dim() < 2 or not input.ragged_dims or input.concat.dim() < 1:
        raise unsupported(operator, "requires a NestedTensor with explicit packed element topology")
    last = input.dim() - 2
    if last in tuple(input.ragged_dims) or tuple(input.packed_dim_order)[-1] != last:
        raise unsupported(operator, "requires the final logical element dimension to be static and physically last",
                          ragged_dims=input.ragged_dims, packed_dim_order=input.packed_dim_order)  # fmt: skip
    if residual is None:
        return input.packed_like(call(input.concat, None))
    if (not is_nested(residual) or tuple(residual.packed_dim_order) != tuple(input.packed_dim_order)
            or residual.element_sizes() != input.element_sizes()):
        raise ValueError(f"{operator} residual must be nested with the input's packing")
    y, summed = call(input.concat, residual.concat)
    return input.packed_like(y), input.packed_like(summed)


def _rows(t: Optional[Tensor]) -> Optional[Tensor]:
    """(rows, C) with unit column stride (a 2-D tensor is used as it is: views add autograd nodes)."""

    if t is None:
        return None
    x = t.resolve_neg()
    if x.dim() != 2:
        x = x.reshape(x.numel() // x.shape[-1], x.shape[-1])
    if (x.stride(1) != 1 and x.shape[1] > 1) or (x.shape[0] > 1 and x.stride(0) < x.shape[1]):
        x = x.contiguous()
    return x


# ----------------------------------------------------------------- launches


@functools.lru_cache(maxsize=256)
def _geometry(dtype, weight_f32: bool, rows: int, width: int, x_row: int, r_row: int, eps: float) -> "ctypes._Pointer":
    """The launch geometry (cached: the library only reads it)."""

    return ctypes.pointer(_lib.RmsNormGeometry(_DTYPE_CODE[dtype], int(weight_f32), width, eps, rows, x_row, r_row))


def _geometry_of(x: Tensor, weight: Optional[Tensor], residual: Optional[Tensor], eps: float) -> "ctypes._Pointer":
    rows, width = x.shape
    x_row = x.stride(0) if rows > 1 else width
    r_row = residual.stride(0) if residual is not None and rows > 1 else width
    return _geometry(x.dtype, weight is not None and weight.dtype == torch.float32, rows, width, x_row, r_row, eps)


@functools.lru_cache(maxsize=64)
def _workspace_bytes(lib, dtype, weight_f32: bool, rows: int, width: int) -> int:
    return lib.oops_rms_norm_backward_workspace_bytes(_geometry(dtype, weight_f32, rows, width, width, width, 0.0))


def _empty_rows(x: Tensor, dtype=None) -> Tensor:
    return torch.empty(x.shape, dtype=dtype or x.dtype, device=x.device)


def _forward_impl(x: Tensor, weight: Optional[Tensor], residual: Optional[Tensor], eps: float,
                  save: bool) -> Tuple[Tensor, Tensor, Tensor]:  # fmt: skip
    lib = _lib.load()
    y = _empty_rows(x)
    summed = _empty_rows(x) if residual is not None else x.new_empty(0)
    rstd = torch.empty(x.shape[0] if save else 0, dtype=torch.float32, device=x.device)
    geo = _geometry_of(x, weight, residual, eps)
    rc = call_on(x.device.index, lib.oops_rms_norm_forward, geo, _ptr(x), _ptr(residual), _ptr(weight), _ptr(y),
                 _ptr(summed), _ptr(rstd))  # fmt: skip
    _lib.check(rc, "rms_norm forward")
    return y, summed, rstd


def _int8_impl(x: Tensor, weight: Optional[Tensor], residual: Optional[Tensor], eps: float) -> Tuple[Tensor, Tensor, Tensor]:
    lib = _lib.load()
    values = _empty_rows(x, torch.int8)
    summed = _empty_rows(x) if residual is not None else x.new_empty(0)
    scales = torch.empty(x.shape[0], dtype=torch.float32, device=x.device)
    geo = _geometry_of(x, weight, residual, eps)
    rc = call_on(x.device.index, lib.oops_rms_norm_int8, geo, _ptr(x), _ptr(residual), _ptr(weight), _ptr(values),
                 _ptr(scales), _ptr(summed))  # fmt: skip
    _lib.check(rc, "rms_norm_int8")
    return values, scales, summed


def _quantize_impl(x: Tensor) -> Tuple[Tensor, Tensor]:
    lib = _lib.load()
    values = _empty_rows(x, torch.int8)
    scales = torch.empty(x.shape[0], dtype=torch.float32, device=x.device)
    geo = _geometry_of(x, None, None, 0.0)
    rc = call_on(x.device.index, lib.oops_quantize_int8, geo, _ptr(x), _ptr(values), _ptr(scales))
    _lib.check(rc, "quantize_int8")
    return values, scales


def _backward_impl(dy: Tensor, dsum: Optional[Tensor], h: Tensor, weight: Optional[Tensor], rstd: Tensor,
                   need_weight: bool) -> Tuple[Tensor, Tensor]:  # fmt: skip
    """(dx, dweight): dx is the gradient of the input and of the residual; dweight is empty where not wanted."""

    lib = _lib.load()
    rows, width = h.shape
    dy = dy.resolve_neg().contiguous()
    dsum = None if dsum is None else dsum.resolve_neg().contiguous()
    dx = _empty_rows(h)
    if rows == 0:
        return dx, torch.zeros_like(weight) if need_weight else h.new_empty(0)
    dw = torch.empty_like(weight) if need_weight else h.new_empty(0)
    f32 = weight is not None and weight.dtype == torch.float32
    ws_bytes = _workspace_bytes(lib, h.dtype, f32, rows, width) if need_weight else 0
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=h.device) if ws_bytes else None
    geo = _geometry_of(h, weight, None, 0.0)
    rc = call_on(h.device.index, lib.oops_rms_norm_backward, geo, _ptr(h), _ptr(rstd), _ptr(weight), _ptr(dy), _ptr(dsum),
                 _ptr(dx), _ptr(dw), _ptr(ws), ws_bytes)  # fmt: skip
    _lib.check(rc, "rms_norm backward")
    return dx, dw


@torch.library.custom_op("oops_amd::rms_norm_forward", mutates_args=(), device_types="cuda")
def rms_norm_forward(x: Tensor, weight: Optional[Tensor], residual: Optional[Tensor], eps: float,
                     save: bool) -> Tuple[Tensor, Tensor, Tensor]:  # fmt: skip
    """Rows ``x`` (rows, width) with unit column stride.  Returns (y, sum or empty, rstd or empty)."""

    return _forward_impl(x, weight, residual, eps, save)


@rms_norm_forward.register_fake
def _(x, weight, residual, eps, save):
    return (x.new_empty(x.shape), x.new_empty(x.shape if residual is not None else (0,)),
            x.new_empty(x.shape[0] if save else 0, dtype=torch.float32))  # fmt: skip


@torch.library.custom_op("oops_amd::rms_norm_backward", mutates_args=(), device_types="cuda")
def rms_norm_backward(dy: Tensor, dsum: Optional[Tensor], h: Tensor, weight: Optional[Tensor], rstd: Tensor,
                      need_weight: bool) -> Tuple[Tensor, Tensor]:  # fmt: skip
    return _backward_impl(dy, dsum, h, weight, rstd, need_weight)


@rms_norm_backward.register_fake
def _(dy, dsum, h, weight, rstd, need_weight):
    return h.new_empty(h.shape), torch.empty_like(weight) if need_weight else h.new_empty(0)


@torch.library.custom_op("oops_amd::rms_norm_int8", mutates_args=(), device_types="cuda")
def rms_norm_int8_forward(x: Tensor, weight: Optional[Tensor], residual: Optional[Tensor],
                          eps: float) -> Tuple[Tensor, Tensor, Tensor]:  # fmt: skip
    return _int8_impl(x, weight, residual, eps)


@rms_norm_int8_forward.register_fake
def _(x, weight, residual, eps):
    return (x.new_empty(x.shape, dtype=torch.int8), x.new_empty(x.shape[0], dtype=torch.float32),
            x.new_empty(x.shape if residual is not None else (0,)))  # fmt: skip


@torch.library.custom_op("oops_amd::quantize_int8", mutates_args=(), device_types="cuda")
def quantize_int8_forward(x: Tensor) -> Tuple[Tensor, Tensor]:
    return _quantize_impl(x)


@quantize_int8_forward.register_fake
def _(x):
    return x.new_empty(x.shape, dtype=torch.int8), x.new_empty(x.shape[0], dtype=torch.float32)


# ----------------------------------------------------------------- autograd


def _grads(ctx, dy, dsum, backward):
    """Gradients of (x, weight, residual)."""

    h, weight, rstd = ctx.saved_tensors
    need_x, need_w, need_r = ctx.needs_input_grad[:3]
    if dy is None:  # only the summed stream was used
        return dsum if need_x else None, None, dsum if need_r else None
    need_w = bool(need_w and weight is not None)
    dx, dw = backward(dy, dsum, h, weight, rstd, need_w)
    # (the input's and the residual's gradient are one tensor)
    return dx if need_x else None, dw if need_w else None, dx if need_r else None


def _setup_context(ctx, inputs, output):
    x, weight, residual, _eps, _save = inputs
    _y, summed, rstd = output
    ctx.save_for_backward(x if residual is None else summed, weight, rstd)
    ctx.has_residual = residual is not None
    ctx.mark_non_differentiable(*((rstd,) if residual is not None else (summed, rstd)))
    ctx.set_materialize_grads(False)


def _backward(ctx, dy, dsum, _drstd):
    if dy is None and dsum is None:
        return (None,) * 5
    dx, dw, dr = _grads(ctx, dy, dsum if ctx.has_residual else None, rms_norm_backward)
    # (a custom operator's gradients may not alias each other)
    return dx, dw, dr.clone() if dr is not None and dx is not None else dr, None, None


rms_norm_forward.register_autograd(_backward, setup_context=_setup_context)


class _EagerRmsNorm(torch.autograd.Function):
    """The same kernels as the custom op for eager calls: autograd calls the backward directly instead of
    through the operator dispatcher.  Traced code takes the custom op."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, summed, rstd = _forward_impl(x, weight, residual, eps, True)
        ctx.save_for_backward(x if residual is None else summed, weight, rstd)
        ctx.set_materialize_grads(False)
        if residual is None:
            ctx.mark_non_differentiable(summed)
        return y, summed

    @staticmethod
    def backward(ctx, dy, dsum):
        if dy is None and dsum is None:
            return None, None, None, None
        grads = _grads(ctx, dy, dsum, rms_norm_backward if any_wrapped(dy, dsum) else _backward_impl)
        later = any(t is not None and t.requires_grad for t in (dy, dsum))
        return (*without_second_derivative(grads, ctx, dy, differentiable=later), None)
