"""``rms_norm_rotary``: the norm of queries and keys for each head, and the rotation by their position, in one pass.

    n = x * (mean(x^2) + eps)^-1/2 * weight                                  over the head's channels
    y_i = n_i cos - n_(i + R/2) sin,   y_(i + R/2) = n_(i + R/2) cos + n_i sin      (i < R/2),   y_i = n_i  (i >= R)

What a decoder layer does between its projections and ``causal_attention`` (or ``cache_write`` and ``cache_attention``).
Operands are head-major ``(*prefix, H, L, D)`` like the attention's and read in place through their strides.  Angles come
from a table that a program makes once (``rotary_table``, or its own frequencies).  Kernels: csrc/rotary.hip.  The
reference has no counterpart.
"""

from __future__ import annotations

import ctypes
import functools
from typing import List, Optional, Tuple

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
from ..attention.linear import _batched, _empty_like, _fake_like, _workspace
from .layer_norm import _ptr
from .rms_norm import _DTYPE_CODE

_OPERATOR = "rms_norm_rotary"
MAX_HEAD_SIZE = 256


def rotary_table(length: int, size: int, base: float = 10000.0, *, device=None) -> Tensor:
    r"""Cosines and sines of the angles ``p * base ** (-2 i / size)`` for positions p below ``length`` and pairs i below
    ``size / 2``: float32 ``(length, 2, size / 2)`` on ``device`` (default: the current GPU).

    Angles are float64, so far positions keep their phase; values are rounded once.
    """

    if length < 0 or size < 0 or size % 2:
        raise ValueError(f"rotary_table takes length >= 0 and an even size, got {length} and {size}")
    device = torch.device("cuda") if device is None else device
    pairs = torch.arange(size // 2, dtype=torch.float64, device=device)
    angles = torch.arange(length, dtype=torch.float64, device=device)[:, None] * float(base) ** (-2 * pairs / max(size, 1))
    return torch.stack((angles.cos(), angles.sin()), 1).float()


def rms_norm_rotary(
    query: Tensor,
    key: Tensor,
    table: Tensor,
    positions: Optional[Tensor] = None,
    query_weight: Optional[Tensor] = None,
    key_weight: Optional[Tensor] = None,
    eps: float = 1e-6,
) -> Tuple[Tensor, Tensor]:
    r"""Norm over each head's channels and rotation by the tokens' positions, of queries and keys.

    Args:
        query: CUDA float16 / bfloat16 / float32 ``(*prefix, H, L, D)``, ``D`` in 1..256.
        key: ``(*prefix, G, L, D)`` of the same dtype.
        table: float32 ``(P, 2, R / 2)``, cosines and sines for each position (see ``rotary_table``), ``R <= D``: the
            first R channels are rotated, channel i with i + R / 2.  A constant of the model: it has no gradient.
        positions: optional int32 / int64, ``(*prefix, L)`` or what expands to it; default 0, 1, ... .  (Values outside
            the table are taken as the nearer end.)
        query_weight, key_weight: optional ``(D,)`` in the operands' dtype or float32.
        eps: added to the mean square before the reciprocal square root.

    Returns ``(query, key)`` of the operands' shapes, dtype and dimension order; everything between is float32.
    Gradients reach both operands and both weights; second derivatives raise.
    """

    weights = (query_weight, key_weight)
    _check(query, key, table, positions, weights)
    *prefix, _, length, _ = query.shape
    if positions is not None:
        positions = positions.resolve_neg().expand(*prefix, length).reshape(-1).contiguous()
    elif table.shape[0] < length:
        raise ValueError(f"{_OPERATOR} table has {table.shape[0]} positions for {length} tokens")
    q, k = _batched(query, length), _batched(key, length)
    operands = (q, k, table.resolve_neg().contiguous(), positions, *(None if w is None else w.resolve_neg().contiguous() for w in weights))
    if needs_custom_op(*operands):
        yq, yk = rms_norm_rotary_forward(*operands, float(eps))
    elif wants_gradient(query, key, *weights):
        yq, yk = _EagerRotary.apply(*operands, float(eps))
    else:
        yq, yk = _forward_impl(*operands, float(eps))
    return (yq, yk) if len(prefix) == 1 else (yq.view(query.shape), yk.view(key.shape))


# ----------------------------------------------------------------- checks


def _check(query, key, table, positions, weights) -> None:
    if is_nested(query) or is_nested(key):
        raise unsupported(_OPERATOR, "takes dense tensors", hint="pass the packed values and their positions")
    require_no_forward_mode(_OPERATOR, query, key, table, *weights)
    if not on_one_device(query.device, key, table, positions, *weights):
        require_same_device(_OPERATOR, query, key, table, positions, *weights)
    if query.dim() < 3 or key.dim() != query.dim() or key.shape[:-3] != query.shape[:-3] or key.shape[-2:] != query.shape[-2:]:
        raise ValueError(f"{_OPERATOR} takes query (*prefix, H, L, D) and key (*prefix, G, L, D), got {tuple(query.shape)} and "
                         f"{tuple(key.shape)}")  # fmt: skip
    size, lead = query.shape[-1], (*query.shape[:-3], query.shape[-2])
    if table.dim() != 3 or table.shape[1] != 2 or 2 * table.shape[2] > size:
        raise ValueError(f"{_OPERATOR} table must have shape (positions, 2, R / 2) with R at most {size}, got {tuple(table.shape)}")
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64):
            raise unsupported(_OPERATOR, "takes positions in int32 or int64", dtype=positions.dtype)
        if positions.dim() > len(lead) or any(p not in (1, n) for p, n in zip(positions.shape[::-1], lead[::-1])):
            raise ValueError(f"{_OPERATOR} positions must expand to {tuple(lead)}, got {tuple(positions.shape)}")
        if table.shape[0] < 1 and query.shape[-2]:
            raise ValueError(f"{_OPERATOR} table has no positions")
    ok = (
        query.is_cuda
        and query.dtype in _DTYPE_CODE
        and key.dtype == query.dtype
        and table.dtype == torch.float32
        and 0 < size <= MAX_HEAD_SIZE
        and query.shape[-3] > 0
        and key.shape[-3] > 0
        and max(query.numel(), key.numel()) // size < 2**31
        and all(w is None or (tuple(w.shape) == (size,) and w.dtype in (query.dtype, torch.float32)) for w in weights)
    )
    if not ok:
        raise unsupported(
            _OPERATOR,
            "requires CUDA half/float32 operands of one dtype with heads of 1..256 channels, a float32 table and matching weights "
            "in their dtype or float32",
            device=query.device,
            dtypes=(query.dtype, key.dtype),
            table_dtype=table.dtype,
            shapes=(tuple(query.shape), tuple(key.shape)),
            weights=tuple(None if w is None else (tuple(w.shape), w.dtype) for w in weights),
        )
    if table.requires_grad and torch.is_grad_enabled():
        raise unsupported(_OPERATOR, "has no gradient for the table", hint="pass table.detach()")


# ----------------------------------------------------------------- launches


@functools.lru_cache(maxsize=512)
def _geometry(lib, dtype, batch: int, heads: tuple, length: int, size: int, table: tuple, i64: bool, weight_f32: tuple, eps: float,
              strides: tuple) -> tuple:  # fmt: skip
    """The launch geometry and the backward's workspace (cached: the library only reads it)."""

    g = _lib.RotaryGeometry()
    g.dtype, g.size, g.rotary, g.positions_i64 = _DTYPE_CODE[dtype], size, 2 * table[1], int(i64)
    g.heads[:], g.weight_f32[:] = heads, weight_f32
    g.batch, g.length, g.table_rows, g.eps = batch, length, table[0], eps
    for i, operand in enumerate(strides):
        for j, s in enumerate(operand):
            g.stride[i][j][:] = s
    ref = ctypes.pointer(g)
    return ref, lib.oops_rms_norm_rotary_backward_workspace_bytes(ref)


def _strides(t: Optional[Tensor]) -> tuple:
    return (0, 0, 0) if t is None or t.dim() != 4 else t.stride()[:3]


def _call_geometry(lib, q, k, table, positions, wq, wk, eps, *pairs) -> tuple:
    f32 = tuple(int(w is not None and w.dtype == torch.float32) for w in (wq, wk))
    strides = tuple((_strides(a), _strides(b)) for a, b in ((q, k), *pairs))
    return _geometry(lib, q.dtype, q.shape[0], (q.shape[1], k.shape[1]), q.shape[2], q.shape[3], (table.shape[0], table.shape[2]),
                     positions is not None and positions.dtype == torch.int64, f32, eps, strides)  # fmt: skip


def _forward_impl(q: Tensor, k: Tensor, table: Tensor, positions: Optional[Tensor], wq: Optional[Tensor], wk: Optional[Tensor],
                  eps: float) -> Tuple[Tensor, Tensor]:  # fmt: skip
    lib = _lib.load()
    yq, yk = _empty_like(q, q.shape[-1]), _empty_like(k, k.shape[-1])
    geo, _ = _call_geometry(lib, q, k, table, positions, wq, wk, eps, (yq, yk))
    rc = call_on(q.device.index, lib.oops_rms_norm_rotary_forward, geo, _ptr(q), _ptr(k), _ptr(wq), _ptr(wk), _ptr(table),
                 _ptr(positions), _ptr(yq), _ptr(yk))  # fmt: skip
    _lib.check(rc, "rms_norm_rotary forward")
    return yq, yk


def _backward_impl(dyq: Optional[Tensor], dyk: Optional[Tensor], q: Tensor, k: Tensor, table: Tensor, positions: Optional[Tensor],
                   wq: Optional[Tensor], wk: Optional[Tensor], eps: float,
                   needs: List[bool]) -> Tuple[Tensor, Tensor, Tensor, Tensor]:  # fmt: skip
    """Gradients of (q, k, query weight, key weight), empty where not wanted."""

    lib = _lib.load()
    dyq, dyk = (None if t is None else t.resolve_neg() for t in (dyq, dyk))
    dyq, dyk = (t.contiguous() if t is not None and t.stride(-1) != 1 and t.shape[-1] > 1 else t for t in (dyq, dyk))
    dq, dk = (_empty_like(t, t.shape[-1]) if need else t.new_empty(0) for t, need in zip((q, k), needs))
    empty = q.shape[0] * q.shape[2] == 0
    make = torch.zeros_like if empty else torch.empty_like
    dwq, dwk = (make(w) if need else q.new_empty(0) for w, need in zip((wq, wk), needs[2:]))
    if empty:
        return dq, dk, dwq, dwk
    geo, ws_bytes = _call_geometry(lib, q, k, table, positions, wq, wk, eps, (None, None), (dyq, dyk), (dq, dk))
    ws_bytes = ws_bytes if needs[2] or needs[3] else 0
    ws = _workspace(ws_bytes, q.device)
    rc = call_on(q.device.index, lib.oops_rms_norm_rotary_backward, geo, _ptr(q), _ptr(k), _ptr(wq), _ptr(wk), _ptr(table),
                 _ptr(positions), _ptr(dyq), _ptr(dyk), _ptr(dq), _ptr(dk), _ptr(dwq), _ptr(dwk), _ptr(ws), ws_bytes)  # fmt: skip
    _lib.check(rc, "rms_norm_rotary backward")
    return dq, dk, dwq, dwk


@torch.library.custom_op("oops_amd::rms_norm_rotary_forward", mutates_args=(), device_types="cuda")
def rms_norm_rotary_forward(q: Tensor, k: Tensor, table: Tensor, positions: Optional[Tensor], wq: Optional[Tensor],
                            wk: Optional[Tensor], eps: float) -> Tuple[Tensor, Tensor]:  # fmt: skip
    """q and k (B, H, L, D) with unit last strides; table, positions (B * L,) and weights contiguous."""

    return _forward_impl(q, k, table, positions, wq, wk, eps)


@rms_norm_rotary_forward.register_fake
def _(q, k, table, positions, wq, wk, eps):
    return _fake_like(q, q.shape[-1]), _fake_like(k, k.shape[-1])


@torch.library.custom_op("oops_amd::rms_norm_rotary_backward", mutates_args=(), device_types="cuda")
def rms_norm_rotary_backward(dyq: Optional[Tensor], dyk: Optional[Tensor], q: Tensor, k: Tensor, table: Tensor,
                             positions: Optional[Tensor], wq: Optional[Tensor], wk: Optional[Tensor], eps: float,
                             needs: List[bool]) -> Tuple[Tensor, Tensor, Tensor, Tensor]:  # fmt: skip
    return _backward_impl(dyq, dyk, q, k, table, positions, wq, wk, eps, needs)


@rms_norm_rotary_backward.register_fake
def _(dyq, dyk, q, k, table, positions, wq, wk, eps, needs):
    dq, dk = (_fake_like(t, t.shape[-1]) if need else t.new_empty(0) for t, need in zip((q, k), needs))
    dwq, dwk = (torch.empty_like(w) if need else q.new_empty(0) for w, need in zip((wq, wk), needs[2:]))
    return dq, dk, dwq, dwk


# ----------------------------------------------------------------- autograd


def _save(ctx, q, k, table, positions, wq, wk, eps):
    ctx.save_for_backward(q, k, table, positions, wq, wk)
    ctx.eps = eps
    ctx.set_materialize_grads(False)


def _grads(ctx, dyq, dyk, backward):
    """Gradients of (q, k, table, positions, query weight, key weight, eps)."""

    q, k, table, positions, wq, wk = ctx.saved_tensors
    need_q, need_k, _, _, need_wq, need_wk = ctx.needs_input_grad[:6]
    needs = [bool(need_q and dyq is not None), bool(need_k and dyk is not None),
             bool(need_wq and dyq is not None), bool(need_wk and dyk is not None)]  # fmt: skip
    grads = backward(dyq, dyk, q, k, table, positions, wq, wk, ctx.eps, needs)
    dq, dk, dwq, dwk = (g if need else None for g, need in zip(grads, needs))
    return dq, dk, None, None, dwq, dwk, None


def _setup_context(ctx, inputs, output):
    _save(ctx, *inputs)


def _backward(ctx, dyq, dyk):
    if dyq is None and dyk is None:
        return (None,) * 7
    return _grads(ctx, dyq, dyk, rms_norm_rotary_backward)


rms_norm_rotary_forward.register_autograd(_backward, setup_context=_setup_context)


class _EagerRotary(torch.autograd.Function):
    """The same kernels as the custom op for eager calls: autograd calls the backward directly instead of
    through the operator dispatcher.  Traced code takes the custom op."""

    @staticmethod
    def forward(ctx, q, k, table, positions, wq, wk, eps):
        _save(ctx, q, k, table, positions, wq, wk, eps)
        return _forward_impl(q, k, table, positions, wq, wk, eps)

    @staticmethod
    def backward(ctx, dyq, dyk):
        if dyq is None and dyk is None:
            return (None,) * 7
        grads = _grads(ctx, dyq, dyk, rms_norm_rotary_backward if any_wrapped(dyq, dyk) else _backward_impl)
        later = any(t is not None and t.requires_grad for t in (dyq, dyk))
        return without_second_derivative(grads, ctx, dyq, differentiable=later)
