"""``causal_attention``: softmax attention over whole prompts, grouped heads, packed sequences.

    o_i = sum_j softmax_j(scale q_i . k_j) v_j        over the tokens j <= i of i's sequence

For training and for prompts; ``cache_attention`` is its form for single tokens.  Operands are head-major
``(*prefix, H, L, D)`` like ``linear_attention``'s and read in place through their strides, so token-major projections
are passed as ``.transpose(-2, -3)`` views; the result feeds ``gate_attention_output``.  Kernels: csrc/causal_attn.hip,
csrc/causal_attn_bwd.hip.  The reference has no counterpart (its attention is neither causal nor grouped).
"""

from __future__ import annotations

import ctypes
import functools
from typing import List, Optional, Tuple

import torch
from torch import Tensor

from .. import _lib
from .._errors import unsupported
from ._core import SUPPORTED_DTYPES, _DTYPE_CODE, _ptr
from ._runtime import (
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
from .linear import _batched, _empty_like, _fake_like, _workspace

_OPERATOR = "causal_attention"
MAX_HEAD_SIZE = 128
MAX_PITCH = 1 << 24  # bytes between tokens (the kernels' 32-bit offsets in a tile)


def causal_attention(
    query: Tensor,
    key: Tensor,
    value: Tensor,
    offsets: Optional[Tensor] = None,
    *,
    scale: Optional[float] = None,
) -> Tensor:
    r"""Causal softmax attention.

    Args:
        query: CUDA float16 / bfloat16 / float32 ``(*prefix, H, L, D)``, ``D`` in 1..128.
        key: ``(*prefix, G, L, D)`` of the same dtype, ``H`` a multiple of ``G``: query head ``h`` reads key head
            ``h // (H // G)``.
        value: ``(*prefix, G, L, E)``, ``E`` in 1..128.
        offsets: optional int32 / int64 ``(N + 1,)`` non-decreasing bounds of ``N`` sequences packed along the tokens
            (of every batch element): sequence n has the tokens ``offsets[n] .. offsets[n + 1] - 1``.  Tokens outside
            all of them are not read; their outputs and gradients are zero.  (Values outside 0..L are taken as the
            nearer bound.)
        scale: of the scores; default ``D ** -0.5``.  (Magnitudes below 2^-120, 0 among them, weigh scores with 2^-120: with
            nothing, up to scores of 2^90.)

    Returns ``(*prefix, H, L, E)`` in the query's dtype and dimension order (head-major where its tokens would be 2^24 bytes
    or more apart).  Gradients reach query, key and value; second derivatives raise.

    Operands whose rows are not whole 16-byte pieces at 16-byte addresses are copied first.  Sums, statistics and
    accumulators are float32.  As operands of the next product, bfloat16's probabilities are rounded to the type,
    float16's forward ones to two terms of it (22 bits), and in the backward 16-bit types round probabilities and the
    scores' gradients, which in float16 have to stay in its range (scale the loss, as elsewhere).  float32 operands
    are three bfloat16 terms: a product is off by 2^-23 of itself at most and 2^-26 on average, where its operands are above
    2^-110 in magnitude; of smaller ones (gradients without a scaled loss, say) up to 2^-134 may be missing.  Infinities
    and NaN reach the tokens whose sum holds them, and no others: neither earlier tokens nor other sequences.  An infinity
    in a value stays one in its column of the outputs, one in an output's gradient in the value's gradient (where its
    weight is zero in float32, one or NaN); float16 and float32 calls that hold such values take up to twice the time.
    """

    _check(query, key, value, offsets)
    *prefix, heads, length, d = query.shape
    e = value.shape[-1]
    scale = d**-0.5 if scale is None else float(scale)
    # whole 16-byte pieces: columns of zeros change no score, and give columns of zeros
    unit = 16 // query.element_size()
    if d % unit:
        query, key = (torch.nn.functional.pad(t, (0, -d % unit)) for t in (query, key))
    if e % unit:
        value = torch.nn.functional.pad(value, (0, -e % unit))
    q, k, v = _batched(query, length), _batched(key, length), _batched(value, length)
    if offsets is not None:
        offsets = offsets.resolve_neg().contiguous()
    operands = (q, k, v, offsets)
    grad = wants_gradient(query, key, value)
    if needs_custom_op(*operands):
        out = causal_attention_forward(*operands, scale, grad)[0]
    elif grad:
        out = _EagerCausalAttention.apply(*operands, scale)
    else:
        out = _forward_impl(*operands, scale, False)[0]
    if e % unit:
        out = out[..., :e].clone()
    return out if len(prefix) == 1 else out.view(*prefix, heads, length, e)


# ----------------------------------------------------------------- checks


def _check(query, key, value, offsets) -> None:
    if is_nested(query) or is_nested(key) or is_nested(value):
        raise unsupported(_OPERATOR, "takes dense tensors", hint="pass the packed values and offsets")
    require_no_forward_mode(_OPERATOR, query, key, value)
    if not on_one_device(query.device, key, value, offsets):
        require_same_device(_OPERATOR, query, key, value, offsets)
    if (query.dim() < 3 or key.dim() != query.dim() or value.dim() != query.dim() or key.shape[:-3] != query.shape[:-3]
            or key.shape[-2:] != query.shape[-2:] or value.shape[:-1] != key.shape[:-1]):  # fmt: skip
        raise ValueError(f"{_OPERATOR} takes query (*prefix, H, L, D), key (*prefix, G, L, D) and value (*prefix, G, L, E), "
                         f"got {tuple(query.shape)}, {tuple(key.shape)} and {tuple(value.shape)}")  # fmt: skip
    heads, groups, d, e = query.shape[-3], key.shape[-3], query.shape[-1], value.shape[-1]
    if groups < 1 or heads < 1 or heads % groups:
        raise ValueError(f"{_OPERATOR} query heads must be a positive multiple of key heads, got {heads} and {groups}")
    if offsets is not None:
        if offsets.dim() != 1 or offsets.shape[0] < 1:
            raise ValueError(f"{_OPERATOR} offsets must have shape (sequences + 1,), got {tuple(offsets.shape)}")
        if offsets.dtype not in (torch.int32, torch.int64):
            raise unsupported(_OPERATOR, "takes offsets in int32 or int64", dtype=offsets.dtype)
    ok = (
        query.is_cuda
        and query.dtype in SUPPORTED_DTYPES
        and key.dtype == value.dtype == query.dtype
        and 0 < d <= MAX_HEAD_SIZE
        and 0 < e <= MAX_HEAD_SIZE
    )
    if not ok:
        raise unsupported(
            _OPERATOR,
            "requires CUDA half/float32 operands of one dtype and head sizes of 1..128",
            device=query.device,
            dtypes=(query.dtype, key.dtype, value.dtype),
            head_sizes=(d, e),
        )


# ----------------------------------------------------------------- launches


@functools.lru_cache(maxsize=512)
def _geometry(lib, dtype, shape: tuple, kv_heads: int, e: int, scale: float, sequences: int, i64: bool, strides: tuple) -> tuple:
    """The launch geometry and its (forward, backward) workspaces (cached: the library only reads it)."""

    b, h, n, d = shape
    g = _lib.CausalGeometry()
    g.dtype, g.heads, g.kv_heads, g.key_size, g.value_size = _DTYPE_CODE[dtype], h, kv_heads, d, e
    g.sequences, g.offsets_i64, g.scale, g.batch, g.length = sequences, int(i64), scale, b, n
    for i, s in enumerate(strides):
        g.stride[i][:] = s
    ref = ctypes.pointer(g)
    return ref, lib.oops_causal_attn_forward_workspace_bytes(ref), lib.oops_causal_attn_backward_workspace_bytes(ref)


def _strides(t: Optional[Tensor]) -> tuple:
    """Strides of batch, head and token (the library does not read those of dimensions of one element)."""

    return (0, 0, 0) if t is None or t.dim() != 4 else t.stride()[:3]


@functools.lru_cache(maxsize=1024)
def _whole_rows(shape: tuple, stride: tuple, el: int) -> bool:
    """Whether rows are dense and whole 16-byte pieces apart, tokens not too far."""

    if stride[3] != 1 and shape[3] > 1:
        return False
    return all(n <= 1 or s * el % 16 == 0 for n, s in zip(shape[:3], stride)) and (shape[2] <= 1 or stride[2] * el < MAX_PITCH)


def _whole(t: Tensor) -> Tensor:
    """``t``, or a copy of it whose rows are whole 16-byte pieces at 16-byte addresses."""

    if t.data_ptr() % 16 or not _whole_rows(t.shape, t.stride(), t.element_size()):
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _result_like(t: Tensor, width: int, empty_like=_empty_like) -> Tensor:
    """A result with ``t``'s order of dimensions, unless its tokens would then lie too far apart."""

    out = empty_like(t, width)
    if out.shape[2] > 1 and out.stride(2) * out.element_size() >= MAX_PITCH:
        return torch.empty(out.shape, dtype=out.dtype, device=out.device)
    return out


def _call_geometry(lib, q, k, v, offsets, scale, *others) -> tuple:
    sequences = 0 if offsets is None else offsets.shape[0] - 1
    return _geometry(lib, q.dtype, q.shape, k.shape[1], v.shape[-1], scale, sequences,
                     offsets is not None and offsets.dtype == torch.int64,
                     (*(t.stride()[:3] for t in (q, k, v)), *map(_strides, others)))  # fmt: skip


def _forward_impl(q: Tensor, k: Tensor, v: Tensor, offsets: Optional[Tensor], scale: float,
                  save: bool) -> Tuple[Tensor, Tensor, Tensor]:  # fmt: skip
    """(out, its rounding's remainder, lse); the last two are empty where no backward follows, the second in float32."""

    lib = _lib.load()
    out = _result_like(q, v.shape[-1])
    q, k, v = _whole(q), _whole(k), _whole(v)
    low = torch.empty_like(out) if save and out.dtype != torch.float32 else out.new_empty(0)
    lse = torch.empty(q.shape[:3] if save else 0, dtype=torch.float32, device=q.device)
    geo, ws_bytes, _ = _call_geometry(lib, q, k, v, offsets, scale, out)
    ws = _workspace(ws_bytes, q.device)
    rc = call_on(q.device.index, lib.oops_causal_attn_forward, geo, _ptr(q), _ptr(k), _ptr(v), _ptr(offsets), _ptr(out),
                 _ptr(low), _ptr(lse), _ptr(ws), ws_bytes)  # fmt: skip
    _lib.check(rc, "causal attention forward")
    return out, low, lse


def _backward_impl(dout: Tensor, q: Tensor, k: Tensor, v: Tensor, offsets: Optional[Tensor], out: Tensor, low: Tensor,
                   lse: Tensor, scale: float, needs: List[bool]) -> Tuple[Tensor, Tensor, Tensor]:  # fmt: skip
    """(dq, dk, dv), empty where not wanted."""

    lib = _lib.load()
    dq, dk, dv = (_result_like(t, t.shape[-1]) if need else t.new_empty(0) for t, need in zip((q, k, v), needs))
    q, k, v, dout = _whole(q), _whole(k), _whole(v), _whole(dout.resolve_neg())
    geo, _, ws_bytes = _call_geometry(lib, q, k, v, offsets, scale, out, dout, dq, dk, dv)
    ws = _workspace(ws_bytes, q.device)
    rc = call_on(q.device.index, lib.oops_causal_attn_backward, geo, _ptr(q), _ptr(k), _ptr(v), _ptr(offsets), _ptr(out),
                 _ptr(low), _ptr(lse), _ptr(dout), _ptr(dq), _ptr(dk), _ptr(dv), _ptr(ws), ws_bytes)  # fmt: skip
    _lib.check(rc, "causal attention backward")
    return dq, dk, dv


@torch.library.custom_op("oops_amd::causal_attention_forward", mutates_args=(), device_types="cuda")
def causal_attention_forward(q: Tensor, k: Tensor, v: Tensor, offsets: Optional[Tensor], scale: float,
                             save: bool) -> Tuple[Tensor, Tensor, Tensor]:  # fmt: skip
    """Operands (B, H, L, .) with unit last strides.  Returns (out, its rounding's remainder or empty, lse or empty)."""

    return _forward_impl(q, k, v, offsets, scale, save)


@causal_attention_forward.register_fake
def _(q, k, v, offsets, scale, save):
    out = _result_like(q, v.shape[-1], _fake_like)
    low = torch.empty_like(out) if save and q.dtype != torch.float32 else out.new_empty(0)
    return out, low, q.new_empty(q.shape[:3] if save else (0,), dtype=torch.float32)


@torch.library.custom_op("oops_amd::causal_attention_backward", mutates_args=(), device_types="cuda")
def causal_attention_backward(dout: Tensor, q: Tensor, k: Tensor, v: Tensor, offsets: Optional[Tensor], out: Tensor,
                              low: Tensor, lse: Tensor, scale: float,
                              needs: List[bool]) -> Tuple[Tensor, Tensor, Tensor]:  # fmt: skip
    return _backward_impl(dout, q, k, v, offsets, out, low, lse, scale, needs)


@causal_attention_backward.register_fake
def _(dout, q, k, v, offsets, out, low, lse, scale, needs):
    return tuple(_result_like(t, t.shape[-1], _fake_like) if need else t.new_empty(0) for t, need in zip((q, k, v), needs))


# ----------------------------------------------------------------- autograd


def _grads(ctx, dout, backward):
    q, k, v, offsets, out, low, lse = ctx.saved_tensors
    needs = [bool(n) for n in ctx.needs_input_grad[:3]]
    grads = backward(dout, q, k, v, offsets, out, low, lse, ctx.scale, needs)
    return tuple(g if need else None for g, need in zip(grads, needs))


def _setup_context(ctx, inputs, output):
    q, k, v, offsets, scale, _save = inputs
    out, low, lse = output
    ctx.save_for_backward(q, k, v, offsets, out, low, lse)
    ctx.scale = scale
    ctx.mark_non_differentiable(low, lse)
    ctx.set_materialize_grads(False)


def _backward(ctx, dout, _dlow, _dlse):
    if dout is None:
        return (None,) * 6
    return (*_grads(ctx, dout, causal_attention_backward), None, None, None)


causal_attention_forward.register_autograd(_backward, setup_context=_setup_context)


class _EagerCausalAttention(torch.autograd.Function):
    """The same kernels as the custom op for eager calls: autograd calls the backward directly instead of
    through the operator dispatcher.  Traced code takes the custom op."""

    @staticmethod
    def forward(ctx, q, k, v, offsets, scale):
        out, low, lse = _forward_impl(q, k, v, offsets, scale, True)
        ctx.save_for_backward(q, k, v, offsets, out, low, lse)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return out

    @staticmethod
    def backward(ctx, dout):
        if dout is None:
            return (None,) * 5
        grads = _grads(ctx, dout, causal_attention_backward if any_wrapped(dout) else _backward_impl)
        return (*without_second_derivative(grads, ctx, dout, differentiable=dout.requires_grad), None, None)
