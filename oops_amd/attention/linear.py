"""``linear_attention`` and ``linear_attention_step``: attention through a decayed state.

    S_t = exp(log_decay[h]) S_(t-1) + k_t^T v_t        o_t = scale q_t S_t

Causal attention without a softmax whose cost grows with the length and not with its square: a state of
``key_size x value_size`` for each head, decayed by the head's own factor.  ``linear_attention`` takes whole
sequences (training and prompts), forward and backward; ``linear_attention_step`` takes one token of each
sequence and updates the states in place (decoding).  Operands are head-major ``(*prefix, H, L, D)`` like
``pair_bias_attention``'s and read in place through their strides, so token-major projections are passed as
``.transpose(-2, -3)`` views and heads that share keys as expanded ones; the result feeds
``gate_attention_output``.  Kernels: csrc/linear_attn.hip.  The reference has no counterpart.
"""

from __future__ import annotations

import ctypes
import functools
from typing import List, Optional, Tuple, Union

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

MAX_HEAD_SIZE = 128
_NO_STRIDES = (0, 0, 0)


def linear_attention(
    query: Tensor,
    key: Tensor,
    value: Tensor,
    log_decay: Tensor,
    initial_state: Optional[Tensor] = None,
    lengths: Optional[Tensor] = None,
    *,
    scale: Optional[float] = None,
    return_state: bool = False,
) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    r"""Causal linear attention with a decay for each head.

    Args:
        query, key: CUDA float16 / bfloat16 / float32 ``(*prefix, H, L, D)``, ``D`` in 1..128.
        value: ``(*prefix, H, L, E)`` of the same dtype, ``E`` in 1..128.
        log_decay: float32 ``(H,)``, the natural logarithm of each head's decay, at most 0 (``-inf``: no memory).
            A constant of the model: it has no gradient.
        initial_state: optional float32 ``(*prefix, H, D, E)`` state before the first token.
        lengths: optional int32 / int64 ``(*prefix,)`` numbers of tokens of a padded batch.  Tokens behind them are
            not read; their outputs and gradients are zero.  (Values outside 0..L are taken as the nearer bound.)
        scale: of the outputs; default ``D ** -0.5``.
        return_state: also return the state behind each sequence's last token, float32 ``(*prefix, H, D, E)``,
            from which ``linear_attention_step`` or another call continues.

    Returns the outputs ``(*prefix, H, L, E)`` in the query's dtype and dimension order, or ``(out, state)``.
    Gradients reach query, key, value and ``initial_state``; second derivatives raise.

    Infinities and NaN act as in the recurrence: what they do not reach stays finite (nothing before their token or in
    other heads, and of a value's only its own column), what they reach is infinite or NaN; a head whose decay is ``-inf``
    multiplies what it forgets by zero, which is NaN for them.
    """

    operator = "linear_attention"
    _check(operator, query, key, value, log_decay, initial_state, True)
    *prefix, heads, length, d = query.shape
    e = value.shape[-1]
    if lengths is not None:
        require_same_device(operator, query, lengths)
        if tuple(lengths.shape) != tuple(prefix):
            raise ValueError(f"{operator} lengths must have the prefix shape {tuple(prefix)}, got {tuple(lengths.shape)}")
        if lengths.dtype not in (torch.int32, torch.int64):
            raise unsupported(operator, "takes lengths in int32 or int64", dtype=lengths.dtype)
        lengths = lengths.resolve_neg().reshape(-1).contiguous()
    q, k, v = _batched(query, length), _batched(key, length), _batched(value, length)
    s0 = None
    if initial_state is not None:
        s0 = initial_state.resolve_neg().reshape(q.shape[0], heads, d, e).contiguous()
    scale = d**-0.5 if scale is None else float(scale)
    ld = log_decay.resolve_neg().contiguous()
    grad = wants_gradient(query, key, value, initial_state)
    operands = (q, k, v, ld, lengths, s0)
    args = (*operands, scale, bool(return_state))
    if needs_custom_op(*operands):
        out, state = linear_attention_forward(*args)
    elif grad:
        out, state = _EagerLinearAttention.apply(*args)
    else:
        out, state = _forward_impl(*args)
    out = out if len(prefix) == 1 else out.view(*prefix, heads, length, e)
    if not return_state:
        return out
    return out, state if len(prefix) == 1 else state.view(*prefix, heads, d, e)


def linear_attention_step(
    query: Tensor, key: Tensor, value: Tensor, log_decay: Tensor, state: Tensor, *, scale: Optional[float] = None
) -> Tensor:
    r"""One token of every sequence: ``state`` is updated in place and read.

    Args:
        query, key: CUDA float16 / bfloat16 / float32 ``(*prefix, H, D)``; value: ``(*prefix, H, E)``.
        log_decay: float32 ``(H,)`` as for ``linear_attention``.
        state: contiguous float32 ``(*prefix, H, D, E)``; every state once (no overlapping memory).
        scale: default ``D ** -0.5``.

    Returns ``(*prefix, H, E)`` in the query's dtype.  Inference only.
    """

    operator = "linear_attention_step"
    _check(operator, query, key, value, log_decay, state, False)
    if wants_gradient(query, key, value, state):
        raise unsupported(operator, "has no gradient", hint="call it under torch.no_grad() or on detached tensors")
    if not state.is_contiguous():
        raise unsupported(operator, "updates the state in place: it must be contiguous", stride=state.stride())
    q, k, v = (_batched(t, None) for t in (query, key, value))
    scale = query.shape[-1] ** -0.5 if scale is None else float(scale)
    operands = (q, k, v, log_decay.resolve_neg().contiguous(), state)
    if needs_custom_op(*operands):
        out = linear_attention_step_op(*operands, scale)
    else:
        out = _step_impl(*operands, scale)
        # (autograd has to know: a graph that saved this state must not be differentiated with the new one)
        torch.autograd.graph.increment_version(state)
    return out if query.dim() == 3 else out.view(*query.shape[:-1], value.shape[-1])


# ----------------------------------------------------------------- checks


def _check(operator: str, query, key, value, log_decay, state, whole: bool) -> None:
    if is_nested(query) or is_nested(key) or is_nested(value):
        raise unsupported(operator, "takes dense tensors", hint="pad the batch and pass lengths")
    require_no_forward_mode(operator, query, key, value, log_decay, state)
    if not on_one_device(query.device, key, value, log_decay, state):
        require_same_device(operator, query, key, value, log_decay, state)
    least = 3 if whole else 2
    names = "(*prefix, H, L, D)" if whole else "(*prefix, H, D)"
    if query.dim() < least or key.shape != query.shape or value.dim() != query.dim() or value.shape[:-1] != query.shape[:-1]:
        raise ValueError(f"{operator} takes query and key {names} and a value of the same leading shape, got "
                         f"{tuple(query.shape)}, {tuple(key.shape)} and {tuple(value.shape)}")  # fmt: skip
    lead = query.shape[:-2] if whole else query.shape[:-1]  # (*prefix, H)
    heads, d, e = lead[-1], query.shape[-1], value.shape[-1]
    if tuple(log_decay.shape) != (heads,):
        raise ValueError(f"{operator} log_decay must have shape ({heads},), got {tuple(log_decay.shape)}")
    if state is not None and tuple(state.shape) != (*lead, d, e):
        raise ValueError(f"{operator} state must have shape {(*lead, d, e)}, got {tuple(state.shape)}")
    ok = (
        query.is_cuda
        and query.dtype in SUPPORTED_DTYPES
        and key.dtype == value.dtype == query.dtype
        and log_decay.dtype == torch.float32
        and (state is None or state.dtype == torch.float32)
        and 0 < d <= MAX_HEAD_SIZE
        and 0 < e <= MAX_HEAD_SIZE
        and heads > 0
    )
    if not ok:
        raise unsupported(
            operator,
            "requires CUDA half/float32 operands of one dtype, head sizes of 1..128, and float32 decays and states",
            device=query.device,
            dtypes=(query.dtype, key.dtype, value.dtype),
            head_sizes=(d, e),
            log_decay_dtype=log_decay.dtype,
            state_dtype=None if state is None else state.dtype,
        )
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise unsupported(operator, "has no gradient for log_decay", hint="pass log_decay.detach()")


def _batched(t: Tensor, length: Optional[int]) -> Tensor:
    """(B, H, L, D), or (B, H, D) for one token, with a unit last stride."""

    t = t.resolve_neg()
    tail = 3 if length is not None else 2
    if t.dim() != tail + 1:
        shape = t.shape[t.dim() - tail :]
        lead = 1
        for n in t.shape[: t.dim() - tail]:
            lead *= n
        t = t.reshape(lead, *shape)
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


# ----------------------------------------------------------------- launches


def _empty_like(t: Tensor, width: int) -> Tensor:
    """(B, H, L, width) with t's order of dimensions (expanded ones take the head-major order)."""

    return torch.empty_strided(*_dense(t.shape, t.stride(), width), dtype=t.dtype, device=t.device)


def _fake_like(t: Tensor, width: int) -> Tensor:
    """``_empty_like`` for traced code, whose sizes may be symbols: they cannot be a cache's key."""

    return torch.empty_strided(*_dense.__wrapped__(t.shape, t.stride(), width), dtype=t.dtype, device=t.device)


@functools.lru_cache(maxsize=256)
def _dense(shape: tuple, stride: tuple, width: int) -> Tuple[tuple, tuple]:
    sizes = (*shape[:-1], width)
    order = range(len(sizes) - 1)
    if not any(s == 0 and n > 1 for s, n in zip(stride, shape)):
        order = sorted(order, key=lambda i: (-stride[i] if shape[i] > 1 else 0, i))
    strides, step = [0] * len(sizes), width
    strides[-1] = 1
    for i in reversed(order):
        strides[i] = step
        step *= max(sizes[i], 1)
    return sizes, tuple(strides)


@functools.lru_cache(maxsize=512)
def _geometry(lib, dtype, shape: tuple, e: int, scale: float, i64: bool, strides: tuple) -> tuple:
    """The launch geometry and its (forward, backward) workspaces (cached: the library only reads it)."""

    b, h, n, d = shape
    g = _lib.LinearAttnGeometry()
    g.dtype, g.heads, g.key_size, g.value_size = _DTYPE_CODE[dtype], h, d, e
    g.batch, g.length, g.scale, g.lengths_i64 = b, n, scale, int(i64)
    for i, s in enumerate(strides):
        g.stride[i][:] = s
    ref = ctypes.pointer(g)
    return ref, lib.oops_linear_attn_forward_workspace_bytes(ref), lib.oops_linear_attn_backward_workspace_bytes(ref)


@functools.lru_cache(maxsize=512)
def _step_geometry(lib, dtype, shape: tuple, e: int, scale: float, q: tuple, k: tuple, v: tuple):
    b, h, d = shape
    strides = ((*q[:2], 0), (*k[:2], 0), (*v[:2], 0), (h * e, e, 0))
    return _geometry(lib, dtype, (b, h, 1, d), e, scale, False, strides)[0]


def _strides(*tensors: Optional[Tensor]) -> tuple:
    return tuple(_NO_STRIDES if t is None or t.dim() != 4 else t.stride()[:3] for t in tensors)


def _workspace(nbytes: int, device) -> Optional[Tensor]:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _is_i64(lengths: Optional[Tensor]) -> bool:
    return lengths is not None and lengths.dtype == torch.int64


def _forward_impl(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, lengths: Optional[Tensor],
                  initial: Optional[Tensor], scale: float, return_state: bool) -> Tuple[Tensor, Tensor]:  # fmt: skip
    return _forward_with_workspace(q, k, v, log_decay, lengths, initial, scale, return_state)[:2]


def _forward_with_workspace(q, k, v, log_decay, lengths, initial, scale, return_state):
    """(out, state or empty, the workspace: the states that the sequence's segments start from, or None)."""

    lib = _lib.load()
    b, h, _, d = q.shape
    e = v.shape[-1]
    out = _empty_like(q, e)
    state = torch.empty((b, h, d, e) if return_state else 0, dtype=torch.float32, device=q.device)
    geo, ws_bytes, _ = _geometry(lib, q.dtype, tuple(q.shape), e, scale, _is_i64(lengths), _strides(q, k, v, out))
    ws = _workspace(ws_bytes, q.device)
    rc = call_on(q.device.index, lib.oops_linear_attn_forward, geo, _ptr(q), _ptr(k), _ptr(v), _ptr(log_decay),
                 _ptr(lengths), _ptr(initial), _ptr(out), _ptr(state), _ptr(ws), ws_bytes)  # fmt: skip
    _lib.check(rc, "linear attention forward")
    return out, state, ws


def _backward_impl(dout: Tensor, dstate: Optional[Tensor], q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor,
                   lengths: Optional[Tensor], initial: Optional[Tensor], scale: float, needs: List[bool],
                   forward_ws: Optional[Tensor] = None) -> Tuple[Tensor, Tensor, Tensor, Tensor]:  # fmt: skip
    """(dq, dk, dv, dinitial), empty where not wanted."""

    lib = _lib.load()
    e = v.shape[-1]
    dout = dout.resolve_neg()
    if dout.stride(-1) != 1 and e > 1:
        dout = dout.contiguous()
    dstate = None if dstate is None else dstate.resolve_neg().contiguous()
    dq, dk, dv = (_empty_like(t, t.shape[-1]) if need else t.new_empty(0) for t, need in zip((q, k, v), needs))
    ds = torch.empty_like(initial) if needs[3] and initial is not None else log_decay.new_empty(0)
    geo, _, ws_bytes = _geometry(lib, q.dtype, tuple(q.shape), e, scale, _is_i64(lengths),
                                 _strides(q, k, v, None, dout, dq, dk, dv))  # fmt: skip
    ws = _workspace(ws_bytes, q.device)
    rc = call_on(q.device.index, lib.oops_linear_attn_backward, geo, _ptr(q), _ptr(k), _ptr(v), _ptr(log_decay),
                 _ptr(lengths), _ptr(initial), _ptr(forward_ws), _ptr(dout), _ptr(dstate), _ptr(dq), _ptr(dk), _ptr(dv),
                 _ptr(ds), _ptr(ws), ws_bytes)  # fmt: skip
    _lib.check(rc, "linear attention backward")
    return dq, dk, dv, ds


def _step_impl(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, state: Tensor, scale: float) -> Tensor:
    if state.is_neg():
        raise unsupported("linear_attention_step", "updates the state in place: it must not be a lazily negated view")
    lib = _lib.load()
    device = q.device
    e = v.shape[-1]
    out = torch.empty((*q.shape[:2], e), dtype=q.dtype, device=device)
    geo = _step_geometry(lib, q.dtype, q.shape, e, scale, q.stride(), k.stride(), v.stride())
    rc = call_on(device.index, lib.oops_linear_attn_step, geo, _ptr(q), _ptr(k), _ptr(v), log_decay.data_ptr(),
                 _ptr(state), _ptr(out))  # fmt: skip
    _lib.check(rc, "linear attention step")
    return out


@torch.library.custom_op("oops_amd::linear_attention_forward", mutates_args=(), device_types="cuda")
def linear_attention_forward(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, lengths: Optional[Tensor],
                             initial: Optional[Tensor], scale: float, return_state: bool) -> Tuple[Tensor, Tensor]:  # fmt: skip
    """Operands (B, H, L, .) with unit last strides.  Returns (out, final state or empty)."""

    return _forward_impl(q, k, v, log_decay, lengths, initial, scale, return_state)


@linear_attention_forward.register_fake
def _(q, k, v, log_decay, lengths, initial, scale, return_state):
    b, h, _, d = q.shape
    return _fake_like(q, v.shape[-1]), log_decay.new_empty((b, h, d, v.shape[-1]) if return_state else (0,))


@torch.library.custom_op("oops_amd::linear_attention_backward", mutates_args=(), device_types="cuda")
def linear_attention_backward(dout: Tensor, dstate: Optional[Tensor], q: Tensor, k: Tensor, v: Tensor,
                              log_decay: Tensor, lengths: Optional[Tensor], initial: Optional[Tensor], scale: float,
                              needs: List[bool]) -> Tuple[Tensor, Tensor, Tensor, Tensor]:  # fmt: skip
    return _backward_impl(dout, dstate, q, k, v, log_decay, lengths, initial, scale, needs)


@linear_attention_backward.register_fake
def _(dout, dstate, q, k, v, log_decay, lengths, initial, scale, needs):
    dq, dk, dv = (_fake_like(t, t.shape[-1]) if need else t.new_empty(0) for t, need in zip((q, k, v), needs))
    return dq, dk, dv, torch.empty_like(initial) if needs[3] and initial is not None else log_decay.new_empty(0)


@torch.library.custom_op("oops_amd::linear_attention_step", mutates_args=("state",), device_types="cuda")
def linear_attention_step_op(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, state: Tensor, scale: float) -> Tensor:
    """One token, q and k (B, H, D), v (B, H, E); state (..., D, E) contiguous, updated in place."""

    return _step_impl(q, k, v, log_decay, state, scale)


@linear_attention_step_op.register_fake
def _(q, k, v, log_decay, state, scale):
    return q.new_empty(*q.shape[:2], v.shape[-1])


# ----------------------------------------------------------------- autograd


def _save(ctx, q, k, v, log_decay, lengths, initial, scale, state, ws=None):
    ctx.save_for_backward(q, k, v, log_decay, lengths, initial, ws)
    ctx.scale = scale
    ctx.set_materialize_grads(False)
    if not state.numel():
        ctx.mark_non_differentiable(state)


def _grads(ctx, dout, dstate, traced):
    """Gradients of (q, k, v, log_decay, lengths, initial, scale, return_state)."""

    q, k, v, log_decay, lengths, initial, ws = ctx.saved_tensors
    needs = [bool(n) for n in (*ctx.needs_input_grad[:3], ctx.needs_input_grad[5])]
    if dout is None:  # only the state was used
        dout = v.new_zeros(1).expand(*q.shape[:3], v.shape[-1])
        dout = dout.contiguous() if v.shape[-1] > 1 else dout
    args = (dout, dstate, q, k, v, log_decay, lengths, initial, ctx.scale, needs)
    dq, dk, dv, ds = linear_attention_backward(*args) if traced else _backward_impl(*args, ws)
    keep = lambda g, need: g if need else None  # noqa: E731
    return (keep(dq, needs[0]), keep(dk, needs[1]), keep(dv, needs[2]), None, None,
            keep(ds, needs[3] and initial is not None), None, None)  # fmt: skip


def _setup_context(ctx, inputs, output):
    q, k, v, log_decay, lengths, initial, scale, _return_state = inputs
    _save(ctx, q, k, v, log_decay, lengths, initial, scale, output[1])


def _backward(ctx, dout, dstate):
    if dout is None and dstate is None:
        return (None,) * 8
    return _grads(ctx, dout, dstate, True)


linear_attention_forward.register_autograd(_backward, setup_context=_setup_context)


class _EagerLinearAttention(torch.autograd.Function):
    """The same kernels as the custom op for eager calls: autograd calls the backward directly instead of
    through the operator dispatcher.  Traced code takes the custom op."""

    @staticmethod
    def forward(ctx, q, k, v, log_decay, lengths, initial, scale, return_state):
        out, state, ws = _forward_with_workspace(q, k, v, log_decay, lengths, initial, scale, return_state)
        _save(ctx, q, k, v, log_decay, lengths, initial, scale, state, ws)
        return out, state

    @staticmethod
    def backward(ctx, dout, dstate):
        if dout is None and dstate is None:
            return (None,) * 8
        grads = _grads(ctx, dout, dstate, any_wrapped(dout, dstate))
        later = any(t is not None and t.requires_grad for t in (dout, dstate))
        return without_second_derivative(grads, ctx, dout, differentiable=later)
