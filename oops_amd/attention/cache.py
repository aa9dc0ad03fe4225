"""A paged key/value cache in 4 bits: ``quantized_cache``, ``cache_write``, ``cache_read`` and ``cache_attention``.

Keys and values of decoded sequences, in 4-bit floating point with one exponent for each block of 32 channels: a
quarter of bfloat16's bytes and a little more, and decoding is bound by these bytes.  The cache is a pair of tensors
that the caller owns,

    codes  uint8 (pages, G, 2, page_size, D / 2)     keys ([:, :, 0]) and values; channel 2 i is the low half of byte i
    scales uint8 (pages, G, 2, page_size, D / 32)    exponents e, 1..252: a block stands for its codes' values times
                                                     2 ** (e - 127), with 255 for NaN (0 in an empty cache)

with codes 0..7 for 0, 0.5, 1, 1.5, 2, 3, 4, 6 and 8..15 for their negatives.  Tokens have slots,
``page * page_size + place``; which page holds which part of a sequence is the caller's table.  ``cache_write`` puts keys
(behind ``rms_norm_rotary``) and values there as a prompt or a step makes them, ``cache_attention`` attends to them with
one token of each sequence, ``cache_read`` gives back what they stand for.  Kernels: csrc/cache.hip.  The reference has
no counterpart.
"""

from __future__ import annotations

import ctypes
import functools
from typing import Optional, Tuple

import torch
from torch import Tensor

from .. import _lib
from .._errors import unsupported
from ._core import SUPPORTED_DTYPES, _DTYPE_CODE, _ptr
from ._runtime import (
    call_on,
    is_nested,
    needs_custom_op,
    on_one_device,
    require_no_forward_mode,
    require_same_device,
    wants_gradient,
)
from .linear import _batched, _workspace

BLOCK = 32  # channels of a scale
HEAD_SIZES = (32, 64, 96, 128)
MAX_PAGE = 1 << 20


def quantized_cache(pages: int, heads: int, size: int, *, page_size: int = 64, device=None) -> Tuple[Tensor, Tensor]:
    r"""The ``(codes, scales)`` of an empty cache of ``pages`` pages (zeros) on ``device`` (default: the current GPU).

    ``heads``: key heads; ``size``: channels of a head, 32, 64, 96 or 128; ``page_size``: tokens of a page, a multiple
    of 16 up to 2^20.
    """

    if pages < 0 or heads < 1:
        raise ValueError(f"quantized_cache takes pages >= 0 and heads >= 1, got {pages} and {heads}")
    _check_sizes("quantized_cache", size, page_size)
    device = torch.device("cuda") if device is None else device
    shape = (pages, heads, 2, page_size)
    return tuple(torch.zeros(*shape, size // n, dtype=torch.uint8, device=device) for n in (2, BLOCK))


def cache_write(codes: Tensor, scales: Tensor, key: Tensor, value: Tensor, slots: Tensor) -> None:
    r"""Quantizes keys and values into their slots of the cache, in place; inference only.

    Args:
        codes, scales: the cache (see ``quantized_cache``), contiguous.
        key, value: CUDA float16 / bfloat16 / float32 ``(*prefix, G, L, D)``, read in place through their strides.
        slots: int32 / int64 ``(*prefix, L)``, each token's ``page * page_size + place``.  Tokens with other values
            (negative ones, say: padding) are not written; of tokens with the same slot the last is kept.

    Each block of 32 channels gets the smallest exponent with ``max|block| <= 6 * 2 ** (e - 127)``, ``e`` in 1..252, and
    the nearest codes (ties to the even one), exactly as in real arithmetic; magnitudes above ``6 * 2 ** 125`` become
    that.  A block with an infinity or a NaN gets ``e = 255`` and reads as NaN.

    A call of more than 1024 tokens takes 4 bytes for each slot of the cache as a workspace.
    """

    operator = "cache_write"
    _check_cache(operator, codes, scales, key, value, slots)
    if key.dim() < 3 or value.shape != key.shape:
        raise ValueError(f"{operator} takes key and value (*prefix, G, L, D) of one shape, got {tuple(key.shape)} and "
                         f"{tuple(value.shape)}")  # fmt: skip
    *prefix, heads, length, size = key.shape
    if (heads, size) != (codes.shape[1], codes.shape[4] * 2):
        raise ValueError(f"{operator} cache has {codes.shape[1]} heads of {codes.shape[4] * 2} channels, the keys {heads} of {size}")
    _check_slots(operator, slots, (*prefix, length))
    if key.dtype not in SUPPORTED_DTYPES or value.dtype != key.dtype:
        raise unsupported(operator, "requires half/float32 keys and values of one dtype", dtypes=(key.dtype, value.dtype))
    _require_inference(operator, key, value)
    args = (codes, scales, _batched(key, length), _batched(value, length), slots.resolve_neg().contiguous())
    if needs_custom_op(*args):
        cache_write_op(*args)
    else:
        _write_impl(*args)
        # (autograd has to know: a graph that saved the cache must not be differentiated with the new one)
        torch.autograd.graph.increment_version((codes, scales))


def cache_read(codes: Tensor, scales: Tensor, slots: Tensor, *, dtype: torch.dtype = torch.bfloat16) -> Tuple[Tensor, Tensor]:
    r"""Keys and values that slots of the cache stand for, ``(*prefix, G, L, D)`` each, rounded to ``dtype``.

    ``slots``: int32 / int64 ``(*prefix, L)`` as for ``cache_write``; others read as zeros.  Codes are exact in bfloat16
    and float32, and in float16 where its range holds them.  The results are token-major in memory.
    """

    operator = "cache_read"
    _check_cache(operator, codes, scales, slots)
    if slots.dim() < 1:
        raise ValueError(f"{operator} takes slots (*prefix, L)")
    _check_slots(operator, slots, tuple(slots.shape))
    if dtype not in SUPPORTED_DTYPES:
        raise unsupported(operator, "reads float16, bfloat16 or float32", dtype=dtype)
    args = (codes.resolve_neg(), scales.resolve_neg(), slots.resolve_neg().contiguous(), dtype)
    out = cache_read_op(*args) if needs_custom_op(*args[:3]) else _read_impl(*args)
    key, value = (t.view(*slots.shape, codes.shape[1], codes.shape[4] * 2).transpose(-2, -3) for t in out)
    return key, value


def cache_attention(
    query: Tensor,
    codes: Tensor,
    scales: Tensor,
    pages: Tensor,
    lengths: Tensor,
    *,
    scale: Optional[float] = None,
) -> Tensor:
    r"""Attention of one token of each sequence to the sequence's tokens in the cache; inference only.

    Args:
        query: CUDA float16 / bfloat16 / float32 ``(*prefix, H, D)``, ``H`` a multiple of the cache's ``G`` heads: query
            head ``h`` reads key head ``h // (H // G)``.
        codes, scales: the cache (see ``quantized_cache``), contiguous.
        pages: int32 ``(*prefix, max_pages)``: token t of a sequence is in page ``pages[..., t // page_size]`` at place
            ``t % page_size``.  Tokens of pages that the cache does not have are left out.
        lengths: int32 / int64 ``(*prefix,)`` numbers of tokens, the current one among them if it is to attend to
            itself (write it first).  Values outside ``0..max_pages * page_size`` are taken as the nearer bound.
        scale: of the scores; default ``D ** -0.5``.

    Returns ``(*prefix, H, D)`` in the query's dtype; zeros for a sequence without tokens.  What the codes stand for
    takes part exactly, weights have 16 bits or more, and sums are float32, so the result has the precision of the query's
    type.  Few sequences take less time with a page table that is not much wider than they are.
    """

    operator = "cache_attention"
    _check_cache(operator, codes, scales, query, pages, lengths)
    if query.dim() < 2 or query.shape[-1] != codes.shape[4] * 2:
        raise ValueError(f"{operator} takes query (*prefix, H, {codes.shape[4] * 2}), got {tuple(query.shape)}")
    *prefix, heads, size = query.shape
    if heads < 1 or heads % codes.shape[1]:
        raise ValueError(f"{operator} query heads must be a positive multiple of the cache's, got {heads} and {codes.shape[1]}")
    if pages.dim() < 1 or tuple(pages.shape[:-1]) != tuple(prefix) or tuple(lengths.shape) != tuple(prefix):
        raise ValueError(f"{operator} takes pages {(*prefix, 'max_pages')} and lengths {tuple(prefix)}, got "
                         f"{tuple(pages.shape)} and {tuple(lengths.shape)}")  # fmt: skip
    if query.dtype not in SUPPORTED_DTYPES or pages.dtype != torch.int32 or lengths.dtype not in (torch.int32, torch.int64):
        raise unsupported(operator, "requires a half/float32 query, int32 pages and int32 or int64 lengths",
                          dtypes=(query.dtype, pages.dtype, lengths.dtype))  # fmt: skip
    _require_inference(operator, query)
    scale = size**-0.5 if scale is None else float(scale)
    lead = lengths.numel()
    table = pages.resolve_neg().reshape(lead, pages.shape[-1]).contiguous()
    args = (_batched(query, None), codes.resolve_neg(), scales.resolve_neg(), table, lengths.resolve_neg().reshape(-1).contiguous())
    out = cache_attention_op(*args, scale) if needs_custom_op(*args) else _attention_impl(*args, scale)
    return out if len(prefix) == 1 else out.view(*prefix, heads, size)


# ----------------------------------------------------------------- checks


def _check_sizes(operator: str, size: int, page_size: int) -> None:
    if size not in HEAD_SIZES or page_size % 16 or not 0 < page_size <= MAX_PAGE:
        raise unsupported(operator, "takes heads of 32, 64, 96 or 128 channels and pages of a multiple of 16 tokens up to 2^20",
                          size=size, page_size=page_size)  # fmt: skip


def _check_cache(operator: str, codes: Tensor, scales: Tensor, *others: Tensor) -> None:
    for t in (codes, scales, *others):
        if is_nested(t):
            raise unsupported(operator, "takes dense tensors", hint="pass the packed values")
    require_no_forward_mode(operator, *others)
    if not on_one_device(codes.device, scales, *others):
        require_same_device(operator, codes, scales, *others)
    if codes.dim() != 5 or scales.dim() != 5 or codes.shape[2] != 2 or codes.shape[:4] != scales.shape[:4] \
            or codes.shape[4] * 2 != scales.shape[4] * BLOCK:  # fmt: skip
        raise ValueError(f"{operator} takes codes (pages, G, 2, page_size, D / 2) and scales (pages, G, 2, page_size, D / 32), got "
                         f"{tuple(codes.shape)} and {tuple(scales.shape)}")  # fmt: skip
    _check_sizes(operator, codes.shape[4] * 2, codes.shape[3])
    ok = codes.is_cuda and codes.dtype == scales.dtype == torch.uint8 and codes.is_contiguous() and scales.is_contiguous()
    if not ok or codes.shape[1] < 1 or codes.shape[0] * codes.shape[3] >= 2**31:
        raise unsupported(operator, "requires a CUDA cache: contiguous uint8 codes and scales of fewer than 2^31 tokens",
                          device=codes.device, dtypes=(codes.dtype, scales.dtype), shape=tuple(codes.shape),
                          contiguous=(codes.is_contiguous(), scales.is_contiguous()))  # fmt: skip


def _check_slots(operator: str, slots: Tensor, shape: tuple) -> None:
    if tuple(slots.shape) != shape:
        raise ValueError(f"{operator} slots must have shape {shape}, got {tuple(slots.shape)}")
    if slots.dtype not in (torch.int32, torch.int64):
        raise unsupported(operator, "takes slots in int32 or int64", dtype=slots.dtype)


def _require_inference(operator: str, *tensors) -> None:
    if wants_gradient(*tensors):
        raise unsupported(operator, "has no gradient", hint="call it under torch.no_grad() or on detached tensors")


# ----------------------------------------------------------------- launches


@functools.lru_cache(maxsize=512)
def _geometry(lib, dtype, cache: tuple, i64: bool, batch: int, length: int, key: tuple, value: tuple) -> tuple:
    """The launch geometry and the writing's workspace (cached: the library only reads it)."""

    pages, heads, _, page, half = cache
    g = _lib.CacheGeometry(_DTYPE_CODE[dtype], heads, half * 2, page, int(i64), pages, batch, length)
    g.stride[0][:], g.stride[1][:] = key, value
    ref = ctypes.pointer(g)
    return ref, lib.oops_cache_write_workspace_bytes(ref)


@functools.lru_cache(maxsize=512)
def _attention_geometry(lib, dtype, cache: tuple, i64: bool, batch: int, heads: int, max_pages: int, stride: tuple, scale: float):
    pages, kv_heads, _, page, half = cache
    g = _lib.CacheAttnGeometry(_DTYPE_CODE[dtype], heads, kv_heads, half * 2, page, int(i64), pages, batch, max_pages)
    g.stride[:], g.scale = stride, scale
    ref = ctypes.pointer(g)
    return ref, lib.oops_cache_attn_workspace_bytes(ref)


def _write_impl(codes: Tensor, scales: Tensor, key: Tensor, value: Tensor, slots: Tensor) -> None:
    if codes.is_neg() or scales.is_neg():
        raise unsupported("cache_write", "updates the cache in place: it must not be a lazily negated view")
    lib = _lib.load()
    geo, ws_bytes = _geometry(lib, key.dtype, tuple(codes.shape), slots.dtype == torch.int64, key.shape[0], key.shape[2],
                              key.stride()[:3], value.stride()[:3])  # fmt: skip
    ws = _workspace(ws_bytes, codes.device)
    rc = call_on(codes.device.index, lib.oops_cache_write, geo, _ptr(codes), _ptr(scales), _ptr(key), _ptr(value), _ptr(slots),
                 _ptr(ws), ws_bytes)  # fmt: skip
    _lib.check(rc, "cache_write")


def _read_impl(codes: Tensor, scales: Tensor, slots: Tensor, dtype: torch.dtype) -> Tuple[Tensor, Tensor]:
    """Keys and values (tokens, G, D)."""

    lib = _lib.load()
    tokens, heads, size = slots.numel(), codes.shape[1], codes.shape[4] * 2
    key, value = (torch.empty((tokens, heads, size), dtype=dtype, device=codes.device) for _ in range(2))
    stride = (0, size, heads * size)
    geo, _ = _geometry(lib, dtype, tuple(codes.shape), slots.dtype == torch.int64, 1, tokens, stride, stride)
    rc = call_on(codes.device.index, lib.oops_cache_read, geo, _ptr(codes), _ptr(scales), _ptr(slots), _ptr(key), _ptr(value))
    _lib.check(rc, "cache_read")
    return key, value


def _attention_impl(query: Tensor, codes: Tensor, scales: Tensor, pages: Tensor, lengths: Tensor, scale: float) -> Tensor:
    lib = _lib.load()
    out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    geo, ws_bytes = _attention_geometry(lib, query.dtype, tuple(codes.shape), lengths.dtype == torch.int64, query.shape[0],
                                        query.shape[1], pages.shape[1], query.stride()[:2], scale)  # fmt: skip
    ws = _workspace(ws_bytes, query.device)
    rc = call_on(query.device.index, lib.oops_cache_attn, geo, _ptr(query), _ptr(codes), _ptr(scales), _ptr(pages), _ptr(lengths),
                 _ptr(out), _ptr(ws), ws_bytes)  # fmt: skip
    _lib.check(rc, "cache_attention")
    return out


@torch.library.custom_op("oops_amd::cache_write", mutates_args=("codes", "scales"), device_types="cuda")
def cache_write_op(codes: Tensor, scales: Tensor, key: Tensor, value: Tensor, slots: Tensor) -> None:
    """key and value (B, G, L, D) with unit last strides, slots contiguous; the cache is updated in place."""

    _write_impl(codes, scales, key, value, slots)


@cache_write_op.register_fake
def _(codes, scales, key, value, slots):
    return None


@torch.library.custom_op("oops_amd::cache_read", mutates_args=(), device_types="cuda")
def cache_read_op(codes: Tensor, scales: Tensor, slots: Tensor, dtype: torch.dtype) -> Tuple[Tensor, Tensor]:
    return _read_impl(codes, scales, slots, dtype)


@cache_read_op.register_fake
def _(codes, scales, slots, dtype):
    shape = (slots.numel(), codes.shape[1], codes.shape[4] * 2)
    return codes.new_empty(shape, dtype=dtype), codes.new_empty(shape, dtype=dtype)


@torch.library.custom_op("oops_amd::cache_attention", mutates_args=(), device_types="cuda")
def cache_attention_op(query: Tensor, codes: Tensor, scales: Tensor, pages: Tensor, lengths: Tensor, scale: float) -> Tensor:
    """query (B, H, D) with a unit last stride, pages (B, max_pages) and lengths (B,) contiguous."""

    return _attention_impl(query, codes, scales, pages, lengths, scale)


@cache_attention_op.register_fake
def _(query, codes, scales, pages, lengths, scale):
    return query.new_empty(query.shape)
