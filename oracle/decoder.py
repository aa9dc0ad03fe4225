"""Float64 definitions of softmax attention in a decoder: norm and rotation, causal attention, the 4-bit cache."""

from __future__ import annotations

import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
BLOCK = 32


def rotate(x, cos, sin, back=False):
    """Channels i and i + R / 2 of x (..., L, D) turned by their token's angle (cos, sin: (..., L, R / 2)), or back."""

    half = cos.shape[-1]
    a, b = x[..., :half], x[..., half : 2 * half]
    s = -sin if back else sin
    return np.concatenate((a * cos - b * s, b * cos + a * s, x[..., 2 * half :]), -1)


def norm_rotary_forward(x, cos, sin, weight=None, eps=1e-6):
    n = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    return rotate(n if weight is None else n * weight, cos, sin)


def norm_rotary_backward(x, cos, sin, dy, weight=None, eps=1e-6):
    """(dx, dweight) of x (B, H, L, D)."""

    rstd = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    n = x * rstd
    g = rotate(dy, cos, sin, back=True)
    dw = (g * n).sum((0, 1, 2))
    g = g if weight is None else g * weight
    return rstd * (g - n * (g * n).mean(-1, keepdims=True)), dw


def causal_pairs(length, offsets=None):
    """(L, L): whether query i is paired with key j."""

    i = np.arange(length)
    pair = i[:, None] >= i[None]
    if offsets is not None:
        o = np.clip(np.asarray(offsets), 0, length)
        seq = np.searchsorted(o, i, side="right") - 1
        inside = (seq >= 0) & (seq < len(o) - 1)
        pair &= (seq[:, None] == seq[None]) & inside[:, None]
    return pair


def causal_weights(q, k, scale, offsets=None):
    """Probabilities (B, H, L, L); rows without keys are zero."""

    pair = causal_pairs(q.shape[2], offsets)
    k = np.repeat(k, q.shape[1] // k.shape[1], 1)
    s = np.where(pair, scale * (q @ np.swapaxes(k, -1, -2)), -np.inf)
    top = s.max(-1, keepdims=True, initial=-np.inf)
    p = np.exp(s - np.where(np.isfinite(top), top, 0))
    total = p.sum(-1, keepdims=True)
    return np.divide(p, total, out=np.zeros_like(p), where=total > 0)


def causal_forward(q, k, v, scale, offsets=None):
    return causal_weights(q, k, scale, offsets) @ np.repeat(v, q.shape[1] // v.shape[1], 1)


def _groups(t, heads):
    b, h, n, d = t.shape
    return t.reshape(b, heads, h // heads, n, d).sum(2)


def causal_backward(q, k, v, do, scale, offsets=None):
    r = q.shape[1] // k.shape[1]
    p = causal_weights(q, k, scale, offsets)
    kk, vv = np.repeat(k, r, 1), np.repeat(v, r, 1)
    dp = do @ np.swapaxes(vv, -1, -2)
    ds = p * (dp - (p * dp).sum(-1, keepdims=True))
    t = lambda a: np.swapaxes(a, -1, -2)  # noqa: E731
    return scale * ds @ kk, _groups(scale * t(ds) @ q, k.shape[1]), _groups(t(p) @ do, k.shape[1])


def quantize(x):
    """Codes (..., D) and exponent bytes (..., D / 32) of x: the smallest exponent in 1..252 with max|block| <= 6 times
    its power of two, the nearest of the grid's points (ties to the even code), blocks that are not finite as 255."""

    b = x.reshape(*x.shape[:-1], -1, BLOCK)
    top = np.abs(b).max(-1)
    fine = np.isfinite(top)
    e = np.full(top.shape, 1)
    for _ in range(251):
        e += fine & (top > 6 * np.exp2(e - 127.0)) & (e < 252)
    a = np.where(fine[..., None], np.abs(b), 0) / np.exp2(e - 127.0)[..., None]
    a = np.minimum(a, 6)
    dist = np.abs(a[..., None] - GRID)
    # (an odd code has to be strictly nearer)
    code = np.argmin(np.where(np.arange(8) % 2 == 0, dist, np.nextafter(dist, np.inf)), -1)
    code = np.where(fine[..., None], code + 8 * (np.signbit(b)), 0)
    return code.reshape(x.shape).astype(np.uint8), np.where(fine, e, 255).astype(np.uint8)


def values(code, e):
    v = GRID[code & 7] * np.where(code >= 8, -1.0, 1.0)
    scale = np.where(e == 255, np.nan, np.exp2(e.astype(float) - 127))
    return v * np.repeat(scale, BLOCK, -1)


def cache_values(codes, scales):
    """What a cache's codes (..., D / 2) stand for, (..., D)."""

    code = np.stack((codes & 15, codes >> 4), -1).reshape(*codes.shape[:-1], 2 * codes.shape[-1])
    return values(code, scales)


def cache_attention(q, kv, pages, lengths, scale):
    """q (B, H, D) over kv (pages, G, 2, page, D), pages (B, max_pages), lengths (B,)."""

    out = np.zeros(q.shape)
    count, groups, _, page, d = kv.shape
    r = q.shape[1] // groups
    for b in range(q.shape[0]):
        t = np.arange(min(max(lengths[b], 0), pages.shape[1] * page))
        ids = pages[b][t // page]
        keep = (ids >= 0) & (ids < count)
        t, ids = t[keep], ids[keep]
        if not len(t):
            continue
        for h in range(q.shape[1]):
            k, v = kv[ids, h // r, 0, t % page], kv[ids, h // r, 1, t % page]
            s = scale * (k @ q[b, h])
            p = np.exp(s - s.max())
            out[b, h] = p @ v / p.sum()
    return out
