"""Float64 definitions of the layer operators: root-mean-square norm, 8-bit rows and products, linear attention."""

from __future__ import annotations

import numpy as np


def rms_norm_forward(h, weight=None, eps=1e-6):
    y = h / np.sqrt((h * h).mean(-1, keepdims=True) + eps)
    return y if weight is None else y * weight


def rms_norm_backward(h, dy, weight=None, eps=1e-6):
    """(dh, dweight) of ``rms_norm_forward`` over rows (R, C)."""

    rstd = 1 / np.sqrt((h * h).mean(-1, keepdims=True) + eps)
    n = h * rstd
    g = dy if weight is None else dy * weight
    return rstd * (g - n * (g * n).mean(-1, keepdims=True)), (dy * n).sum(0)


def quantize_rows(y):
    """(y * 127 / max|row| before rounding, scales); rows of zeros have scale 0."""

    top = np.abs(y).max(-1, keepdims=True)
    return np.divide(y * 127, top, out=np.zeros_like(y), where=top > 0), top[..., 0] / 127


def int8_linear(x, x_scale, w, w_scale, bias=None):
    y = (x.astype(np.int64) @ w.astype(np.int64).T) * x_scale[..., None] * w_scale
    return y if bias is None else y + bias


def _live(shape, lengths):
    """(B, L) of a padded batch, and the lengths."""

    b, _, length, _ = shape
    n = np.full(b, length) if lengths is None else np.clip(np.asarray(lengths), 0, length)
    return np.arange(length)[None] < n[:, None], n


def linear_attention_forward(q, k, v, log_decay, initial=None, lengths=None, scale=None):
    """(out, final state) token by token; q, k (B, H, L, D), v (B, H, L, E), states (B, H, D, E)."""

    b, h, length, d = q.shape
    scale = d**-0.5 if scale is None else scale
    live, _ = _live(q.shape, lengths)
    decay = np.exp(log_decay)[None, :, None, None]
    s = np.zeros((b, h, d, v.shape[-1])) if initial is None else initial.copy()
    out = np.zeros(v.shape)
    for t in range(length):
        on = live[:, t, None, None, None]
        with np.errstate(invalid="ignore"):
            s = np.where(on, decay * s + k[:, :, t, :, None] * v[:, :, t, None, :], s)
            out[:, :, t] = np.where(on[..., 0], scale * (q[:, :, t, None, :] @ s)[:, :, 0], 0)
    return out, s


def linear_attention_backward(q, k, v, log_decay, dout, dfinal=None, initial=None, lengths=None, scale=None):
    """(dq, dk, dv, dinitial) token by token, states recomputed forwards and their gradients backwards."""

    b, h, length, d = q.shape
    scale = d**-0.5 if scale is None else scale
    live, _ = _live(q.shape, lengths)
    decay = np.exp(log_decay)[None, :, None, None]
    s = np.zeros((b, h, d, v.shape[-1])) if initial is None else initial.copy()
    dq, dk, dv = np.zeros(q.shape), np.zeros(k.shape), np.zeros(v.shape)
    for t in range(length):
        on = live[:, t, None, None, None]
        s = np.where(on, decay * s + k[:, :, t, :, None] * v[:, :, t, None, :], s)
        dq[:, :, t] = np.where(on[..., 0], scale * (s @ dout[:, :, t, :, None])[..., 0], 0)
    r = np.zeros_like(s) if dfinal is None else dfinal.copy()  # the gradient of the state behind token t
    for t in reversed(range(length)):
        on = live[:, t, None, None, None]
        r = np.where(on, r + scale * q[:, :, t, :, None] * dout[:, :, t, None, :], r)
        dk[:, :, t] = np.where(on[..., 0], (r @ v[:, :, t, :, None])[..., 0], 0)
        dv[:, :, t] = np.where(on[..., 0], (k[:, :, t, None, :] @ r)[:, :, 0], 0)
        r = np.where(on, decay * r, r)
    return dq, dk, dv, r
