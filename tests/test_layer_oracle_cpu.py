"""The float64 definitions of the layer operators against differences and brute force."""

import numpy as np
import pytest

from oracle import layers


def _differences(f, x, dy, step=1e-6):
    """d<f(x), dy>/dx by central differences."""

    g = np.zeros_like(x)
    for i in np.ndindex(x.shape):
        x[i] += step
        up = (f(x) * dy).sum()
        x[i] -= 2 * step
        down = (f(x) * dy).sum()
        x[i] += step
        g[i] = (up - down) / (2 * step)
    return g


def test_rms_norm_gradients():
    rng = np.random.default_rng(0)
    h, w, dy = rng.normal(size=(3, 5)), rng.normal(size=5), rng.normal(size=(3, 5))
    dh, dw = layers.rms_norm_backward(h, dy, w)
    np.testing.assert_allclose(dh, _differences(lambda x: layers.rms_norm_forward(x, w), h, dy), atol=1e-8)
    np.testing.assert_allclose(dw, _differences(lambda x: layers.rms_norm_forward(h, x), w, dy), atol=1e-8)


def _brute(q, k, v, log_decay, initial, n, scale):
    out = np.zeros(v.shape)
    for b, h, t in np.ndindex(*q.shape[:3]):
        if t < n[b]:
            for s in range(t + 1):
                out[b, h, t] += scale * np.exp(log_decay[h] * (t - s)) * (q[b, h, t] @ k[b, h, s]) * v[b, h, s]
            out[b, h, t] += scale * np.exp(log_decay[h] * (t + 1)) * (q[b, h, t] @ initial[b, h])
    return out


@pytest.mark.parametrize("lengths", [None, [4, 0]])
def test_linear_attention(lengths):
    rng = np.random.default_rng(1)
    b, h, n, d, e = 2, 2, 5, 3, 2
    q, k = rng.normal(size=(2, b, h, n, d))
    v, do = rng.normal(size=(2, b, h, n, e))
    s0, ds = rng.normal(size=(2, b, h, d, e))
    ld = -np.array([0.3, 1.1])
    out, _ = layers.linear_attention_forward(q, k, v, ld, s0, lengths, 0.7)
    np.testing.assert_allclose(out, _brute(q, k, v, ld, s0, [n, n] if lengths is None else lengths, 0.7), atol=1e-12)

    def loss(**new):
        a = {"q": q, "k": k, "v": v, "initial": s0, **new}
        o, s = layers.linear_attention_forward(a["q"], a["k"], a["v"], ld, a["initial"], lengths, 0.7)
        return np.concatenate([(o * do).ravel(), (s * ds).ravel()])

    got = layers.linear_attention_backward(q, k, v, ld, do, ds, s0, lengths, 0.7)
    for name, x, g in zip(("q", "k", "v", "initial"), (q, k, v, s0), got):
        np.testing.assert_allclose(g, _differences(lambda x, name=name: loss(**{name: x}), x, 1.0), atol=1e-7, err_msg=name)


def test_int8_forms():
    rng = np.random.default_rng(2)
    y = rng.normal(size=(4, 9))
    y[2] = 0
    q, s = layers.quantize_rows(y)
    assert np.abs(q).max() == 127 and s[2] == 0 and not q[2].any()
    np.testing.assert_allclose(q * s[:, None], y, atol=1e-12)
    x, w = rng.integers(-128, 128, (3, 7)), rng.integers(-128, 128, (5, 7))
    xs, ws, b = rng.random(3), rng.random(5), rng.random(5)
    np.testing.assert_allclose(layers.int8_linear(x, xs, w, ws, b), (xs[:, None] * x) @ (ws[:, None] * w).T + b)
