"""The float64 definitions of the decoder's attention against differences, brute force and torch."""

import numpy as np
import pytest
import torch

from oracle import decoder
from test_layer_oracle_cpu import _differences


def test_norm_rotary():
    rng = np.random.default_rng(0)
    x, dy, w = rng.normal(size=(2, 2, 3, 6)), rng.normal(size=(2, 2, 3, 6)), rng.normal(size=6)
    angle = rng.normal(size=(2, 1, 3, 2))
    cos, sin = np.cos(angle), np.sin(angle)
    y = decoder.norm_rotary_forward(x, cos, sin, w)
    n = x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6) * w
    turned = (n[..., :2] + 1j * n[..., 2:4]) * np.exp(1j * angle)
    np.testing.assert_allclose(y, np.concatenate((turned.real, turned.imag, n[..., 4:]), -1), atol=1e-12)
    dx, dw = decoder.norm_rotary_backward(x, cos, sin, dy, w)
    np.testing.assert_allclose(dx, _differences(lambda t: decoder.norm_rotary_forward(t, cos, sin, w), x, dy), atol=1e-7)
    np.testing.assert_allclose(dw, _differences(lambda t: decoder.norm_rotary_forward(x, cos, sin, t), w, dy), atol=1e-7)


@pytest.mark.parametrize("offsets", [None, [0, 1, 1, 4, 7], [2, 5]])
def test_causal_attention(offsets):
    rng = np.random.default_rng(1)
    q, do = rng.normal(size=(1, 4, 7, 3)), rng.normal(size=(1, 4, 7, 2))
    k, v = rng.normal(size=(1, 2, 7, 3)), rng.normal(size=(1, 2, 7, 2))
    out = decoder.causal_forward(q, k, v, 0.7, offsets)
    want = np.zeros(out.shape)
    for lo, hi in zip((offsets or [0, 7])[:-1], (offsets or [0, 7])[1:]):
        for h in range(4):
            for i in range(lo, hi):
                w = np.exp(0.7 * k[0, h // 2, lo : i + 1] @ q[0, h, i])
                want[0, h, i] = w @ v[0, h // 2, lo : i + 1] / w.sum()
    np.testing.assert_allclose(out, want, atol=1e-12)
    got = decoder.causal_backward(q, k, v, do, 0.7, offsets)
    for name, x, g in zip("qkv", (q, k, v), got):
        f = lambda t, name=name: decoder.causal_forward(*({"q": q, "k": k, "v": v} | {name: t}).values(), 0.7, offsets)  # noqa: E731
        np.testing.assert_allclose(g, _differences(f, x, do), atol=1e-7, err_msg=name)


def test_quantized_blocks():
    rng = np.random.default_rng(2)
    x = rng.normal(size=(50, 64)) * np.exp2(rng.integers(-20, 20, size=(50, 1)))
    x[0] = 0
    x[1, :32] = 6.0  # the largest code at its border
    x[2, :32] = np.nextafter(6.0, 7)
    x[3, 3], x[4, 40] = np.inf, np.nan
    x[5, :10] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -2.5, 6]  # ties, exponent 127
    x[5, 10:32] = 0
    code, e = decoder.quantize(x)
    assert e[0].tolist() == [1, 1] and e[1, 0] == 127 and e[2, 0] == 128 and e[3, 0] == 255 and e[4, 1] == 255
    np.testing.assert_array_equal(decoder.values(code, e)[5, :10], [0, 1, 1, 2, 2, 4, 4, 0, -2, 6])
    fine = np.isfinite(x).reshape(50, 2, 32).all(-1)
    y = decoder.values(code, e)
    assert np.isnan(y.reshape(50, 2, 32)[~fine]).all()
    # half the distance to the next point: a quarter of the scale below 2, half below 4, one below 6
    unit = np.repeat(np.exp2(e - 127.0), 32, -1)
    a = np.abs(x) / unit
    step = np.where(a < 2, 0.25, np.where(a < 4, 0.5, 1.0))
    ok = np.repeat(fine, 32, -1)
    assert (np.abs(y - x)[ok] <= (step * unit)[ok]).all()
    # no smaller exponent would hold the block
    top = np.abs(x).reshape(50, 2, 32).max(-1)
    assert (top[fine] <= 6 * np.exp2(e - 127.0)[fine]).all() and ((top > 6 * np.exp2(e - 128.0)) | (e == 1))[fine].all()


def test_cache_attention():
    rng = np.random.default_rng(3)
    kv = rng.normal(size=(4, 2, 2, 16, 8))
    q = rng.normal(size=(3, 4, 8))
    pages = np.array([[2, 0], [1, 9], [3, 3]])
    out = decoder.cache_attention(q, kv, pages, [20, 30, 0], 0.5)
    k = torch.from_numpy(np.concatenate((kv[2], kv[0][:, :, :4]), 2))
    want = torch.softmax(torch.from_numpy(q[0]).view(2, 2, 8) @ k[:, 0].transpose(1, 2) * 0.5, -1) @ k[:, 1]
    np.testing.assert_allclose(out[0], want.view(4, 8).numpy(), atol=1e-12)
    k = torch.from_numpy(kv[1])  # the second page does not exist
    want = torch.softmax(torch.from_numpy(q[1]).view(2, 2, 8) @ k[:, 0].transpose(1, 2) * 0.5, -1) @ k[:, 1]
    np.testing.assert_allclose(out[1], want.view(4, 8).numpy(), atol=1e-12)
    assert (out[2] == 0).all()
