"""causal_attention with infinities and NaN: which results are finite is decided by the formula, taken literally in float64.

A sum over the pairs of a row (or of a key) holds what is not finite in them and nothing else.  Weights are positive, so an
infinity in a value or in an output's gradient stays an infinity in the output's or the value gradient's column; everything
else that is not finite may be an infinity or a NaN, as float32 sums have it.  Elements that hold none keep their bits.
"""

import numpy as np
import pytest
import torch

from layer_tolerance import f64
from oops_amd import causal_attention

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
INF, NAN = float("inf"), float("nan")


def _case(seed, h, kv, n, d, dtype):
    g = torch.Generator().manual_seed(seed)
    make = lambda heads: torch.randn(1, n, heads, d, generator=g).to(dtype).to(DEV).transpose(1, 2)  # noqa: E731
    return {"q": make(h), "k": make(kv), "v": make(kv), "do": make(h)}


def _run(x, offsets=None, scale=None):
    leaves = [x[name].detach().clone().requires_grad_(True) for name in ("q", "k", "v")]
    o = None if offsets is None else torch.tensor(offsets, device=DEV)
    out = causal_attention(*leaves, o, scale=scale)
    return [out.detach(), *torch.autograd.grad(out, leaves, x["do"])]


def _start(offsets, i):
    """The first token of token i's sequence, or None."""

    if offsets is None:
        return 0
    for lo, hi in zip(offsets, offsets[1:]):
        if lo <= i < hi:
            return lo
    return None


def _literal(x, offsets=None, scale=None):
    """out, dq, dk, dv by their sums over the pairs that there are, float64."""

    q, k, v, do = (f64(x[name])[0] for name in ("q", "k", "v", "do"))
    r, scale = q.shape[0] // k.shape[0], q.shape[2] ** -0.5 if scale is None else scale
    out, dq, dk, dv = (np.zeros(t.shape) for t in (q, q, k, v))
    with np.errstate(all="ignore"):
        for h in range(q.shape[0]):
            for i in range(q.shape[1]):
                lo = _start(offsets, i)
                if lo is None:
                    continue
                at = slice(lo, i + 1)
                kk, vv, w = k[h // r, at], v[h // r, at], do[h, i]
                s = scale * (kk * q[h, i]).sum(-1)
                p = np.exp(s - s.max())
                p = p / p.sum()
                out[h, i] = (p[:, None] * vv).sum(0)
                dp = (vv * w).sum(-1)
                ds = scale * p * (dp - (p * dp).sum())
                dq[h, i] = (ds[:, None] * kk).sum(0)
                dk[h // r, at] += ds[:, None] * q[h, i]
                dv[h // r, at] += p[:, None] * w
    return [t[None] for t in (out, dq, dk, dv)]


# heads, key heads, tokens, channels, bounds, the token with the value
PLACES = [
    (4, 2, 1, 64, None, 0),  # a row of one key
    (4, 2, 40, 64, None, 3),  # the first tile that its rows meet
    (4, 2, 40, 128, None, 39),
    (4, 2, 20, 64, [0, 7, 20], 9),  # a sequence inside a tile
    (4, 2, 300, 128, None, 5),  # rows of later blocks, to whom the tile is whole
    (4, 2, 300, 64, None, 259),  # ... a query behind whole tiles of keys
    (4, 2, 300, 128, [0, 130, 300], 140),
    (1, 1, 1100, 64, None, 70),  # walks in parts
    (1, 1, 1100, 128, None, 700),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("which", ["q", "k", "v", "do"])
@pytest.mark.parametrize("value", [NAN, INF, -INF])
@pytest.mark.parametrize("h,kv,n,d,offsets,token", PLACES)
def test_what_holds_it_and_nothing_else(dtype, which, value, h, kv, n, d, offsets, token):
    x = _case(n + token, h, kv, n, d, dtype)
    y = {name: t.clone() for name, t in x.items()}
    head = min(1, x[which].shape[1] - 1)
    y[which][0, head, token, 5] = value
    want, clean, got = _literal(y, offsets), _run(x, offsets), _run(y, offsets)
    for name, a, b in zip(("out", "dq", "dk", "dv"), got, want):
        assert np.array_equal(np.isfinite(f64(a)), np.isfinite(b)), name
    if which in ("v", "do"):
        # its own column takes the value itself, in the rows (or keys) that are paired with it; nothing else changes
        a, b = (got[0], clean[0]) if which == "v" else (got[3], clean[3])
        lost = torch.from_numpy(~np.isfinite(want[0] if which == "v" else want[3])).to(DEV)
        assert lost.any() and not lost[..., :5].any() and not lost[..., 6:].any()
        assert (torch.isnan(a[lost]) if value != value else a[lost] == value).all()
        assert torch.equal(a[~lost], b[~lost])


@pytest.mark.parametrize("dtype", DTYPES)
def test_an_infinity_where_the_maximum_rises_far(dtype):
    """Scores of -200, then of 200: what earlier tiles have left underflows, the infinity of a later tile does not."""

    x = _case(1, 1, 1, 128, 64, dtype)
    x["q"], x["k"] = torch.zeros_like(x["q"]), torch.zeros_like(x["k"])
    x["q"][..., 0] = 1
    x["k"][:, :, :64, 0], x["k"][:, :, 64:, 0] = -200, 200
    x["v"][0, 0, 70, 5] = INF
    out = causal_attention(x["q"], x["k"], x["v"], scale=1.0)
    assert (out[0, 0, 70:, 5] == INF).all() and torch.isfinite(out[0, 0, :70]).all() and torch.isfinite(out[0, 0, 70:, 6:]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_an_infinity_with_small_weights(dtype):
    """Weights down to e^-40 or so, positive all the same: the infinity reaches every row or key that is paired with it."""

    x = _case(2, 1, 1, 400, 64, dtype)
    y = {name: t.clone() for name, t in x.items()}
    y["v"][0, 0, 30, 5] = INF
    assert (_run(y, scale=1.0)[0][0, 0, 30:, 5] == INF).all()
    y = {name: t.clone() for name, t in x.items()}
    y["do"][0, 0, 390, 5] = -INF
    dv = _run(y, scale=1.0)[3]
    assert (dv[0, 0, :391, 5] == -INF).all() and torch.isfinite(dv[0, 0, 391:]).all() and torch.isfinite(dv[..., :5]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,token", [(1, 0), (40, 39), (40, 0), (300, 299)])
def test_a_row_whose_scores_are_all_minus_infinity(dtype, n, token):
    """0 / 0 in its output, and in all gradients that its weights reach."""

    x = _case(3, 1, 1, n, 64, dtype)
    x["k"][..., 5] = x["k"][..., 5].abs() + 1
    x["q"][0, 0, token, 5] = -INF
    out, dq, dk, dv = _run(x)
    for t in (out[0, 0, token], dq[0, 0, token], dk[0, 0, : token + 1], dv[0, 0, : token + 1]):
        assert torch.isnan(t).all()
    others = [i for i in range(n) if i != token]
    assert torch.isfinite(out[0, 0, others]).all() and torch.isfinite(dv[0, 0, token + 1 :]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,token", [(1, 0), (40, 0), (1100, 0), (1100, 1000)])
def test_an_infinity_in_a_row_whose_scores_are_all_minus_infinity(dtype, n, token):
    """NaN in every column, the infinite value's too; keys of -inf up to the row's own, walks in parts among them."""

    x = _case(5, 1, 1, n, 64, dtype)
    x["q"][..., 5] = x["q"][..., 5].abs() + 1
    x["k"][0, 0, : token + 1, 5] = -INF
    x["v"][0, 0, token // 2, 7] = INF
    out = causal_attention(x["q"], x["k"], x["v"])
    assert torch.isnan(out[0, 0, : token + 1]).all() and torch.isfinite(out[0, 0, token + 1 :, 8:]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [NAN, INF, -INF])
@pytest.mark.parametrize("n,offsets", [(40, None), (300, [0, 1, 200, 290])])
def test_scales_that_are_not_finite(dtype, scale, n, offsets):
    """Every score is an infinity or a NaN, so every row is 0 / 0 or inf / inf; rows of no sequence are zeros."""

    last = n if offsets is None else offsets[-1]
    for t in _run(_case(4, 4, 2, n, 64, dtype), offsets, scale):
        assert torch.isnan(t[:, :, :last]).all() and not t[:, :, last:].any()
