"""GPU parity of rms_norm_rotary (forward and every gradient) with float64 (oracle/decoder.py).

Tolerances (U: half a step of float32, h: of the result's type).  A row's mean square is off by (D / 16 + 8) U of itself
at most (a lane adds 8, lanes are added in a tree; the other layout 4 and a tree), its reciprocal square root by half of
that and 3 U; products and the rotation add one rounding each, of the pair's magnitudes |z_i c| + |z_j s|: 32 U of them in
all.  In the backward the mean of g n is a sum of magnitudes with the same count; the weights' gradients add R rows in
chains of at most R / 16 + 128 additions.  The result is rounded once.
"""

import numpy as np
import pytest
import torch

from layer_tolerance import U, assert_within, f64, half, smallest
from oops_amd import OOpsUnsupportedError, rms_norm_rotary, rotary_table
from oracle import decoder

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
EPS = 1e-6


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def _case(seed, b, h, kv, n, d, rotary, dtype, weight=torch.float32, positions=True, rows=5000):
    g = torch.Generator().manual_seed(seed)
    make = lambda heads: _randn(g, b, n, heads, d, dtype=dtype).transpose(1, 2)  # noqa: E731
    x = {"q": make(h), "k": make(kv), "dq": make(h), "dk": make(kv), "table": rotary_table(rows, rotary, 500.0, device=DEV)}
    if weight is not None:
        x["wq"], x["wk"] = ((1 + 0.2 * _randn(g, d)).to(weight) for _ in range(2))
    if positions:
        x["positions"] = torch.randint(0, rows, (b, n), generator=g, dtype=torch.int32).to(DEV)
    return x


def _args(x, leaves):
    return (leaves[0], leaves[1], x["table"], x.get("positions"), *(leaves[2:] or (None, None)), EPS)


def _leaves(x):
    return [x[name].detach().requires_grad_(True) for name in ("q", "k", "wq", "wk") if name in x]


def _run(x):
    dtype = x["q"].dtype
    leaves = _leaves(x)
    outs = rms_norm_rotary(*_args(x, leaves))
    grads = torch.autograd.grad(outs, leaves, (x["dq"], x["dk"]))
    b, _, n, d = x["q"].shape
    p = np.broadcast_to(np.arange(n), (b, n)) if "positions" not in x else x["positions"].cpu().numpy()
    p = np.clip(np.broadcast_to(p, (b, n)), 0, x["table"].shape[0] - 1)
    row = f64(x["table"])[p][:, None]
    cos, sin = row[..., 0, :], row[..., 1, :]
    for i, name in enumerate(("q", "k")):
        t, w, dy = f64(x[name]), f64(x.get("w" + name)), f64(x["d" + name])
        y = decoder.norm_rotary_forward(t, cos, sin, w, EPS)
        z = np.abs(t) / np.sqrt((t * t).mean(-1, keepdims=True) + EPS) * (1 if w is None else np.abs(w))
        both = decoder.rotate(z, np.abs(cos), -np.abs(sin))  # |z_i c| + |z_j s| in the first half
        both = np.maximum(both, decoder.rotate(z, np.abs(cos), np.abs(sin)))
        count = d / 16 + 32
        # (the strides of dimensions of one element are nobody's)
        same = [a == b for a, b, m in zip(outs[i].stride(), x[name].stride(), x[name].shape) if m > 1]
        assert outs[i].dtype == dtype and outs[i].shape == x[name].shape and all(same)
        assert_within(outs[i], y, count * U * both + half(dtype) * np.abs(y) + smallest(dtype), name)
        dx, dw = decoder.norm_rotary_backward(t, cos, sin, dy, w, EPS)
        rstd = 1 / np.sqrt((t * t).mean(-1, keepdims=True) + EPS)
        nn = np.abs(t) * rstd
        gg = np.maximum(decoder.rotate(np.abs(dy), np.abs(cos), -np.abs(sin)), decoder.rotate(np.abs(dy), np.abs(cos), np.abs(sin)))
        gw = gg * (1 if w is None else np.abs(w))
        size = rstd * (gw + nn * (gw * nn).mean(-1, keepdims=True))
        assert_within(grads[i], dx, 2 * count * U * size + half(dtype) * np.abs(dx) + smallest(dtype), "d" + name)
        if w is not None:
            rows = t.shape[0] * t.shape[1] * t.shape[2]
            dt = x["w" + name].dtype
            bound = (rows / 16 + 128 + count) * U * (gg * nn).sum((0, 1, 2))
            assert grads[2 + i].dtype == dt
            assert_within(grads[2 + i], dw, bound + half(dt) * np.abs(dw) + smallest(dt), "dw" + name)
    return outs, grads


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,rotary", [(128, 128), (64, 64), (256, 256), (128, 64), (128, 16), (80, 40), (80, 32), (96, 96), (24, 16),
                                      (8, 8), (1, 0), (2, 2), (7, 4), (130, 130), (255, 254), (64, 0), (128, 2)])  # fmt: skip
def test_sizes(dtype, d, rotary):
    _run(_case(d, 2, 4, 2, 37, d, rotary, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 2, 15, 16, 500])
def test_lengths(dtype, n):
    _run(_case(n, 3, 5, 1, n, 128, 128, dtype, weight=dtype, positions=n != 15))


@pytest.mark.parametrize("dtype", DTYPES)
def test_without_weights_and_with_one(dtype):
    _run(_case(1, 1, 2, 2, 40, 64, 64, dtype, weight=None))
    x = _case(2, 1, 2, 2, 40, 64, 64, dtype)
    q, k = rms_norm_rotary(x["q"], x["k"], x["table"], x["positions"], None, x["wk"])
    both = rms_norm_rotary(x["q"], x["k"], x["table"], x["positions"], torch.ones_like(x["wk"]), x["wk"])
    assert torch.equal(q, both[0]) and torch.equal(k, both[1])


def test_positions():
    """int64, expanded, outside the table (the nearer end), and the default's 0, 1, ..."""

    x = _case(3, 2, 3, 2, 30, 64, 64, torch.bfloat16, rows=100)
    a = (x["q"], x["k"], x["table"])
    want = rms_norm_rotary(*a, x["positions"])
    assert all(torch.equal(s, t) for s, t in zip(rms_norm_rotary(*a, x["positions"].long()), want))
    line = x["positions"][:1]
    want = rms_norm_rotary(*a, line.expand(2, -1).contiguous())
    for p in (line, line[0], line.expand(2, -1)):
        assert all(torch.equal(s, t) for s, t in zip(rms_norm_rotary(*a, p), want))
    want = rms_norm_rotary(*a, torch.arange(30, device=DEV))
    assert all(torch.equal(s, t) for s, t in zip(rms_norm_rotary(*a), want))
    far = torch.tensor([-7, 1 << 40], device=DEV).repeat(15)
    want = rms_norm_rotary(*a, torch.tensor([0, 99], device=DEV).repeat(15))
    assert all(torch.equal(s, t) for s, t in zip(rms_norm_rotary(*a, far), want))
    # (one position for all tokens)
    want = rms_norm_rotary(*a, torch.full((2, 30), 7, device=DEV))
    assert all(torch.equal(s, t) for s, t in zip(rms_norm_rotary(*a, torch.tensor([7], device=DEV)), want))


def test_table():
    t = rotary_table(100000, 64, 10000.0, device=DEV)
    a = np.arange(100000)[:, None] * 10000.0 ** (-np.arange(32) / 32)
    # (float64 angles up to 1e5: 1e-11 off at most; one rounding)
    assert_within(t, np.stack((np.cos(a), np.sin(a)), 1), U + 1e-10, "table")
    assert rotary_table(0, 8, device=DEV).shape == (0, 2, 4) and rotary_table(3, 0, device=DEV).shape == (3, 2, 0)
    with pytest.raises(ValueError):
        rotary_table(4, 7, device=DEV)


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dtype):
    x = _case(4, 2, 4, 2, 50, 128, 128, dtype)
    outs, grads = _run(x)
    pad = lambda t, n=1: torch.nn.functional.pad(t, (n, n))[..., n:-n]  # noqa: E731
    head = {name: x[name].contiguous() for name in ("q", "k", "dq", "dk")}
    odd = {name: pad(x[name]) for name in ("q", "k", "dq", "dk")}
    innermost = {name: x[name].transpose(2, 3).contiguous().transpose(2, 3) for name in ("q", "k", "dq", "dk")}
    for other in (head, odd, innermost):
        y = x | other
        leaves = _leaves(y)
        o = rms_norm_rotary(*_args(y, leaves))
        got = [*o, *torch.autograd.grad(o, leaves, (y["dq"], y["dk"]))]
        for a, b in zip(got, (*outs, *grads)):
            # (the other layout adds a row's squares in another order)
            torch.testing.assert_close(a, b, rtol=2.1 * half(dtype) + 200 * U, atol=300 * U * b.detach().abs().max().item())
    one = rms_norm_rotary(x["q"][0], x["k"][0], x["table"], x["positions"][0], x["wq"], x["wk"], EPS)
    assert torch.equal(one[0], outs[0][0]) and torch.equal(one[1], outs[1][0])
    two = rms_norm_rotary(x["q"][None], x["k"][None], x["table"], x["positions"][None], x["wq"], x["wk"], EPS)
    assert torch.equal(two[0][0], outs[0]) and torch.equal(two[1][0], outs[1])


def test_some_gradients():
    x = _case(5, 2, 4, 2, 20, 64, 64, torch.bfloat16)
    _, want = _run(x)
    names = ("q", "k", "wq", "wk")
    for need in ((0,), (1,), (2,), (3,), (0, 3), (1, 2)):
        leaves = [x[name].detach().requires_grad_(i in need) for i, name in enumerate(names)]
        outs = rms_norm_rotary(*_args(x, leaves))
        got = torch.autograd.grad(outs, [leaves[i] for i in need], (x["dq"], x["dk"]))
        assert all(torch.equal(g, want[i]) for i, g in zip(need, got))
    # one output used
    for which in (0, 1):
        leaves = _leaves(x)
        out = rms_norm_rotary(*_args(x, leaves))[which]
        got = torch.autograd.grad(out, leaves, x[("dq", "dk")[which]], allow_unused=True)
        for i, g in enumerate(got):
            assert torch.equal(g, want[i]) if i % 2 == which else g is None


def test_many_rows():
    """More rows than one walk of the backward's workgroups, twice the same bits."""

    x = _case(6, 1, 16, 4, 9000, 64, 64, torch.bfloat16)
    _, grads = _run(x)
    _, again = _run(x)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


def test_more_than_32_bits_of_elements():
    q = torch.zeros(1, 33, 1 << 19, 256, dtype=torch.bfloat16, device=DEV)
    q[0, 32, -1] = torch.arange(256, device=DEV)
    k = q[:, 32:, -4:]
    table = rotary_table(8, 256, device=DEV)
    p = torch.tensor([0, 1, 2, 3], device=DEV)
    y, _ = rms_norm_rotary(q, q[:, :1], table, torch.zeros(1, dtype=torch.int32, device=DEV))
    want, _ = rms_norm_rotary(k, k, table, p * 0)
    assert torch.equal(y[0, 32, -4:], want[0, 0]) and y.view(torch.int16)[0, :32].count_nonzero() == 0


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_non_finite_rows(value):
    x = _case(7, 1, 4, 2, 20, 64, 64, torch.bfloat16)
    want = rms_norm_rotary(*_args(x, [x["q"], x["k"], x["wq"], x["wk"]]))
    x["q"][0, 1, 5, 3] = value
    got = rms_norm_rotary(*_args(x, [x["q"], x["k"], x["wq"], x["wk"]]))
    assert torch.equal(got[1], want[1])
    assert torch.isnan(got[0][0, 1, 5]).any()
    got[0][0, 1, 5] = want[0][0, 1, 5]
    assert torch.equal(got[0], want[0])


def test_no_tokens():
    for b, n in ((0, 4), (2, 0)):
        x = _case(8, b, 4, 2, n, 64, 64, torch.float16)
        leaves = _leaves(x)
        outs = rms_norm_rotary(*_args(x, leaves))
        assert outs[0].shape == x["q"].shape and outs[1].shape == x["k"].shape
        grads = torch.autograd.grad(outs, leaves, (x["dq"], x["dk"]))
        assert all(g.shape == t.shape for g, t in zip(grads, leaves)) and not grads[2].any() and not grads[3].any()


def test_refusals():
    x = _case(9, 1, 4, 2, 8, 32, 32, torch.bfloat16, rows=8)
    q, k, t = x["q"], x["k"], x["table"]
    for bad in ((q.float(), k, t), (q.double(), k.double(), t), (q, k, t.double()), (q, k, t, x["positions"].float()),
                (q, k, t, None, x["wq"].double()), (q, k, t, None, x["wq"][:5]), (q, k, t.requires_grad_(True)),
                tuple(torch.zeros(1, h, 8, 257, device=DEV) for h in (4, 2)) + (t.detach(),)):  # fmt: skip
        with pytest.raises(OOpsUnsupportedError):
            rms_norm_rotary(*bad)
    t = t.detach()
    for bad in ((q, k[:, :, :4], t), (q[0], k, t), (q, k, t[:, 0]), (q, k, rotary_table(8, 34, device=DEV)), (q, k, t[:5]),
                (q, k, t, torch.zeros(2, 8, dtype=torch.int32, device=DEV)), (q, k, t[:0], x["positions"])):  # fmt: skip
        with pytest.raises(ValueError):
            rms_norm_rotary(*bad)
    leaf = q.detach().requires_grad_(True)
    (g,) = torch.autograd.grad(rms_norm_rotary(leaf, k, t)[0].float().square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.float().sum(), leaf)


def test_compile_with_sizes_that_change():
    def f(q, k, t, p, wq, wk, eps):
        return rms_norm_rotary(q * 1.0, k * 1.0, t, p, wq, wk, eps)

    g = torch.compile(f, dynamic=True, fullgraph=True)
    for n in (5, 9, 33):
        x = _case(n, 2, 4, 2, n, 64, 64, torch.bfloat16)
        results = []
        for fn in (f, g):
            leaves = _leaves(x)
            outs = fn(*_args(x, leaves))
            results.append((*outs, *torch.autograd.grad(outs, leaves, (x["dq"], x["dk"]))))
        assert all(torch.equal(a, b) for a, b in zip(*results))


def test_graph_replays_and_streams():
    x = _case(10, 2, 8, 2, 64, 128, 128, torch.bfloat16)

    def step():
        leaves = _leaves(x)
        outs = rms_norm_rotary(*_args(x, leaves))
        return (*(t.detach() for t in outs), *torch.autograd.grad(outs, leaves, (x["dq"], x["dk"])))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(there, step()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for replay in range(3):
        y = _case(20 + replay, 2, 8, 2, 64, 128, 128, torch.bfloat16)
        for name in x:
            x[name].copy_(y[name])
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want)), replay
