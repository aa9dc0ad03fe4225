"""GPU parity of causal_attention (forward and every gradient) with float64 (oracle/decoder.py).

Tolerances, elementwise, from the roundings on the way (U: half a step of float32, h: of the type):
* a score is off by (D + 4) U times the sum of its products' magnitudes, its exponent's argument by 4 U of itself, so a
  probability by that relative amount, once for its own score and once for the row's sum (whose n additions and whose
  maximum's slack add n U + 8 U);
* 16-bit types round a probability as an operand (h, and in float16 a subnormal step, of weights that are at most 2^8
  over sums of at least 1), and in the backward the score's gradient likewise;
* sums of n products are off by n U of their magnitudes; results are rounded once.
The backward's delta is the forward's output (its rounding's remainder kept to h^2) times dO.  In the 2-norm, roundings of
independent terms do not add up: errors stay below three half steps there.
"""

import numpy as np
import pytest
import torch

from layer_tolerance import U, assert_within, f64, half, smallest
from oops_amd import OOpsUnsupportedError, causal_attention, gate_attention_output
from oracle import decoder

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def _case(seed, b, h, kv, n, d, e, dtype, scale=1.0, layout="token"):
    g = torch.Generator().manual_seed(seed)

    def make(heads, w):
        if layout == "token":
            return _randn(g, b, n, heads, w, dtype=dtype, scale=scale).transpose(1, 2)
        return _randn(g, b, heads, n, w, dtype=dtype, scale=scale)

    return {"q": make(h, d), "k": make(kv, d), "v": make(kv, e), "do": make(h, e)}


def _bounds(x, scale, offsets, dtype):
    """Elementwise bounds of the errors of out, dq, dk, dv."""

    q, k, v, do = (f64(x[name]) for name in ("q", "k", "v", "do"))
    r, n, d, e = q.shape[1] // k.shape[1], q.shape[2], q.shape[3], v.shape[3]
    t = lambda a: np.swapaxes(a, -1, -2)  # noqa: E731
    a = np.abs
    h = half(dtype) if dtype != torch.float32 else 0.0
    tiny = smallest(dtype) * 2**8 if dtype == torch.float16 else 0.0  # a subnormal step of a weight, over sums >= 1
    kk, vv = np.repeat(k, r, 1), np.repeat(v, r, 1)
    pair = decoder.causal_pairs(n, offsets)
    p = decoder.causal_weights(q, k, scale, offsets)
    size = abs(scale) * (a(q) @ t(a(kk)))
    score = ((d + 4) * U + 4 * U) * np.where(pair, size, 0)
    rel = score + score.max(-1, keepdims=True) + (n + 16) * U  # of a probability
    rel = np.expm1(rel)
    out = p @ vv
    w = p * (rel + h + n * U) + tiny * pair
    err_out = w @ a(vv)
    dp = do @ t(vv)
    delta = (p * dp).sum(-1, keepdims=True)
    err_dp = (e + 2) * U * (a(do) @ t(a(vv)))
    err_delta = (a(do) * (err_out + (h * h + 4 * U) * a(out))).sum(-1, keepdims=True) + (e + 4) * U * (a(do) * a(out)).sum(-1, keepdims=True)
    ds = p * (dp - delta)
    err_ds = p * (rel * a(dp - delta) + err_dp + err_delta + 4 * U * a(dp - delta)) + h * a(ds) + np.where(pair, smallest(dtype) if h else 0.0, 0)
    sized = err_ds * (1 + n * U) + n * U * a(ds)
    group = lambda m: decoder._groups(m, k.shape[1])  # noqa: E731
    bounds = [err_out, abs(scale) * sized @ a(kk), group(abs(scale) * t(sized) @ a(q)), group(t(w * (1 + n * r * U)) @ a(do))]
    want = [out, *decoder.causal_backward(q, k, v, do, scale, offsets)]
    return want, [bound + half(dtype) * a(y) + smallest(dtype) for bound, y in zip(bounds, want)]


def _run(x, offsets=None, scale=None, grads=True):
    dtype = x["q"].dtype
    leaves = [x[name].detach().requires_grad_(True) for name in ("q", "k", "v")]
    o = None if offsets is None else torch.tensor(offsets, dtype=torch.int32, device=DEV)
    out = causal_attention(*leaves, o, scale=scale)
    assert out.dtype == dtype and out.shape == x["do"].shape
    got = [out, *(torch.autograd.grad(out, leaves, x["do"]) if grads else ())]
    scale = x["q"].shape[-1] ** -0.5 if scale is None else scale
    want, bound = _bounds(x, scale, offsets, dtype)
    for name, a, b, c in zip(("out", "dq", "dk", "dv"), got, want, bound):
        assert a.dtype == dtype
        assert_within(a, b, c, name)
        size = np.linalg.norm(b)
        if dtype != torch.float32 and size > 0 and name in ("out", "dv"):
            off = np.linalg.norm(f64(a) - b) / size
            assert off <= 3 * half(dtype), f"{name}: {off:.3g} off in the 2-norm"
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 2, 31, 33, 64, 65, 127, 128, 129, 300])
def test_lengths(dtype, n):
    _run(_case(n, 2, 2, 1, n, 64, 64, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,e", [(128, 128), (8, 8), (32, 32), (1, 1), (40, 128), (128, 40), (96, 96), (33, 17), (100, 64), (64, 3)])
def test_head_sizes(dtype, d, e):
    _run(_case(d * e, 1, 2, 2, 150, d, e, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h,kv", [(1, 1), (8, 8), (8, 1), (6, 3), (10, 2), (16, 8)])
def test_head_groups(dtype, h, kv):
    _run(_case(h * kv, 2, h, kv, 140, 128, 128, dtype))


PACKED = [
    [0, 300],
    [0, 1, 2, 3, 300],
    [0, 0, 64, 64, 128, 256, 300],
    [0, 63, 127, 129, 200, 300, 300],
    [0, 150, 151, 151, 290],  # ten tokens behind the last sequence
    [17, 31, 140, 260],  # and before the first
    [5],  # no sequence
    [300, 300],
    [-4, 20, 1000],  # taken as 0 and 300
    list(range(0, 301, 7)),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offsets", PACKED)
def test_packed_sequences(dtype, offsets):
    """NaN outside every sequence must stay unread; outputs and gradients there are zero."""

    x = _case(len(offsets), 1, 4, 2, 300, 64, 64, dtype)
    lo, hi = max(offsets[0], 0), min(offsets[-1], 300) if len(offsets) > 1 else 0
    clean = {name: t.clone() for name, t in x.items()}
    for t in clean.values():
        t[:, :, :lo], t[:, :, max(hi, lo):] = 0, 0
    for t in x.values():
        t[:, :, :lo], t[:, :, max(hi, lo):] = float("nan"), float("nan")
    got = _run(clean, offsets)
    leaves = [x[name].detach().requires_grad_(True) for name in ("q", "k", "v")]
    out = causal_attention(*leaves, torch.tensor(offsets, device=DEV))
    for a, b in zip(got, (out, *torch.autograd.grad(out, leaves, x["do"]))):
        assert torch.equal(a, b)
        assert (b[:, :, :lo] == 0).all() and (b[:, :, max(hi, lo):] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_is_each_sequence_alone(dtype):
    """Two batch elements packed alike, with int64 bounds: rows of a sequence depend on nothing else."""

    x = _case(3, 2, 4, 2, 333, 128, 128, dtype)
    offsets = [0, 100, 101, 333]
    out = causal_attention(x["q"], x["k"], x["v"], torch.tensor(offsets, device=DEV))
    want, bound = _bounds(x, 128**-0.5, offsets, dtype)
    assert_within(out, want[0], bound[0], "out")
    for lo, hi in zip(offsets, offsets[1:]):
        part = causal_attention(*(x[name][:, :, lo:hi] for name in ("q", "k", "v")))
        assert_within(out[:, :, lo:hi], f64(part), 2 * bound[0][:, :, lo:hi], "part")


@pytest.mark.parametrize("dtype", DTYPES)
def test_scales(dtype):
    for scale in (-0.4, 0.0, 1.0):
        _run(_case(11, 1, 2, 1, 140, 64, 64, dtype), scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_scores(dtype):
    """Scores of some hundreds: the running maximum is raised far and often, most weights underflow."""

    x = _case(12, 1, 2, 1, 260, 128, 128, dtype)
    x["q"] = x["q"] * 24
    x["k"] = (x["k"] * torch.linspace(0.1, 4, 260, device=DEV)[:, None]).to(dtype)
    out = causal_attention(x["q"], x["k"], x["v"])
    want, bound = _bounds(x, 128**-0.5, None, dtype)
    assert_within(out, want[0], bound[0], "out")


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dtype):
    x = _case(13, 2, 4, 2, 100, 64, 64, dtype)
    want = _run(x)
    pad = lambda t, n=1: torch.nn.functional.pad(t, (n, n))[..., n:-n]  # noqa: E731
    head = {name: t.contiguous() for name, t in x.items()}
    odd = {name: pad(t) for name, t in x.items()}  # addresses of 2 or 4 bytes
    wide = {name: pad(t, 8) for name, t in x.items()}
    across = {name: t.transpose(2, 3).contiguous().transpose(2, 3) for name, t in x.items()}  # tokens innermost
    for y in (head, odd, wide, across):
        leaves = [y[name].detach().requires_grad_(True) for name in ("q", "k", "v")]
        out = causal_attention(*leaves)
        for a, b in zip(want, (out, *torch.autograd.grad(out, leaves, y["do"]))):
            assert torch.equal(a, b)
    assert want[0].stride() == x["q"].stride()  # the query's dimension order
    # prefixes, none and two
    one = causal_attention(x["q"][0], x["k"][0], x["v"][0])
    assert torch.equal(one, want[0][0])
    two = causal_attention(*(x[name].unflatten(0, (1, 2)) for name in ("q", "k", "v")))
    assert two.shape == (1, 2, 4, 100, 64) and torch.equal(two[0], want[0])
    # broadcast operands: the gradient of an expanded key is the sum over what it was expanded to
    k1 = x["k"][:1].detach().clone().requires_grad_(True)
    out = causal_attention(x["q"], k1.expand(2, -1, -1, -1), x["v"])
    full = x["k"][:1].expand(2, -1, -1, -1).contiguous().requires_grad_(True)
    ref = causal_attention(x["q"], full, x["v"])
    assert torch.equal(out, ref)
    got = torch.autograd.grad(out, k1, x["do"])[0]
    parts = torch.autograd.grad(ref, full, x["do"])[0]
    torch.testing.assert_close(got, parts.sum(0, keepdim=True), rtol=4 * half(dtype), atol=smallest(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_some_gradients(dtype):
    x = _case(14, 1, 4, 2, 130, 64, 64, dtype)
    want = _run(x)[1:]
    for need in ((0,), (1,), (2,), (0, 2), (1, 2)):
        leaves = [x[name].detach().requires_grad_(i in need) for i, name in enumerate(("q", "k", "v"))]
        out = causal_attention(*leaves)
        for i, g in zip(need, torch.autograd.grad(out, [leaves[i] for i in need], x["do"])):
            assert torch.equal(g, want[i])
    # gradients of other layouts: broadcast (a sum's) and odd addresses
    leaves = [x[name].detach().requires_grad_(True) for name in ("q", "k", "v")]
    got = torch.autograd.grad(causal_attention(*leaves).sum(), leaves)
    ones = torch.autograd.grad(causal_attention(*leaves), leaves, torch.ones_like(x["do"]))
    assert all(torch.equal(a, b) for a, b in zip(got, ones))


def test_gradients_against_differences():
    """float32, directional differences of the operator itself."""

    x = _case(15, 1, 4, 2, 70, 32, 32, torch.float32)
    leaves = [x[name].detach().requires_grad_(True) for name in ("q", "k", "v")]
    grads = torch.autograd.grad(causal_attention(*leaves), leaves, x["do"])
    g = torch.Generator().manual_seed(1)
    for i, grad in enumerate(grads):
        way = _randn(g, *grad.shape)
        step = 2.0**-7
        ends = []
        for s in (step, -step):
            moved = [t.detach() + s * way if i == j else t.detach() for j, t in enumerate(leaves)]
            ends.append((causal_attention(*moved).double() * x["do"].double()).sum())
        want = (ends[0] - ends[1]).item() / (2 * step)
        got = (grad.double() * way.double()).sum().item()
        # (third order: step^2; rounding of 70 * 4 * 32 outputs: U / step each, random)
        size = (grad.double().square().sum() * way.double().square().mean()).sqrt().item()
        assert abs(got - want) <= 0.02 * size, (i, got, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("which", ["q", "k", "v", "do"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_non_finite_values_stay_with_their_tokens(dtype, which, value):
    """One element of token 75 of head 1: earlier tokens, other heads and other sequences keep their bits."""

    x = _case(16, 1, 4, 2, 200, 64, 64, dtype)
    offsets = torch.tensor([0, 10, 90, 200], device=DEV)

    def run(y):
        leaves = [y[name].detach().requires_grad_(True) for name in ("q", "k", "v")]
        out = causal_attention(*leaves, offsets)
        return [out.detach(), *torch.autograd.grad(out, leaves, y["do"])]

    want = run(x)
    y = {name: t.clone() for name, t in x.items()}
    y[which][0, 1, 75, 5] = value
    got = run(y)
    kv = 1 if which in ("k", "v") else 0  # the key head it belongs to
    heads = [2, 3] if kv else ([1] if which in ("q", "do") else [])
    for name, a, b in zip(("out", "dq", "dk", "dv"), got, want):
        same = torch.ones_like(b, dtype=torch.bool)
        if name in ("out", "dq"):
            for h in heads:
                # rows from token 75 to its sequence's end see a key or value; a query's or dO's only its own row
                same[0, h, 75 : 90 if kv else 76] = False
            if name == "out" and which == "do":
                same[:] = True
        else:
            # keys up to token 75 are paired with it; what reaches later rows of the sequence reaches its earlier keys
            same[0, kv, 10:90] = False
            if not kv:
                same[0, kv, 76:90] = True  # (a query or dO reaches the keys before it)
        assert torch.equal(a[same], b[same]), name
    if which == "v":  # only its own column; an infinity stays one
        col = got[0][0, 2:4, 75:90]
        assert (torch.isnan(col[..., 5]) if value != value else col[..., 5] == value).all()
        assert torch.equal(torch.cat((col[..., :5], col[..., 6:]), -1), torch.cat((want[0][0, 2:4, 75:90, :5], want[0][0, 2:4, 75:90, 6:]), -1))
    elif which != "do":
        rows = got[0][0, 2:4, 75] if kv else got[0][0, 1, 75]
        assert kv or not torch.isfinite(rows).any()


def test_no_tokens():
    for b, n in ((0, 5), (2, 0)):
        x = _case(17, b, 4, 2, n, 64, 64, torch.bfloat16)
        leaves = [x[name].detach().requires_grad_(True) for name in ("q", "k", "v")]
        out = causal_attention(*leaves)
        assert out.shape == x["do"].shape
        for g, t in zip(torch.autograd.grad(out, leaves, x["do"]), leaves):
            assert g.shape == t.shape


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_offsets_past_32_bits(dtype):
    """Tokens two MB apart in a buffer of more than 2^32 bytes (and elements)."""

    n, pitch = 2304, 1 << 21
    buf = torch.zeros(n * pitch, dtype=torch.bfloat16, device=DEV).view(torch.bfloat16 if dtype == torch.bfloat16 else torch.float32)
    pitch = buf.numel() // n
    x = _case(18, 1, 1, 1, n, 64, 64, dtype)
    far = buf.view(n, pitch)[:, :192].unflatten(1, (3, 64)).permute(1, 0, 2)  # (3, n, 64)
    for i, name in enumerate(("q", "k", "v")):
        far[i].copy_(x[name][0, 0])
    leaves = [far[i][None, None].detach().requires_grad_(True) for i in range(3)]
    near = [x[name].detach().requires_grad_(True) for name in ("q", "k", "v")]
    out = causal_attention(*leaves)
    ref = causal_attention(*near)
    assert torch.equal(out, ref)
    for a, b in zip(torch.autograd.grad(out, leaves, x["do"]), torch.autograd.grad(ref, near, x["do"])):
        assert torch.equal(a, b)


def test_long_rows_against_float32():
    """4097 tokens in two sequences: bfloat16 outputs and gradients against float32 ones of the same operands."""

    x = _case(19, 1, 4, 1, 4097, 128, 128, torch.bfloat16)
    offsets = torch.tensor([0, 1500, 4097], device=DEV)

    def run(y):
        leaves = [y[name].detach().requires_grad_(True) for name in ("q", "k", "v")]
        out = causal_attention(*leaves, offsets)
        return out.detach(), *torch.autograd.grad(out, leaves, y["do"])

    for name, a, b in zip(("out", "dq", "dk", "dv"), run(x), run({name: t.float() for name, t in x.items()})):
        off = ((a.double() - b.double()).norm() / b.double().norm()).item()
        # P, dS and the result are rounded once each, half a step at most, independent terms
        assert off <= 3 * half(torch.bfloat16), f"{name}: {off:.3g}"
    again = run(x)
    assert all(torch.equal(a, b) for a, b in zip(again, run(x)))  # no order of workgroups changes a bit


def test_refusals():
    x = _case(20, 1, 4, 2, 8, 32, 32, torch.bfloat16)
    q, k, v = x["q"], x["k"], x["v"]
    for bad in ((q.float(), k, v), (q.double(), k.double(), v.double()), (q, k, v, torch.tensor([0.0, 8.0], device=DEV)),
                tuple(torch.zeros(1, h, 8, 160, device=DEV) for h in (4, 2, 2))):  # fmt: skip
        with pytest.raises(OOpsUnsupportedError):
            causal_attention(*bad)
    for bad in ((q, k[:, :, :4], v), (q[:, :3], k, v), (q, k, v[:, :1]), (q, k, v, torch.zeros(2, 2, dtype=torch.int32, device=DEV))):
        with pytest.raises(ValueError):
            causal_attention(*bad)
    with pytest.raises(ValueError, match="device"):
        causal_attention(q, k.cpu(), v)
    leaf = q.detach().requires_grad_(True)
    (g,) = torch.autograd.grad(causal_attention(leaf, k, v).float().square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.float().sum(), leaf)


def test_compile_with_sizes_that_change():
    def f(q, k, v, o):
        return causal_attention(q * 1.0, k, v, o)

    g = torch.compile(f, dynamic=True, fullgraph=True)
    for n in (40, 70, 133):
        x = _case(n, 1, 4, 2, n, 64, 64, torch.bfloat16)
        o = torch.tensor([0, n // 3, n], device=DEV)
        results = []
        for fn in (f, g):
            leaves = [x[name].detach().requires_grad_(True) for name in ("q", "k", "v")]
            out = fn(*leaves, o)
            results.append((out, *torch.autograd.grad(out, leaves, x["do"])))
        assert all(torch.equal(a, b) for a, b in zip(*results))


def test_graph_replays():
    """A captured training step over changing inputs and bounds, replayed with eager work between."""

    x = _case(21, 1, 8, 2, 200, 64, 64, torch.bfloat16)
    offsets = torch.tensor([0, 60, 200], device=DEV)

    def step():
        leaves = [x[name].detach().requires_grad_(True) for name in ("q", "k", "v")]
        out = causal_attention(*leaves, offsets)
        return (out.detach(), *torch.autograd.grad(out, leaves, x["do"]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for replay in range(4):
        new = _case(30 + replay, 1, 8, 2, 200, 64, 64, torch.bfloat16)
        for name, t in x.items():
            t.copy_(new[name])
        offsets.copy_(torch.tensor([replay, 60 + 30 * replay, 200]))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want)), replay


def test_two_streams():
    xs = [_case(40 + i, 1, 8, 2, 500, 128, 128, torch.bfloat16) for i in range(2)]
    want = [_run_bits(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(3):
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(_run_bits(x))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 2]))


def _run_bits(x):
    leaves = [x[name].detach().requires_grad_(True) for name in ("q", "k", "v")]
    out = causal_attention(*leaves)
    return [out.detach(), *torch.autograd.grad(out, leaves, x["do"])]


def test_into_the_gated_output_stage():
    x = _case(22, 2, 4, 2, 50, 32, 32, torch.bfloat16)
    g = torch.Generator().manual_seed(1)
    y, wg, wo = _randn(g, 2, 50, 64, dtype=torch.bfloat16), _randn(g, 128, 64, dtype=torch.bfloat16), _randn(g, 64, 128, dtype=torch.bfloat16)
    att = causal_attention(x["q"], x["k"], x["v"])
    out = gate_attention_output(att, y, wg, wo)
    want = (torch.sigmoid(y.double() @ wg.double().t()) * att.double().transpose(1, 2).flatten(2)) @ wo.double().t()
    assert ((out.double() - want).norm() / want.norm()).item() <= 4 * half(torch.bfloat16)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offsets", [None, [0, 1100], [0, 3, 1000], [40, 1060], [0, 0, 1100, 1100]])
def test_few_heads_of_long_rows(dtype, offsets):
    """Walks that are split into parts and joined, some of which have no tile, or no pair of a row, among them."""

    _run(_case(31, 1, 2, 1, 1100, 48, 64, dtype), offsets)
    if offsets is None:
        _run(_case(32, 1, 1, 1, 1100, 128, 128, dtype), scale=-0.05)


@pytest.mark.parametrize("dtype", DTYPES)
def test_non_finite_values_of_split_rows(dtype):
    """Tokens before an infinity or a NaN have the values that they have without it; from it on nothing is finite."""

    x = _case(33, 1, 1, 1, 1200, 32, 32, dtype)
    clean = _run(x)
    for name, value in (("k", float("nan")), ("v", float("inf")), ("v", float("nan"))):
        y = {n: t.clone() for n, t in x.items()}
        y[name][0, 0, 700, 5] = value
        leaves = [y[n].requires_grad_(True) for n in ("q", "k", "v")]
        out = causal_attention(*leaves)
        assert torch.equal(out[:, :, :700], clean[0][:, :, :700])
        rest = out[:, :, 700:] if name == "k" else out[:, :, 700:, 5]
        assert not torch.isfinite(rest).any()
        if name == "v":
            other = [c for c in range(32) if c != 5]
            assert torch.equal(out[..., other], clean[0][..., other])
        dq, _, _ = torch.autograd.grad(out, leaves, x["do"])
        assert torch.equal(dq[:, :, :700], clean[1][:, :, :700])
    y = x["k"].clone()
    y[0, 0, :1150] = 0
    y[0, 0, :1150, 0] = float("-inf")
    q = x["q"].abs()
    # (every logit of a row -inf: 0 / 0; the tokens with others have those alone)
    out = causal_attention(q, y, x["v"])
    assert out[:, :, :1150].isnan().all()
    alone = causal_attention(q[:, :, 1150:].contiguous(), y[:, :, 1150:].contiguous(), x["v"][:, :, 1150:].contiguous())
    assert ((out[:, :, 1150:].double() - alone.double()).norm() / alone.double().norm()).item() <= 2 * half(dtype) + 2000 * U


def test_graphs_of_split_rows():
    """Two captured training steps whose walks are split, replayed in turn beside eager calls: the eager bits each time."""

    cases = [_case(41, 1, 2, 1, 1100, 64, 64, torch.bfloat16), _case(42, 1, 3, 3, 700, 40, 32, torch.float32)]
    want = []
    side = torch.cuda.Stream()
    for x in cases:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want.append(_run_bits(x))
        torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for x in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = _run_bits(x)
        graphs.append((graph, got))
    for _ in range(3):
        for (graph, got), expected, x in zip(graphs, want, cases):
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(got, expected))
            assert all(torch.equal(a, b) for a, b in zip(_run_bits(x), expected))
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,offsets", [(1, None), (40, list(range(41)))])
def test_rows_of_one_key(dtype, n, offsets):
    """A weight that is 1 whatever its score: dQ and dK are zeros, to the last bit."""

    _, dq, dk, _ = _run(_case(51, 2, 4, 2, n, 64, 48, dtype), offsets)
    assert not dq.any() and not dk.any()
