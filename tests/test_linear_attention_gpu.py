"""GPU parity of linear_attention (forward, every gradient, states, lengths) and linear_attention_step with the
float64 recurrence (oracle/layers.py).

Tolerances.  With M the same operator over the operands' magnitudes (|q|, |k|, |v|, |S0|), which bounds the
magnitudes of all terms of a sum: float32 arithmetic is off by at most a count of additions and roundings times
U M (chains of a head's 128 rows and of the tokens; decays are powers, each off by a few U and as many as chunks
meet), taken as 2000 U; 16-bit kernels may round the in-chunk weights and the state that the second products read
once each, half a step of M together (they are different terms), their update a 2^-16 of M; the result is rounded
once.  In the 2-norm two roundings of independent terms stay below a full step of the result.
"""

import numpy as np
import pytest
import torch

from layer_tolerance import U, assert_within, f64, half, smallest
from oops_amd import OOpsUnsupportedError, gate_attention_output, linear_attention, linear_attention_step
from oracle import layers

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def _case(seed, b, h, n, d, e, dtype, state=True, layout="token"):
    g = torch.Generator().manual_seed(seed)

    def make(w):
        if layout == "token":
            return _randn(g, b, n, h, w, dtype=dtype).transpose(1, 2)
        return _randn(g, b, h, n, w, dtype=dtype)

    x = {"q": make(d), "k": make(d), "v": make(e), "do": make(e)}
    x["ld"] = -torch.exp2(-torch.linspace(0.0, 9.0, h)).to(DEV) if h > 1 else torch.tensor([-0.05], device=DEV)
    if state:
        x["s0"], x["ds"] = _randn(g, b, h, d, e), _randn(g, b, h, d, e)
    return x


def _bound(want, size, dtype):
    rounded = 0.0 if dtype == torch.float32 else 1.01 * half(dtype) + 2.0**-15
    return (rounded + 2000 * U) * size + half(dtype) * abs(want) + smallest(dtype)


def _check(got, want, size, dtype, what, kind=None):
    """``kind``: the type of the kernels' operands where it is not the result's (float32 states)."""

    got_dtype = got.dtype
    if got_dtype == torch.float32 and kind not in (None, torch.float32):
        bound = 2000 * U * size + U * abs(want)  # states are kept in float32 whatever the operands' type
    else:
        bound = _bound(want, size, dtype)
    assert_within(got, want, bound, what)
    if got_dtype != torch.float32 and np.linalg.norm(want) > 0:
        off = np.linalg.norm(f64(got) - want) / max(np.linalg.norm(want), 0.1 * np.linalg.norm(size))
        assert off <= 2 * half(dtype), f"{what}: {off:.3g} off in the 2-norm"


def _run(x, lengths=None, scale=None, want_state=True, check_grads=True):
    dtype = x["q"].dtype
    names = ["q", "k", "v"] + (["s0"] if "s0" in x else [])
    leaves = [x[n].detach().requires_grad_(True) for n in names]
    s0 = leaves[3] if "s0" in x else None
    res = linear_attention(*leaves[:3], x["ld"], s0, lengths, scale=scale, return_state=want_state)
    out, state = res if want_state else (res, None)
    assert out.dtype == dtype and out.shape == x["do"].shape
    q, k, v, do, ld = (f64(x[n]) for n in ("q", "k", "v", "do", "ld"))
    s, ds = (f64(x.get(n)) for n in ("s0", "ds"))
    n = None if lengths is None else lengths.cpu().numpy()
    a = lambda t: None if t is None else abs(t)  # noqa: E731
    want = layers.linear_attention_forward(q, k, v, ld, s, n, scale)
    size = layers.linear_attention_forward(a(q), a(k), a(v), ld, a(s), n, None if scale is None else abs(scale))
    _check(out, want[0], size[0], dtype, "out")
    if want_state:
        assert state.dtype == torch.float32
        _check(state, want[1], size[1], torch.float32, "state", dtype)
    if not check_grads:
        return out, state
    use = want_state and "ds" in x
    outs, gs = ((out, state), (x["do"], x["ds"])) if use else ((out,), (x["do"],))
    grads = torch.autograd.grad(outs, leaves, gs)
    want = layers.linear_attention_backward(q, k, v, ld, do, ds if use else None, s, n, scale)
    size = layers.linear_attention_backward(a(q), a(k), a(v), ld, a(do), a(ds) if use else None, a(s), n,
                                            None if scale is None else abs(scale))  # fmt: skip
    for i, name in enumerate(names):
        assert grads[i].dtype == leaves[i].dtype
        _check(grads[i], want[i], size[i], leaves[i].dtype, "d" + name, dtype)
    return out, state


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 2, 31, 32, 63, 64, 65, 127, 130, 257, 700])
def test_lengths(dtype, n):
    _run(_case(n, 2, 3, n, 64, 64, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,e", [(1, 1), (8, 8), (32, 32), (16, 64), (64, 24), (33, 17), (96, 96), (100, 128), (128, 128),
                                 (128, 40), (3, 128)])  # fmt: skip
def test_head_sizes(dtype, d, e):
    _run(_case(d * e, 1, 2, 150, d, e, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_without_states(dtype):
    _run(_case(5, 2, 2, 200, 32, 64, dtype, state=False), want_state=False)
    _run(_case(6, 2, 2, 200, 64, 64, dtype, state=False), want_state=True)  # its gradient unused
    _run(_case(7, 2, 2, 200, 128, 128, dtype, layout="head"), want_state=False, scale=-0.3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_ragged_batches(dtype, kind):
    """Lengths of zero, one, a chunk, all; NaN in the rows behind them, which must stay unread."""

    n = 200
    lengths = torch.tensor([n, 0, 1, 64, 65, 137], dtype=kind, device=DEV)
    x = _case(11, 6, 2, n, 64, 64, dtype)
    for name in ("q", "k", "v", "do"):
        for b, m in enumerate(lengths.tolist()):
            x[name][b, :, m:] = float("nan")
    clean = {k: torch.nan_to_num(t) if t.dim() == 4 else t for k, t in x.items()}
    leaves = [x[m].detach().requires_grad_(True) for m in ("q", "k", "v", "s0")]
    out, state = linear_attention(*leaves[:3], x["ld"], leaves[3], lengths, return_state=True)
    grads = torch.autograd.grad((out, state), leaves, (x["do"], x["ds"]))
    ref, ref_state = _run(clean, lengths)
    leaves = [clean[m].detach().requires_grad_(True) for m in ("q", "k", "v", "s0")]
    o2, s2 = linear_attention(*leaves[:3], x["ld"], leaves[3], lengths, return_state=True)
    want = torch.autograd.grad((o2, s2), leaves, (clean["do"], x["ds"]))
    assert torch.equal(out, ref) and torch.equal(state, ref_state)
    for a, b in zip(grads, want):
        assert torch.equal(a, b)
    for b, m in enumerate(lengths.tolist()):
        assert not out[b, :, m:].any() and not any(g[b, :, m:].any() for g in grads[:3])
    assert torch.equal(state[1], x["s0"][1])  # no token: the state is the initial one
    over = torch.tensor([n + 5, -3, 1, 64, 65, 137], dtype=kind, device=DEV)  # the nearer bound
    assert torch.equal(linear_attention(*clean_qkv(clean), x["ld"], x["s0"], over), ref)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,e", [(128, 128), (64, 40), (24, 32)])
def test_ragged_batches_in_segments(dtype, d, e):
    """Sequences that end in the first, a middle and the last of a walk's segments, at their borders and before them."""

    n = 900
    lengths = torch.tensor([n, 0, 1, 128, 129, 500, 512, 700], dtype=torch.int32, device=DEV)
    x = _case(13, 8, 1, n, d, e, dtype)
    _run(x, lengths)
    x = {k: t for k, t in x.items() if k not in ("s0", "ds")}
    _run(x, lengths)


def clean_qkv(x):
    return x["q"], x["k"], x["v"]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("decay", [0.0, -1e-4, -30.0, -1e4, float("-inf"), 0.002])
def test_decays(dtype, decay):
    """No decay, hardly any, nothing left after one token, no memory at all, a slow growth."""

    x = _case(17, 1, 2, 190, 32, 32, dtype)
    x["ld"] = torch.full((2,), decay, device=DEV)
    _run(x)


@pytest.mark.parametrize("dtype", [torch.float16])
def test_half_precision_range(dtype):
    """States and products past 65504 whose outputs are not."""

    x = _case(19, 1, 2, 300, 64, 64, dtype)
    x["q"], x["k"] = x["q"] * 40, x["k"] * 40
    x["v"], x["do"], x["s0"], x["ds"] = x["v"] * 0.02, x["do"] * 1e-4, x["s0"] * 100, x["ds"] * 1e-3
    _run(x)


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dtype):
    """Token-major and head-major views, keys shared by heads, rows inside wider ones, odd strides, prefixes."""

    g = torch.Generator().manual_seed(23)
    ld = torch.tensor([-0.5, -0.1, -0.02, -0.004], device=DEV)
    wide = _randn(g, 2, 150, 4, 3, 72, dtype=dtype)  # (B, L, H, qkv, .)
    q, k, v = (wide[..., i, :64].transpose(1, 2) for i in range(3))
    odd = _randn(g, 2, 150, 4, 67, dtype=dtype).transpose(1, 2)[..., 1:65]
    shared = _randn(g, 2, 1, 150, 64, dtype=dtype).expand(2, 4, 150, 64)
    for qq, kk, vv in ((q, k, v), (q.contiguous(), k, v), (q, shared, v), (q, shared, shared), (odd, k, odd),
                       (q, k, odd.flip(-1))):  # fmt: skip
        got = linear_attention(qq, kk, vv, ld)
        want = layers.linear_attention_forward(f64(qq), f64(kk), f64(vv), f64(ld))[0]
        size = layers.linear_attention_forward(abs(f64(qq)), abs(f64(kk)), abs(f64(vv)), f64(ld))[0]
        _check(got, want, size, dtype, "out")
    flat = linear_attention(q, k, v, ld)
    more = [t.reshape(2, 1, 4, 150, 64) for t in (q, k, v)]
    assert torch.equal(linear_attention(*more, ld), flat.view(2, 1, 4, 150, 64))
    one, state = linear_attention(q[0], k[0], v[0], ld, lengths=torch.tensor(150, device=DEV), return_state=True)
    assert torch.equal(one, flat[0]) and state.shape == (4, 64, 64)
    leaf = shared[:, :1].detach().clone().requires_grad_(True)
    do = _randn(g, 2, 4, 150, 64, dtype=dtype)
    (dk,) = torch.autograd.grad(linear_attention(q, leaf.expand(2, 4, 150, 64), v, ld), leaf, do)
    full = [f64(t) for t in (q, leaf.expand(2, 4, 150, 64), v, ld, do)]
    want = layers.linear_attention_backward(*full)[1]
    size = layers.linear_attention_backward(*[abs(t) if i != 3 else t for i, t in enumerate(full)])[1]
    bound = _bound(want, size, dtype).sum(1, keepdims=True) + 5 * half(dtype) * abs(want).sum(1, keepdims=True)
    assert_within(dk, want.sum(1, keepdims=True), bound, "shared keys' gradient")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradient_layouts(dtype):
    """Expanded and strided gradients of the output, of the state alone, and of one operand alone."""

    x = _case(29, 2, 2, 90, 32, 32, dtype)
    base = [x[n].detach().requires_grad_(True) for n in ("q", "k", "v", "s0")]
    run = lambda: linear_attention(*base[:3], x["ld"], base[3], return_state=True)  # noqa: E731
    ones = torch.ones_like(x["do"])
    want = torch.autograd.grad(run()[0], base, ones)
    for a, b in zip(torch.autograd.grad(run()[0].sum(), base), want):
        assert torch.equal(a, b)
    strided = x["do"].transpose(2, 3).contiguous().transpose(2, 3)
    for a, b in zip(torch.autograd.grad(run()[0], base, strided), torch.autograd.grad(run()[0], base, x["do"])):
        assert torch.equal(a, b)
    full = torch.autograd.grad(run(), base, (torch.zeros_like(ones), x["ds"]))
    for a, b in zip(torch.autograd.grad(run()[1], base, x["ds"], allow_unused=True), full):
        assert torch.equal(a, b) if a is not None else not b.any()
    both = torch.autograd.grad(run(), base, (x["do"], x["ds"]))
    for i in range(4):
        only = [t if i == j else t.detach() for j, t in enumerate(base)]
        out = linear_attention(*only[:3], x["ld"], only[3], return_state=True)
        (g,) = torch.autograd.grad(out, base[i], (x["do"], x["ds"]))
        assert torch.equal(g, both[i])


def test_a_prompt_in_pieces_and_token_by_token():
    for dtype in DTYPES:
        x = _case(31, 2, 4, 300, 64, 48, dtype)
        whole, last = linear_attention(x["q"], x["k"], x["v"], x["ld"], x["s0"], return_state=True)
        state, size = x["s0"], layers.linear_attention_forward(
            *(abs(f64(x[n])) for n in ("q", "k", "v")), f64(x["ld"]), abs(f64(x["s0"])))
        parts = []
        for lo, hi in ((0, 1), (1, 130), (130, 257), (257, 300)):
            out, state = linear_attention(*(x[n][:, :, lo:hi] for n in ("q", "k", "v")), x["ld"], state, return_state=True)
            parts.append(out)
        _check(torch.cat(parts, 2), f64(whole), 2 * size[0], dtype, "pieces")
        assert_within(state, f64(last), 4000 * U * size[1], "state in pieces")
        state = x["s0"].clone()
        steps = [linear_attention_step(*(x[n][:, :, t] for n in ("q", "k", "v")), x["ld"], state) for t in range(300)]
        _check(torch.stack(steps, 2), f64(whole), 2 * size[0], dtype, "steps")
        assert_within(state, f64(last), 4000 * U * size[1], "state by steps")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,h,d,e", [(1, 1, 1, 1), (1, 16, 128, 128), (3, 5, 33, 17), (2, 4, 64, 128), (1, 2, 128, 36),
                                     (64, 16, 128, 96), (40, 16, 24, 64), (2, 3, 100, 2)])  # fmt: skip
def test_step(dtype, b, h, d, e):
    g = torch.Generator().manual_seed(b * h + d)
    q, k, v = (_randn(g, b, h, w, dtype=dtype) for w in (d, d, e))
    state = _randn(g, b, h, d, e)
    ld = -torch.rand(h, generator=g).to(DEV)
    args = [f64(t)[:, :, None] for t in (q, k, v)]
    want, last = layers.linear_attention_forward(*args, f64(ld), f64(state))
    size, ssize = layers.linear_attention_forward(*[abs(t) for t in args], f64(ld), abs(f64(state)))
    out = linear_attention_step(q, k, v, ld, state)
    # one update: the decay (3 U), two products and a sum; then a sum of d products
    assert_within(state, last, 8 * U * ssize, "state")
    want, size = want[:, :, 0], size[:, :, 0]
    assert_within(out, want, (140 + 8) * U * size + half(dtype) * abs(want) + smallest(dtype), "out")


def test_step_counts_as_a_change_of_the_state():
    """A state that a recorded call started from and a step then changed: the call's backward raises."""

    gen = torch.Generator(device=DEV).manual_seed(5)
    q, k, v = (torch.randn(1, 2, 6, 16, device=DEV, generator=gen) for _ in range(3))
    ld, state = torch.full((2,), -0.1, device=DEV), torch.randn(1, 2, 16, 16, device=DEV, generator=gen)
    out = linear_attention(q.requires_grad_(True), k, v, ld, state)
    with torch.no_grad():
        linear_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], ld, state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    with torch.inference_mode():
        own = torch.zeros(1, 2, 16, 16, device=DEV)
        linear_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], ld, own)
    assert bool(own.any())


def test_step_layouts():
    g = torch.Generator().manual_seed(41)
    qkv = _randn(g, 3, 1, 4, 3, 40, dtype=torch.bfloat16)
    q, k, v = (qkv[:, 0, :, i, 3:35] for i in range(3))  # rows inside wider ones
    shared = k[:, :1].expand(3, 4, 32)
    ld, s = torch.full((4,), -0.1, device=DEV), _randn(g, 3, 4, 32, 32)
    for qq, kk in ((q, k), (q, shared)):
        a, b = s.clone(), s.clone()
        got = linear_attention_step(qq, kk, v, ld, a)
        want = linear_attention_step(qq.contiguous(), kk.contiguous(), v.contiguous(), ld, b)
        assert torch.equal(got, want) and torch.equal(a, b)
    a = s.clone()
    assert torch.equal(linear_attention_step(q[0], k[0], v[0], ld, a[0]), linear_attention_step(q, k, v, ld, s.clone())[0])
    assert torch.equal(a[1:], s[1:])  # the other sequences' states as they were
    empty = linear_attention_step(q[:0], k[:0], v[:0], ld, s[:0])
    assert empty.shape == (0, 4, 32)


def test_no_tokens():
    x = _case(43, 2, 2, 3, 16, 16, torch.float32)
    q, k, v = (x[n][:, :, :0].detach().requires_grad_(True) for n in ("q", "k", "v"))
    s0 = x["s0"].detach().requires_grad_(True)
    out, state = linear_attention(q, k, v, x["ld"], s0, return_state=True)
    assert out.shape == (2, 2, 0, 16) and torch.equal(state, x["s0"])
    grads = torch.autograd.grad((out, state), (q, k, v, s0), (torch.empty_like(out), x["ds"]))
    assert torch.equal(grads[3], x["ds"])
    assert linear_attention(q[:0], k[:0], v[:0], x["ld"]).shape == (0, 2, 0, 16)
    assert not linear_attention(q.detach(), k.detach(), v.detach(), x["ld"], return_state=True)[1].any()


def test_non_finite_values_stay_with_their_tokens():
    """A NaN or an infinity in a value reaches its own column from its token on, and nothing before it."""

    for dtype in DTYPES:
        x = _case(47, 1, 2, 160, 32, 32, dtype, state=False)
        x["v"][0, 0, 70, 5] = float("inf")
        x["v"][0, 1, 100, 9] = float("nan")
        out = linear_attention(x["q"], x["k"], x["v"], x["ld"])
        fine = torch.isfinite(out)
        assert fine[0, 0, :70].all() and fine[0, 1, :100].all()
        assert not fine[0, 0, 70, 5] and not fine[0, 1, 100, 9]
        other = torch.ones(32, dtype=torch.bool, device=DEV)
        other[5] = False
        assert fine[0, 0][:, other].all()


def test_a_decay_that_is_nan():
    x = _case(49, 1, 2, 70, 32, 32, torch.bfloat16, state=False)
    x["ld"][1] = float("nan")
    out, state = linear_attention(x["q"], x["k"], x["v"], x["ld"], return_state=True)
    assert out[:, 1, 1:].isnan().all() and state[:, 1].isnan().all() and not out[:, 0].isnan().any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_offsets_past_32_bits(dtype):
    """Batch elements, heads and tokens further apart than 2^31 elements."""

    far = 2**31 + 64
    base = torch.empty(far + 3 * 64 * 200, dtype=dtype, device=DEV)
    ld = torch.tensor([-0.1, -0.02], device=DEV)
    g = torch.Generator().manual_seed(51)
    tight = [_randn(g, 2, 2, 50, 64, dtype=dtype) for _ in range(3)]
    for strides in ((far, 64 * 50, 64), (64 * 50, far, 64)):
        views = [base[64 * 200 * i :].as_strided((2, 2, 50, 64), (*strides, 1)) for i in range(3)]
        for v, t in zip(views, tight):
            v.copy_(t)
        got, want = (linear_attention(*ts, ld, return_state=True) for ts in (views, tight))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    del base, views
    apart = 2**26 + 8  # 33 tokens span more than 2^31 elements, 32 less
    base = torch.empty(34 * apart, dtype=dtype, device=DEV)
    q = base.as_strided((1, 1, 34, 64), (0, 0, apart, 1))
    small = _randn(g, 1, 1, 34, 64, dtype=dtype)
    q.copy_(small)
    assert torch.equal(linear_attention(q, q, q, ld[:1]), linear_attention(small, small, small, ld[:1]))
    state = torch.empty(2**17 + 1, 1, 128, 128, device=DEV)  # more than 2^31 elements
    state[-1], state[0] = 1.0, 2.0
    qs = torch.ones(2**17 + 1, 1, 128, device=DEV, dtype=dtype)
    out = linear_attention_step(qs, qs, qs, torch.zeros(1, device=DEV), state)
    assert (state[-1] == 2).all() and (state[0] == 3).all()
    assert torch.equal(out[-1].float(), torch.full((1, 128), 256 * 128**-0.5, device=DEV).to(dtype).float())


def test_refusals():
    x = _case(53, 1, 2, 8, 16, 16, torch.float32)
    q, k, v, ld, s0 = (x[n] for n in ("q", "k", "v", "ld", "s0"))
    big = torch.randn(1, 2, 8, 129, device=DEV)
    for call in (lambda: linear_attention(q.double(), k.double(), v.double(), ld), lambda: linear_attention(q, k, v.half(), ld),
                 lambda: linear_attention(big, big, v, ld), lambda: linear_attention(q, k, big, ld),
                 lambda: linear_attention(q, k, v, ld.double()), lambda: linear_attention(q, k, v, ld, s0.half()),
                 lambda: linear_attention(q, k, v, ld.clone().requires_grad_(True)),
                 lambda: linear_attention(q, k, v, ld, lengths=torch.ones(1, device=DEV)),
                 lambda: linear_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], ld, s0.transpose(2, 3)),
                 lambda: linear_attention_step(q[:, :, 0].clone().requires_grad_(True), k[:, :, 0], v[:, :, 0], ld, s0)):  # fmt: skip
        with pytest.raises(OOpsUnsupportedError):
            call()
    with pytest.raises(ValueError):
        linear_attention(q, k, v, ld.cpu())
    leaf = q.detach().requires_grad_(True)
    (dq,) = torch.autograd.grad(linear_attention(leaf, k, v, ld).square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        dq.sum().backward()
    with pytest.raises(OOpsUnsupportedError):
        linear_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], ld, torch._neg_view(s0))


def test_compile():
    x = _case(59, 2, 2, 150, 64, 64, torch.bfloat16)

    def run(q, k, v, s0):
        return linear_attention(q, k, v, x["ld"], s0, return_state=True)

    results = []
    for fn in (run, torch.compile(run, fullgraph=True)):
        leaves = [x[n].detach().clone().requires_grad_(True) for n in ("q", "k", "v", "s0")]
        outs = fn(*leaves)
        results.append((*outs, *torch.autograd.grad(outs, leaves, (x["do"], x["ds"]))))
    for got, ref in zip(*results):
        torch.testing.assert_close(got, ref, atol=0, rtol=0)
    with torch.no_grad():
        states = [x["s0"].clone() for _ in range(2)]
        step = lambda s: linear_attention_step(x["q"][:, :, 0], x["k"][:, :, 0], x["v"][:, :, 0], x["ld"], s)  # noqa: E731
        assert torch.equal(torch.compile(step, fullgraph=True)(states[0]), step(states[1]))
        assert torch.equal(*states)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_graph_replays(dtype):
    """A training step and a decoding step captured, replayed over changing inputs and lengths, eager work between."""

    x = _case(61, 3, 2, 260, 64, 64, dtype)
    lengths = torch.tensor([260, 100, 7], dtype=torch.int32, device=DEV)
    state = x["s0"].clone()

    def run():
        leaves = [x[n].detach().requires_grad_(True) for n in ("q", "k", "v", "s0")]
        outs = linear_attention(*leaves[:3], x["ld"], leaves[3], lengths, return_state=True)
        return (*(t.detach() for t in outs), *torch.autograd.grad(outs, leaves, (x["do"], x["ds"])))

    def step(s):
        return linear_attention_step(x["q"][:, :, 0], x["k"][:, :, 0], x["v"][:, :, 0], x["ld"], s)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = (*run(), step(state))
    eager = state.clone()
    for i in range(3):
        y = _case(70 + i, 3, 2, 260, 64, 64, dtype)
        for n in ("q", "k", "v", "do"):
            x[n].copy_(y[n])
        lengths.copy_(torch.tensor([13 * i, 260 - i, 64], dtype=torch.int32))
        graph.replay()
        want = (*run(), step(eager))
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b), i
        assert torch.equal(state, eager)


def test_two_streams():
    xs = [_case(80 + i, 2, 4, 1000, 64, 64, torch.bfloat16) for i in range(2)]
    run = lambda x: linear_attention(x["q"], x["k"], x["v"], x["ld"], x["s0"], return_state=True)  # noqa: E731
    want = [run(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(6):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].append(run(xs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for got in outs[i] for a, b in zip(got, want[i]))


def test_into_the_gated_output_stage():
    """The result of token-major operands goes into gate_attention_output as it is, like pair_bias_attention's."""

    x = _case(83, 2, 4, 100, 32, 32, torch.bfloat16)
    g = torch.Generator().manual_seed(84)
    single = _randn(g, 2, 100, 128, dtype=torch.bfloat16)
    wg, wo = (_randn(g, 128, 128, dtype=torch.bfloat16, scale=128**-0.5) for _ in range(2))
    out = linear_attention(x["q"], x["k"], x["v"], x["ld"])
    assert out.transpose(1, 2).is_contiguous()
    got = gate_attention_output(out, single, wg, wo)
    assert torch.equal(got, gate_attention_output(out.contiguous(), single, wg, wo))


def test_compile_with_sizes_that_change():
    """One compiled function over several lengths and batches: the second one makes the sizes dynamic."""

    def run(q, k, v, ld, s0):
        return linear_attention(q, k, v, ld, s0, return_state=True)

    compiled = torch.compile(run, fullgraph=True)
    for b, n in ((2, 150), (2, 70), (3, 201), (2, 64)):
        x = _case(63, b, 2, n, 64, 32, torch.bfloat16)
        results = []
        for fn in (run, compiled):
            leaves = [x[name].detach().clone().requires_grad_(True) for name in ("q", "k", "v", "s0")]
            outs = fn(*leaves[:3], x["ld"], leaves[3])
            results.append((*outs, *torch.autograd.grad(outs, leaves, (x["do"], x["ds"]))))
        for got, ref in zip(*results):
            torch.testing.assert_close(got, ref, atol=0, rtol=0)


def _gradients_and_results(x):
    """(name, the operator's, the recurrence's), of the first and last batch element's first and last head."""

    names = ("q", "k", "v", "s0")
    b, h = x["q"].shape[:2]
    ends = lambda t: t[:: max(b - 1, 1), :: max(h - 1, 1)]  # noqa: E731
    leaves = [x[name].detach().requires_grad_(True) for name in names]
    outs = linear_attention(*leaves[:3], x["ld"], leaves[3], return_state=True)
    got = [t.detach() for t in (*outs, *torch.autograd.grad(outs, leaves, (x["do"], x["ds"])))]
    q, k, v, s0, do, ds = (f64(ends(x[name])) for name in (*names, "do", "ds"))
    ld = f64(x["ld"])[:: max(h - 1, 1)]
    with np.errstate(invalid="ignore"):
        want = layers.linear_attention_forward(q, k, v, ld, s0)
        want += layers.linear_attention_backward(q, k, v, ld, do, ds, s0)
    return zip(("out", "state", "dq", "dk", "dv", "dinitial"), map(ends, got), want, strict=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,e,b,h", [(32, 32, 1, 2), (40, 24, 2, 1), (64, 64, 1, 2), (128, 128, 1, 2), (128, 64, 2, 1),
                                     (64, 64, 32, 12), (128, 128, 16, 12)])  # fmt: skip
def test_non_finite_operands(dtype, d, e, b, h):
    """An infinity or a NaN in any operand or gradient: results are finite exactly where the recurrence's are, with
    one, two and four waves a workgroup, in segments and in one."""

    for i, (name, value) in enumerate([("v", "inf"), ("v", "nan"), ("k", "-inf"), ("q", "inf"), ("do", "inf"), ("s0", "nan"),
                                       ("ds", "inf")]):  # fmt: skip
        x = _case(67 + i, b, h, 150, d, e, dtype)
        x["ld"] = torch.linspace(-0.3, -0.01, h, device=DEV)
        row = 70 if name not in ("s0", "ds") else 3
        x[name][0, -1, row, 5] = float(value)
        for what, got, want in _gradients_and_results(x):
            assert np.array_equal(np.isfinite(f64(got)), np.isfinite(want)), f"{what}: {value} in {name}"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("decay", [float("-inf"), -200.0])
def test_non_finite_operands_and_no_memory(dtype, decay):
    """A head without memory multiplies what it forgets by zero: after an infinity its column is NaN, as the
    recurrence's is; the other heads stay finite."""

    x = _case(75, 1, 2, 150, 32, 32, dtype)
    x["ld"] = torch.tensor([decay, -0.01], device=DEV)
    x["v"][0, 0, 70, 5] = float("inf")
    out, state = linear_attention(x["q"], x["k"], x["v"], x["ld"], x["s0"], return_state=True)
    with np.errstate(invalid="ignore"):
        want, last = layers.linear_attention_forward(*(f64(x[n]) for n in ("q", "k", "v", "ld", "s0")))
    assert np.array_equal(np.isfinite(f64(out)), np.isfinite(want))
    assert np.array_equal(np.isfinite(f64(state)), np.isfinite(last))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,b,h", [(32, 1, 2), (64, 1, 2), (128, 1, 2), (128, 16, 12)])
def test_an_infinite_value_leaves_an_infinity_in_the_state(dtype, d, b, h):
    """Positive keys and queries: the state's column and the outputs are that infinity, not NaN; so is a gradient's."""

    x = _case(77, b, h, 150, d, d, dtype)
    x["ld"] = torch.linspace(-0.1, -0.01, h, device=DEV)
    for name in ("q", "k"):
        x[name] = x[name].abs() + 0.125
    x["v"][0, -1, 70, 5] = float("-inf")
    x["do"][0, 0, 30, 7] = float("inf")
    for what, got, want in _gradients_and_results(x):
        if what in ("out", "state", "dv", "dinitial"):
            got = f64(got)
            assert np.array_equal(np.isnan(got), np.isnan(want)), what
            assert np.array_equal(np.where(np.isinf(got), got, 0), np.where(np.isinf(want), want, 0)), what
