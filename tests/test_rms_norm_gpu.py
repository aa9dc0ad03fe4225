"""GPU parity of rms_norm, rms_norm_int8 and quantize_int8 with the float64 definitions (oracle/layers.py).

Tolerances: one rounding to the result's type, plus float32 arithmetic.  A row's sums run over at most 64 values
a lane and eight joining steps: 72 U of the terms' magnitudes, and half of it for the square root; 64 U covers the
statistics and the three products of a value.
"""

import pytest
import torch

import oops_amd
from layer_tolerance import U, assert_within, f64, half, smallest
from nested_standin import NestedTensor
from oops_amd import OOpsUnsupportedError, RMSNorm, quantize_int8, rms_norm, rms_norm_int8
from oracle import layers

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ARITH = 64 * U


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def _sum(x, r):
    """What the operator defines: the float32 sum rounded to the dtype."""

    return x if r is None else (x.float() + r.float()).to(x.dtype)


def _check_forward(y, h, w, dtype, eps=1e-6):
    want = layers.rms_norm_forward(f64(h), f64(w), eps)
    assert y.dtype == dtype
    assert_within(y, want, (half(dtype) + ARITH) * abs(want) + smallest(dtype), "y")


def _check_backward(got, h, dy, dsum, w, dtype, rows_per_sum):
    dx, dw = layers.rms_norm_backward(f64(h), f64(dy), f64(w))
    rstd = 1 / ((f64(h) ** 2).mean(-1, keepdims=True) + 1e-6) ** 0.5
    n, g = abs(f64(h)) * rstd, abs(f64(dy)) * (1 if w is None else abs(f64(w)))
    size = rstd * (g + n * (g * n).mean(-1, keepdims=True))  # magnitudes of the terms of dx
    if dsum is not None:
        dx, size = dx + f64(dsum), size + abs(f64(dsum))
    assert_within(got[0], dx, half(dtype) * abs(dx) + 2 * ARITH * size + smallest(dtype), "dx")
    if w is not None:
        terms = (abs(f64(dy)) * n).sum(0)
        # a chain of the rows one workgroup adds, its 16 groups, the partials' chunks
        bound = half(w.dtype) * abs(dw) + (ARITH + (rows_per_sum + 16 + 160) * U) * terms + smallest(w.dtype)
        assert_within(got[1], dw, bound, "dweight")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [1, 17, 128, 384, 1000, 2048, 4104, 16384])
@pytest.mark.parametrize("residual,weight", [(False, "same"), (True, "f32"), (True, None)])
def test_rms_norm(dtype, width, residual, weight):
    g = torch.Generator().manual_seed(width)
    rows = 1500 if width <= 384 else 67
    x = _randn(g, rows, width, dtype=dtype, scale=2).requires_grad_(True)
    r = _randn(g, rows, width, dtype=dtype).requires_grad_(True) if residual else None
    w = None if weight is None else _randn(g, width, dtype=dtype if weight == "same" else torch.float32).requires_grad_(True)
    h = _sum(x, r).detach()
    dy, ds = _randn(g, rows, width, dtype=dtype), _randn(g, rows, width, dtype=dtype) if residual else None
    leaves = [t for t in (x, w, r) if t is not None]
    if residual:
        y, summed = rms_norm(x, width, w, residual=r)
        assert torch.equal(summed, h)
        grads = list(torch.autograd.grad((y, summed), leaves, (dy, ds)))
        assert torch.equal(grads[0], grads.pop())  # the residual's gradient is the input's
    else:
        y = rms_norm(x, (width,), w)
        grads = torch.autograd.grad(y, leaves, dy)
    _check_forward(y, h, w, dtype)
    _check_backward(grads, h, dy, ds, w, dtype, 2)
    if w is not None:
        assert grads[1].dtype == w.dtype


def test_many_rows_and_repeated_calls():
    """More rows than the backward's grid: each workgroup walks several; sums are the same bits every time."""

    g = torch.Generator().manual_seed(3)
    x, w = _randn(g, 70001, 64, dtype=torch.bfloat16), _randn(g, 64)
    dy = _randn(g, 70001, 64, dtype=torch.bfloat16)
    x.requires_grad_(True), w.requires_grad_(True)
    runs = [torch.autograd.grad(rms_norm(x, 64, w), (x, w), dy) for _ in range(2)]
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    _check_backward(runs[0], x, dy, None, w, torch.bfloat16, 16)


def test_more_than_32_bits_of_elements():
    rows, width = 2**17 + 3, 16384
    x = torch.empty(rows, width, dtype=torch.bfloat16, device=DEV)
    x.fill_(1.0)
    x[-1].normal_(), x[0].normal_()
    y = rms_norm(x, width)
    values, scales = quantize_int8(x)
    for i in (0, rows - 1):
        assert torch.equal(y[i], rms_norm(x[i], width))
        assert torch.equal(values[i], quantize_int8(x[i])[0]) and torch.equal(scales[i], quantize_int8(x[i])[1])
    assert (values[1:-1] == 127).all()


def test_strides_and_prefixes():
    g = torch.Generator().manual_seed(5)
    base, rbase = (_randn(g, 3, 20, 80, dtype=torch.bfloat16) for _ in range(2))
    w = _randn(g, 64)
    for x, r in ((base[:, :, :64], rbase[:, :, 8:72]), (base[:, :, 1:65], rbase[:, :, :64]),
                 (base.transpose(1, 2)[:, :64].transpose(1, 2), rbase[..., :64]),
                 (base[:1, :1, :64].expand(3, 20, 64), rbase[..., :64])):  # fmt: skip
        y, summed = rms_norm(x, 64, w, residual=r)
        h = _sum(x, r)
        assert y.shape == x.shape and torch.equal(summed, h)
        _check_forward(y, h, w, torch.bfloat16)
        values, scales, again = rms_norm_int8(x, 64, w, residual=r)
        assert values.shape == x.shape and scales.shape == x.shape[:-1] and torch.equal(again, h)
        assert _check_int8(values, scales, layers.rms_norm_forward(f64(h), f64(w)))
    one = _randn(g, 64, dtype=torch.float16)
    _check_forward(rms_norm(one, 64), one, None, torch.float16)


def test_only_one_output_used_and_views_of_gradients():
    g = torch.Generator().manual_seed(6)
    x, r, w = (_randn(g, 9, 32).requires_grad_(True), _randn(g, 9, 32).requires_grad_(True), _randn(g, 32).requires_grad_(True))
    dy = _randn(g, 32, 9).t()  # not contiguous
    y, summed = rms_norm(x, 32, w, residual=r)
    got = torch.autograd.grad(y, (x, w, r), dy, retain_graph=True)
    _check_backward(got, _sum(x, r), dy, None, w, torch.float32, 2)
    first = got[2]
    dx, dw, dr = torch.autograd.grad(summed, (x, w, r), dy, allow_unused=True, retain_graph=True)
    assert torch.equal(dx, dy) and torch.equal(dr, dy) and (dw is None or not dw.any())
    got = torch.autograd.grad(y.sum(), (x, w), retain_graph=True)  # an expanded gradient
    _check_backward(got, _sum(x, r), torch.ones_like(x), None, w, torch.float32, 2)
    (dr,) = torch.autograd.grad(y, (r,), dy)  # the residual alone
    assert torch.equal(dr, first)
    x0 = x.detach()
    with torch.no_grad():
        assert torch.equal(rms_norm(x0, 32, w), rms_norm(x, 32, w))
    neg = torch._neg_view(x0)
    assert torch.equal(rms_norm(neg, 32, w.detach()), rms_norm(-x0, 32, w.detach()))


def test_no_rows():
    x = torch.empty(0, 16, device=DEV, requires_grad=True)
    w = torch.ones(16, device=DEV, requires_grad=True)
    y, s = rms_norm(x, 16, w, residual=torch.empty(0, 16, device=DEV))
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert y.shape == s.shape == dx.shape == (0, 16) and not dw.any()
    assert quantize_int8(x.detach())[1].shape == (0,)


def test_second_derivative_raises():
    x = torch.randn(4, 8, device=DEV, requires_grad=True)
    (dx,) = torch.autograd.grad(rms_norm(x, 8).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        dx.sum().backward()


def _check_int8(values, scales, y, arith=2 * ARITH):
    """Values within half a step (and arithmetic) of y / scale, scales to float32 arithmetic."""

    q, s = layers.quantize_rows(y)
    assert values.dtype == torch.int8 and scales.dtype == torch.float32
    assert_within(scales, s, arith * s + 2.0**-149, "scales")
    assert_within(values, q, 0.5 + 127 * arith, "values")
    return True


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [1, 17, 200, 1024, 5000, 8192])
def test_int8_rows(dtype, width):
    g = torch.Generator().manual_seed(width + 1)
    x, r, w = _randn(g, 33, width, dtype=dtype), _randn(g, 33, width, dtype=dtype), _randn(g, width)
    values, scales = rms_norm_int8(x, width, w)
    _check_int8(values, scales, layers.rms_norm_forward(f64(x), f64(w)))
    values, scales, summed = rms_norm_int8(x, width, None, residual=r)
    assert torch.equal(summed, _sum(x, r))
    _check_int8(values, scales, layers.rms_norm_forward(f64(summed)))
    values, scales = quantize_int8(x)
    # the largest magnitude of a row is +-127, what lies between two steps rounds to the nearer one, ties to even
    _check_int8(values, scales, f64(x), arith=4 * U)
    assert (values.abs().amax(-1) == 127).all()


@pytest.mark.parametrize("width", [40, 41, 4096])
def test_int8_special_rows(width):
    x = torch.randn(6, width, device=DEV)
    x[0] = 0
    x[1, -1] = float("nan")
    x[2, 0] = float("-inf")
    x[3] *= 1e-40  # subnormal
    x[4] *= 1e37
    values, scales = quantize_int8(x)
    assert scales[0] == 0 and not values[0].any()
    assert scales[1:3].isnan().all() and not values[1:3].any()
    _check_int8(values[4:], scales[4:], f64(x[4:]), arith=4 * U)
    q, s = layers.quantize_rows(f64(x[3:4]))
    assert_within(scales[3:4], s, 2.0**-149, "subnormal scale")
    assert_within(values[3:4], q, 0.5 + 1e-3, "subnormal values")
    y = rms_norm(x[1:3], width)
    assert y[0].isnan().all()
    zeros = rms_norm_int8(torch.zeros(2, width, device=DEV), width)
    assert not zeros[0].any() and not zeros[1].any()


def test_refusals():
    x, i = torch.randn(4, 8, device=DEV), torch.zeros(4, 8, device=DEV, dtype=torch.int32)
    for call in (lambda: rms_norm(x.double(), 8), lambda: rms_norm(x, 7), lambda: rms_norm(x, 8, torch.ones(4, device=DEV)),
                 lambda: rms_norm(x, 8, torch.ones(8, device=DEV, dtype=torch.bfloat16)), lambda: quantize_int8(i),
                 lambda: rms_norm(x, 8, residual=x.half()), lambda: rms_norm(torch.randn(1, 16385, device=DEV), 16385),
                 lambda: rms_norm_int8(x.clone().requires_grad_(True), 8)):  # fmt: skip
        with pytest.raises(OOpsUnsupportedError):
            call()
    with pytest.raises(ValueError):
        rms_norm(x, 8, residual=x[:1])
    with pytest.raises(ValueError):
        rms_norm(x, 8, torch.ones(8))


def test_module_and_nested():
    m = RMSNorm(96, eps=1e-5).to(DEV)
    with torch.no_grad():
        m.weight.normal_()
    x, r = (torch.randn(5, 7, 96, device=DEV).bfloat16() for _ in range(2))
    _check_forward(m(x), x, m.weight, torch.bfloat16, 1e-5)
    y, s = m(x, r)
    assert torch.equal(s, _sum(x, r))
    _check_forward(y, s, m.weight, torch.bfloat16, 1e-5)
    m64 = RMSNorm(96).to(DEV).double()  # declined: PyTorch's own
    x64 = x.double()
    torch.testing.assert_close(m64(x64), torch.nn.functional.rms_norm(x64, (96,), m64.weight))
    torch.testing.assert_close(m64(x64, x64)[1], 2 * x64)
    tmpl = NestedTensor([torch.empty(n, 3, 32) for n in (5, 9)], ragged_dims=(0,))
    a, b = (tmpl.packed_like(torch.randn(tmpl.concat.shape, device=DEV)) for _ in range(2))
    _check_forward(rms_norm(a, 32).concat, a.concat, None, torch.float32)
    y, s = rms_norm(a, 32, residual=b)
    assert torch.equal(s.concat, a.concat + b.concat)
    _check_forward(y.concat, s.concat, None, torch.float32)
    with pytest.raises(ValueError):
        rms_norm(a, 32, residual=b.concat)


def test_compile_and_fake():
    g = torch.Generator().manual_seed(8)
    x0, r0, w = _randn(g, 64, 96, dtype=torch.bfloat16), _randn(g, 64, 96, dtype=torch.bfloat16), _randn(g, 96).requires_grad_(True)
    dy = _randn(g, 64, 96, dtype=torch.bfloat16)

    def run(x, r):
        y, s = rms_norm(x, 96, w, residual=r)
        return y, s

    results = []
    for fn in (run, torch.compile(run, fullgraph=True)):
        x, r = x0.clone().requires_grad_(True), r0.clone().requires_grad_(True)
        out = fn(x, r)
        results.append((*out, *torch.autograd.grad(out, [x, r, w], (dy, dy))))
    for got, ref in zip(*results):
        torch.testing.assert_close(got, ref, atol=0, rtol=0)
    with torch.no_grad():
        got = torch.compile(lambda x: (*rms_norm_int8(x, 96, w), *quantize_int8(x)), fullgraph=True)(x0)
        for a, b in zip(got, (*rms_norm_int8(x0, 96, w), *quantize_int8(x0))):
            assert torch.equal(a, b)


def test_graph_replays():
    """Forward, backward and the 8-bit rows captured into one graph, replayed over changing inputs with eager work
    between the replays."""

    g = torch.Generator().manual_seed(9)
    x, r, w = _randn(g, 700, 256, dtype=torch.float16), _randn(g, 700, 256, dtype=torch.float16), _randn(g, 256)
    dy = _randn(g, 700, 256, dtype=torch.float16)

    def run():
        xs, rs, ws = (t.detach().requires_grad_(True) for t in (x, r, w))
        y, s = rms_norm(xs, 256, ws, residual=rs)
        grads = torch.autograd.grad((y, s), (xs, ws, rs), (dy, dy))
        with torch.no_grad():
            return (y.detach(), s.detach(), *grads, *rms_norm_int8(x, 256, w))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for k in range(3):
        x.copy_(_randn(g, 700, 256, dtype=torch.float16))
        graph.replay()
        want = run()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b), k


def test_other_stream():
    g = torch.Generator().manual_seed(10)
    x = _randn(g, 512, 512)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        big = x + 1
        got = oops_amd.rms_norm(big, 512)
    torch.cuda.current_stream().wait_stream(side)
    _check_forward(got, x + 1, None, torch.float32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [1e-4, 0.02, 1.0])
def test_default_eps_of_the_module(dtype, scale):
    """A module of default eps against PyTorch's, on rows small enough that the eps decides the result: each result is
    rounded once, and a gradient of the type is off by one rounding and the arithmetic of its terms on either side."""

    g = torch.Generator().manual_seed(21)
    ours, theirs = (m(96, device=DEV, dtype=dtype) for m in (RMSNorm, torch.nn.RMSNorm))
    x, dy = _randn(g, 40, 96, dtype=dtype, scale=scale), _randn(g, 40, 96, dtype=dtype)
    eps = torch.finfo(torch.float32).eps
    _check_forward(ours(x), x, None, dtype, eps)
    want = f64(theirs(x))
    assert_within(ours(x), want, (2 * half(dtype) + 2 * ARITH) * abs(want) + 2 * smallest(dtype), "y")
    y, s = ours(x, x)
    _check_forward(y, s, None, dtype, eps)
    leaf = x.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(ours(leaf), leaf, dy)
    h, want_dx = f64(x), layers.rms_norm_backward(f64(x), f64(dy), None, eps)[0]
    rstd = 1 / ((h**2).mean(-1, keepdims=True) + eps) ** 0.5
    n, d = abs(h) * rstd, abs(f64(dy))
    size = rstd * (d + n * (d * n).mean(-1, keepdims=True))
    assert_within(dx, want_dx, half(dtype) * abs(want_dx) + 2 * ARITH * size + smallest(dtype), "dx")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [24, 1000, 4096])
def test_int8_values_are_the_exact_quotients(dtype, width):
    """rint(x 127 / max|row|) with ties to even: half the largest lies exactly between 63 and 64.  16-bit rows have the
    values of exact arithmetic everywhere: with significands of p bits, a quotient that is no tie n + 1/2 is at least
    1 / (254 2^p) of itself away from one (254 x and (2 n + 1) max|row| are different whole multiples of one power of
    two, the first below 254 2^p of them), 2^-19 in float16, where float32 arithmetic is off by a few 2^-24."""

    g = torch.Generator().manual_seed(31)
    x = _randn(g, 700, width, dtype=dtype)
    x[:, 0] = x.abs().amax(-1) * 1.5
    x[:, 1], x[:, 2] = x[:, 0] / 2, x[:, 0] / -2
    x[350:] *= -1
    for scale in (1.0, 2.0**-9, 2.0**7) if dtype == torch.float16 else (1.0, 2.0**-110, 2.0**120):
        rows = x * scale
        values, _ = quantize_int8(rows)
        y = rows.double()
        want = torch.round(y * 127 / y.abs().amax(-1, keepdim=True))
        assert (values[:, 1:3].abs() == 64).all()
        if dtype != torch.float32:
            assert torch.equal(values.double(), want)
        assert (values.double() - want).abs().max() <= 1
    values, _ = rms_norm_int8(x, width)  # (a norm without weight keeps the half exactly)
    assert (values[:, 1:3].abs() == 64).all()
