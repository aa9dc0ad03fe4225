"""GPU parity of int8_linear with exact integer sums.

Tolerances: the sum is exact; its conversion to float32, two products and the bias's addition are off by U each
relative to the scaled sum (the last also to the result), then one rounding to the result's type.
"""

import pytest
import torch

from layer_tolerance import U, assert_within, f64, half, smallest
from oops_amd import OOpsUnsupportedError, int8_linear
from oracle import layers

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _operands(rows, k, n, seed=0, low=-128):
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(low, 128, (rows, k), generator=g, dtype=torch.int8)
    w = torch.randint(low, 128, (n, k), generator=g, dtype=torch.int8)
    xs, ws = torch.rand(rows, generator=g) + 0.5, (torch.rand(n, generator=g) + 0.5) / (74 * 74 * max(k, 1) ** 0.5)
    return [t.to(DEV) for t in (x, xs, w, ws)], torch.randn(n, generator=g).to(DEV)


def _check(out, x, xs, w, ws, bias, dtype):
    assert out.dtype == dtype
    xi, wi = (t.cpu().numpy() for t in (x, w))
    base = layers.int8_linear(xi, f64(xs), wi, f64(ws))
    want = base if bias is None else base + f64(bias)
    bound = 4 * U * abs(base) + (half(dtype) + U) * abs(want) + smallest(dtype)
    assert_within(out, want, bound, "out")


SIZES = [(1, 64, 16), (1, 4096, 4096), (3, 100, 5), (4, 1024, 1000), (16, 512, 96), (17, 2064, 130), (33, 256, 257),
         (64, 4096, 512), (65, 640, 64), (100, 1, 1), (130, 77, 300), (256, 1536, 768), (333, 1001, 777), (600, 528, 1040),
         (1, 131071, 3), (1025, 320, 2050), (2048, 1024, 2048)]  # fmt: skip


@pytest.mark.parametrize("rows,k,n", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_sizes(rows, k, n, dtype):
    args, bias = _operands(rows, k, n, seed=k)
    _check(int8_linear(*args, dtype=dtype), *args, None, dtype)
    _check(int8_linear(*args, bias, dtype=dtype), *args, bias, dtype)
    if dtype != torch.float32:
        b = bias.to(dtype)
        _check(int8_linear(*args, b, dtype=dtype), *args, b, dtype)


@pytest.mark.parametrize("rows,k,n", [(20, 8192, 100), (70, 16400, 72), (128, 9008, 256), (17, 65536, 16)])
def test_long_sums_of_few_outputs(rows, k, n):
    """k in parts that are joined: whole and partial last ones; and a longer call right behind a shorter one."""

    args, bias = _operands(rows, k, n, seed=k)
    _check(int8_linear(*args, bias, dtype=torch.float32), *args, bias, torch.float32)
    _check(int8_linear(*args), *args, None, torch.bfloat16)


@pytest.mark.parametrize("rows,k,n,xpad,wpad", [(1025, 1001, 1100, 0, 0), (700, 2064, 900, 3, 0), (700, 2064, 900, 0, 5),
                                                 (300, 8201, 600, 7, 9)])  # fmt: skip
def test_many_products_of_odd_rows(rows, k, n, xpad, wpad):
    """Rows that are no whole 16-byte pieces, copied to padded ones where there are many products."""

    (x, xs, w, ws), bias = _operands(rows, k, n, seed=k + xpad)
    wide = lambda t, pad: torch.full((t.shape[0], k + pad), 99, dtype=torch.int8, device=DEV)[:, :k]  # noqa: E731
    xv, wv = wide(x, xpad).copy_(x), wide(w, wpad).copy_(w)
    _check(int8_linear(xv, xs, wv, ws, bias), x, xs, w, ws, bias, torch.bfloat16)


@pytest.mark.parametrize("rows,k,n", [(500, 1001, 1000), (570, 333, 1050), (31, 777, 95), (64, 5, 64), (200, 2049, 33)])
def test_fewer_products_of_odd_rows(rows, k, n):
    """Few tiles, and more of them."""

    args, bias = _operands(rows, k, n, seed=k)
    _check(int8_linear(*args, bias), *args, bias, torch.bfloat16)
    _check(int8_linear(*args, dtype=torch.float32), *args, None, torch.float32)


def test_more_than_32_bits_of_results():
    rows, n, k = 40003, 54000, 32
    (x, xs, w, ws), bias = _operands(rows, k, n, seed=7)
    out = int8_linear(x, xs, w, ws, bias)
    for r in (0, 20001, rows - 1):
        assert torch.equal(out[r : r + 1], int8_linear(x[r : r + 1], xs[r : r + 1], w, ws, bias))


@pytest.mark.parametrize("rows", [1, 7, 40, 300])
@pytest.mark.parametrize("value", [-128, 127])
def test_largest_sums(rows, value):
    """Every product at its largest: the 32-bit sums hold 131071 of them."""

    k, n = 131056 if rows == 1 else 16384, 48
    x = torch.full((rows, k), value, dtype=torch.int8, device=DEV)
    w = torch.full((n, k), -128, dtype=torch.int8, device=DEV)
    xs, ws = torch.ones(rows, device=DEV), torch.full((n,), 2.0**-20, device=DEV)
    _check(int8_linear(x, xs, w, ws, dtype=torch.float32), x, xs, w, ws, None, torch.float32)


@pytest.mark.parametrize("rows", [2, 20, 150])
@pytest.mark.parametrize("k,offset,pad", [(256, 0, 16), (256, 0, 3), (256, 16, 32), (256, 5, 16), (250, 0, 6), (248, 8, 8)])
def test_row_strides_and_offsets(rows, k, offset, pad):
    """Rows inside wider ones, at aligned and unaligned places: bytes around them must not count."""

    (x, xs, w, ws), bias = _operands(rows, k, 200, seed=offset + pad)
    wide = lambda t: torch.full((t.shape[0], offset + k + pad), 77, dtype=torch.int8, device=DEV)  # noqa: E731
    xw, ww = wide(x), wide(w)
    xv, wv = xw[:, offset : offset + k], ww[:, offset : offset + k]
    xv.copy_(x), wv.copy_(w)
    want = int8_linear(x.contiguous(), xs, w.contiguous(), ws, bias, dtype=torch.float32)
    assert torch.equal(int8_linear(xv, xs, wv, ws, bias, dtype=torch.float32), want)
    _check(want, x, xs, w, ws, bias, torch.float32)


def test_prefixes_transposes_and_empty():
    (x, xs, w, ws), bias = _operands(24, 64, 40)
    flat = int8_linear(x, xs, w, ws, bias)
    out = int8_linear(x.view(2, 3, 4, 64), xs.view(2, 3, 4), w, ws, bias)
    assert out.shape == (2, 3, 4, 40) and torch.equal(out.view(24, 40), flat)
    assert torch.equal(int8_linear(x[0], xs[0], w, ws, bias), flat[0])
    assert torch.equal(int8_linear(x, xs, w.t().contiguous().t(), ws, bias), flat)
    assert torch.equal(int8_linear(x[:1].expand(5, 64), xs[:1].expand(5), w, ws, bias), flat[:1].expand(5, 40))
    assert int8_linear(x[:0], xs[:0], w, ws).shape == (0, 40)
    assert int8_linear(x, xs, w[:0], ws[:0]).shape == (24, 0)
    none = int8_linear(x[:, :0], xs, w[:, :0], ws, bias, dtype=torch.float32)  # no features: the bias
    assert torch.equal(none, bias.expand(24, 40))


def test_scales_that_are_not_finite():
    (x, xs, w, ws), _ = _operands(20, 64, 40)
    xs[3], ws[7] = float("nan"), float("inf")
    out = int8_linear(x, xs, w, ws)
    assert out[3].isnan().all() and not out[:3, :7].isnan().any() and not out[4:, 8:].isnan().any()


def test_refusals():
    (x, xs, w, ws), bias = _operands(4, 32, 8)
    for call in (lambda: int8_linear(x, xs, w.half(), ws), lambda: int8_linear(x, xs.half(), w, ws),
                 lambda: int8_linear(x, xs, w, ws, bias.double()), lambda: int8_linear(x, xs, w, ws, dtype=torch.float64),
                 lambda: int8_linear(x, xs, w, ws, bias.half(), dtype=torch.bfloat16),
                 lambda: int8_linear(x, xs, w, ws.clone().requires_grad_(True))):  # fmt: skip
        with pytest.raises(OOpsUnsupportedError):
            call()
    big = torch.zeros(1, 131072, dtype=torch.int8, device=DEV)
    with pytest.raises(OOpsUnsupportedError):
        int8_linear(big, xs[:1], big, ws[:1])
    with pytest.raises(ValueError):
        int8_linear(x, xs.cpu(), w, ws)


def test_compile_and_graph():
    for rows in (3, 200):
        args, bias = _operands(rows, 512, 384, seed=rows)
        want = int8_linear(*args, bias)
        got = torch.compile(lambda a, b, c, d, e: int8_linear(a, b, c, d, e), fullgraph=True)(*args, bias)
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = int8_linear(*args, bias)
        for k in range(3):
            args[0].copy_(_operands(rows, 512, 384, seed=100 + k)[0][0])
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, int8_linear(*args, bias)), k


def test_two_streams():
    """Two calls of one shape at once, each with a workspace of its own."""

    a, b = (_operands(48, 4096, 640, seed=s)[0] for s in (1, 2))
    want = [int8_linear(*t) for t in (a, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(8):
        for i, t in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                outs[i].append(int8_linear(*t))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])


def test_lazily_negated_operands():
    args, bias = _operands(5, 48, 20, low=-127)
    want = int8_linear(*args, bias)
    for i in range(5):
        ops = [torch._neg_view(-t) if i == j else t for j, t in enumerate((*args, bias))]
        assert ops[i].is_neg()
        assert torch.equal(int8_linear(*ops), want)
