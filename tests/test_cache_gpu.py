"""GPU parity of the 4-bit key/value cache: cache_write, cache_read and cache_attention with float64 (oracle/decoder.py).

Codes and exponents are those of exact arithmetic, bit for bit.  Attention (U: half a step of float32, h: of the query's
type): what the codes stand for and the query enter exactly, as bfloat16 terms; a score is off by (3 D + 8) U of its
products' magnitudes (three terms in float32), so a weight by that, once for itself and once for the sum, and n U + 16 U for
the sum and the exponent; bfloat16 rounds a weight as an operand (h), float16 and float32 keep 16 and 24 bits of it;
sums of n products are off by 3 n U; the result is rounded once.
"""

import numpy as np
import pytest
import torch

from layer_tolerance import U, assert_within, f64, half, smallest
from oops_amd import OOpsUnsupportedError, cache_attention, cache_read, cache_write, quantized_cache
from oracle import decoder

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def _rows(cache, slots):
    """Codes (T, G, 2, D) and exponents (T, G, 2, D / 32) at slots, as numpy."""

    codes, scales = (t.cpu().numpy() for t in cache)
    page = codes.shape[3]
    c, s = codes[slots // page, :, :, slots % page], scales[slots // page, :, :, slots % page]
    return np.stack((c & 15, c >> 4), -1).reshape(*c.shape[:-1], 2 * c.shape[-1]), s


def _check_rows(cache, slots, key, value):
    """The cache at slots holds key and value (G, T, D) exactly as the definition has them."""

    code, e = _rows(cache, slots)
    for i, t in enumerate((key, value)):
        want_code, want_e = decoder.quantize(f64(t).transpose(1, 0, 2))
        np.testing.assert_array_equal(e[:, :, i], want_e)
        # (a rounded zero keeps its sign, as a number does)
        np.testing.assert_array_equal(code[:, :, i], want_code)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,page,heads", [(128, 64, 8), (64, 16, 3), (32, 16, 1), (96, 48, 2)])
def test_write_and_read(dtype, d, page, heads):
    g = torch.Generator().manual_seed(d)
    cache = quantized_cache(9, heads, d, page_size=page, device=DEV)
    n = 4 * page + 5
    key, value = (_randn(g, n, heads, d, dtype=dtype).transpose(0, 1) for _ in range(2))
    slots = torch.randperm(9 * page, generator=g)[:n]
    before = [t.clone() for t in cache]
    cache_write(*cache, key, value, slots.to(DEV))
    _check_rows(cache, slots.numpy(), key, value)
    # nothing else was touched
    other = torch.tensor(sorted(set(range(9 * page)) - set(slots.tolist())))
    for a, b in zip(cache, before):
        assert torch.equal(a.cpu()[other // page, :, :, other % page], b.cpu()[other // page, :, :, other % page])
    for out_type in DTYPES:
        k, v = cache_read(*cache, slots.to(DEV), dtype=out_type)
        assert k.shape == key.shape and k.dtype == out_type
        for got, t in ((k, key), (v, value)):
            want = decoder.values(*decoder.quantize(f64(t)))
            np.testing.assert_array_equal(f64(got), want)  # (codes of unit normals are exact in every type)


@pytest.mark.parametrize("dtype", DTYPES)
def test_values_at_borders(dtype):
    """Ties between codes, the border between two exponents, zeros, the smallest and the largest numbers."""

    info = torch.finfo(dtype)
    rows = []
    base = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 4, dtype=torch.float64)
    for e in (0, -3, 5):
        rows += [base * 2.0**e, -base * 2.0**e]
    up = base.clone()
    up[7] = 6 * (1 + info.eps)  # above the border: the next exponent
    down = base.clone()
    down[[7, 15, 23, 31]] = 6 * (1 - info.eps)
    near = base * (1 + info.eps)
    rows += [up, down, near, base * (1 - info.eps), torch.zeros(32, dtype=torch.float64), -torch.zeros(32, dtype=torch.float64)]
    rows += [torch.full((32,), info.smallest_normal, dtype=torch.float64), torch.full((32,), info.smallest_normal * info.eps, dtype=torch.float64)]
    rows += [torch.full((32,), info.max, dtype=torch.float64), torch.linspace(-info.max, info.max, 32, dtype=torch.float64)]
    if dtype != torch.float16:  # subnormal numbers at the smallest scale, 2^-126
        rows += [base * 2.0**-126, base * 2.0**-128, near * 2.0**-126]
    x = torch.stack(rows).to(dtype).to(DEV)[None]  # (1, T, 32)
    cache = quantized_cache(4, 1, 32, page_size=16, device=DEV)
    slots = torch.arange(x.shape[1], device=DEV)
    cache_write(*cache, x, -x, slots)
    _check_rows(cache, slots.cpu().numpy(), x, -x)
    k, v = cache_read(*cache, slots, dtype=torch.float32)
    assert torch.isfinite(k).all() and torch.equal(k, -v)


@pytest.mark.parametrize("dtype", DTYPES)
def test_blocks_that_are_not_finite(dtype):
    g = torch.Generator().manual_seed(1)
    key, value = (_randn(g, 2, 6, 128, dtype=dtype) for _ in range(2))
    key[0, 1, 40], key[1, 2, 0], value[0, 3, 127] = float("nan"), float("inf"), -float("inf")
    cache = quantized_cache(1, 2, 128, page_size=16, device=DEV)
    slots = torch.arange(6, device=DEV)
    cache_write(*cache, key, value, slots)
    _check_rows(cache, slots.cpu().numpy(), key, value)
    for got, t in zip(cache_read(*cache, slots, dtype=dtype), (key, value)):
        fine = torch.isfinite(t).unflatten(-1, (4, 32)).all(-1, keepdim=True).expand(-1, -1, -1, 32).flatten(-2)
        assert torch.equal(torch.isnan(got), ~fine)


@pytest.mark.parametrize("n", [3, 64, 1000, 1025, 5000])
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_slots(n, kind):
    """Slots that are not there, and the same slot twice: the last of its tokens is kept, whatever the call's size."""

    g = torch.Generator().manual_seed(n)
    cache = quantized_cache(5, 2, 64, page_size=32, device=DEV)
    key, value = (_randn(g, n, 2, 64, dtype=torch.bfloat16).transpose(0, 1) for _ in range(2))
    slots = torch.randint(-40, 200, (n,), generator=g)  # 160 places
    cache_write(*cache, key, value, slots.to(kind).to(DEV))
    last = {int(s): i for i, s in enumerate(slots) if 0 <= s < 160}
    at = np.array(sorted(last))
    if len(at):
        _check_rows(cache, at, key[:, [last[s] for s in at]], value[:, [last[s] for s in at]])
    rest = np.array(sorted(set(range(160)) - set(last)), dtype=int)
    codes, e = _rows(cache, rest)
    assert not codes.any() and not e.any()
    k, v = cache_read(*cache, slots.to(kind).to(DEV))
    gone = torch.tensor([not 0 <= s < 160 for s in slots])
    assert not k[:, gone].any() and not v[:, gone].any()


def test_write_layouts():
    g = torch.Generator().manual_seed(2)
    key, value = (_randn(g, 2, 3, 40, 64, dtype=torch.float16) for _ in range(2))
    slots = torch.randperm(160, generator=g)[:80].view(2, 40).to(DEV)

    def write(k, v, s=slots):
        cache = quantized_cache(10, 3, 64, page_size=16, device=DEV)
        cache_write(*cache, k, v, s)
        return cache

    want = write(key, value)
    token = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    odd = lambda t: torch.nn.functional.pad(t, (1, 1))[..., 1:-1]  # noqa: E731
    inner = lambda t: t.transpose(2, 3).contiguous().transpose(2, 3)  # noqa: E731
    for f in (token, odd, inner):
        assert all(torch.equal(a, b) for a, b in zip(write(f(key), f(value)), want))
    # one token of each sequence
    cache = quantized_cache(10, 3, 64, page_size=16, device=DEV)
    for t in range(40):
        cache_write(*cache, key[:, :, t : t + 1], value[:, :, t : t + 1], slots[:, t : t + 1])
    assert all(torch.equal(a, b) for a, b in zip(cache, want))
    k, v = cache_read(*want, slots, dtype=torch.float16)
    assert k.shape == key.shape
    flat = cache_read(*want, slots.flatten(), dtype=torch.float16)
    assert torch.equal(flat[0].view(3, 2, 40, 64).transpose(0, 1), k)


# ----------------------------------------------------------------- attention


def _attend(seed, lengths, h, kv, d, page, dtype, extra=1, scale=None, kind=torch.int32, width=None):
    g = torch.Generator().manual_seed(seed)
    b = len(lengths)
    width = width or max(1, max(-(-n // page) for n in lengths))
    pages = b * width + extra
    cache = quantized_cache(pages, kv, d, page_size=page, device=DEV)
    key, value = (_randn(g, pages * page, kv, d, dtype=torch.float32).transpose(0, 1) for _ in range(2))
    cache_write(*cache, key, value, torch.arange(pages * page, device=DEV))
    table = torch.randperm(pages, generator=g)[: b * width].view(b, width).int()
    q = _randn(g, b, h, d, dtype=dtype)
    n = torch.tensor(lengths, dtype=kind, device=DEV)
    out = cache_attention(q, *cache, table.to(DEV), n, scale=scale)
    assert out.shape == q.shape and out.dtype == dtype
    _check_attention(out, q, cache, table.numpy(), lengths, scale)
    return q, cache, table.to(DEV), n, out


def _check_attention(out, q, cache, table, lengths, scale=None):
    dtype, d = q.dtype, q.shape[-1]
    scale = d**-0.5 if scale is None else scale
    kv = decoder.cache_values(*(t.cpu().numpy() for t in cache))
    page = kv.shape[3]
    lengths = [min(max(n, 0), table.shape[1] * page) for n in lengths]
    want = decoder.cache_attention(f64(q), kv, table, lengths, scale)
    n = max([1, *lengths])
    # |p| |v| and the scores' magnitudes
    size = decoder.cache_attention(f64(q), np.stack((kv[:, :, 0], np.abs(kv[:, :, 1])), 2), table, lengths, scale)
    score = abs(scale) * np.abs(f64(q)).sum(-1, keepdims=True) * np.abs(kv[:, :, 0]).max()
    rounded = {torch.bfloat16: half(dtype), torch.float16: 2.0**-16, torch.float32: 2.0**-24}[dtype]
    rel = np.expm1(2 * (3 * d + 8) * U * score + (n + 16) * U) + rounded + 3 * n * U
    assert_within(out, want, rel * size + half(dtype) * np.abs(want) + smallest(dtype), "out")
    if dtype == torch.bfloat16 and np.linalg.norm(want) > 0:
        off = np.linalg.norm(f64(out) - want) / np.linalg.norm(want)
        assert off <= 2 * half(dtype), off


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,page,h,kv", [(128, 64, 8, 2), (128, 16, 32, 2), (64, 16, 6, 3), (96, 48, 9, 3), (32, 32, 5, 1), (128, 128, 4, 4),
                                         (64, 64, 40, 2)])  # fmt: skip
def test_attention(dtype, d, page, h, kv):
    _attend(d + h, [1, 0, 2, 15, 16, 17, 31, 32, 33, 100, 127, 128, 129, 260], h, kv, d, page, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths", [[3000], [1], [0], [2049, 5], [700, 0, 1, 1500]])
def test_few_sequences(dtype, lengths):
    """Split over the length: parts without tokens among them."""

    _attend(len(lengths), lengths, 8, 2, 128, 64, dtype, kind=torch.int64)
    _attend(len(lengths), lengths, 3, 1, 64, 16, dtype, scale=-0.3)


def test_a_long_sequence_against_float32():
    """70000 tokens: bfloat16 against float32 of the same cache and query."""

    g = torch.Generator().manual_seed(3)
    n = 70000
    cache = quantized_cache(n // 64 + 1, 2, 128, device=DEV)
    key, value = (_randn(g, n, 2, 128, dtype=torch.bfloat16).transpose(0, 1) for _ in range(2))
    cache_write(*cache, key, value, torch.arange(n, device=DEV))
    table = torch.arange(n // 64 + 1, device=DEV, dtype=torch.int32)[None]
    q = _randn(g, 1, 8, 128, dtype=torch.bfloat16)
    lengths = torch.tensor([n], device=DEV)
    a, b = (cache_attention(t, *cache, table, lengths) for t in (q, q.float()))
    # weights rounded to half a step each, and the result
    assert ((a.double() - b.double()).norm() / b.double().norm()).item() <= 2 * half(torch.bfloat16)
    k, v = cache_read(*cache, torch.arange(n, device=DEV), dtype=torch.float32)
    p = torch.softmax(q.double().view(2, 4, 128) @ k.double().transpose(1, 2) * 128**-0.5, -1)
    want = (p @ v.double()).view(1, 8, 128)
    assert ((b.double() - want).norm() / want.norm()).item() <= 64 * U


@pytest.mark.parametrize("dtype", DTYPES)
def test_pages_that_are_not_there(dtype):
    """Bad page numbers: their tokens are left out; behind the length they are not looked at."""

    q, cache, table, n, out = _attend(4, [100, 100, 64, 10], 4, 2, 64, 16, dtype)
    pages = cache[0].shape[0]
    bad = table.clone()
    bad[0, 1], bad[0, 4], bad[1, 6] = -1, pages, 2**31 - 1
    bad[2, :], bad[3, 1:] = -(2**31), 12345
    got = cache_attention(q, *cache, bad, n)
    _check_attention(got, q, cache, bad.cpu().numpy(), n.tolist())
    assert not got[2].any() and torch.equal(got[3], out[3])


@pytest.mark.parametrize("dtype", DTYPES)
def test_what_lies_behind_the_length(dtype):
    """NaN in places behind the last token, in the same page and tile, does not take part; lengths out of range."""

    lengths = [5, 17, 40, 0]
    q, cache, table, n, out = _attend(5, lengths, 4, 2, 64, 16, dtype, width=4)
    for b, count in enumerate(lengths):
        for t in range(count, 64):
            page = int(table[b, t // 16])
            cache[0][page, :, :, t % 16] = 255
            cache[1][page, :, :, t % 16] = 255
    assert torch.equal(cache_attention(q, *cache, table, n), out)
    q, cache, table, n, _ = _attend(6, [64, 64], 4, 2, 64, 16, dtype)
    full = cache_attention(q, *cache, table, n)
    assert torch.equal(cache_attention(q, *cache, table, torch.tensor([1 << 40, 65], device=DEV)), full)
    assert not cache_attention(q, *cache, table, torch.tensor([-1, -(1 << 40)], device=DEV)).any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_non_finite_blocks_and_queries(dtype):
    """A key's lost block makes its head group's rows NaN, a value's its own 32 channels, a query's NaN its own row."""

    q, cache, table, n, out = _attend(7, [50, 50], 4, 2, 64, 16, dtype)
    page, place = int(table[0, 2]), 3
    broken = [t.clone() for t in cache]
    broken[1][page, 1, 0, place, 0] = 255
    got = cache_attention(q, *broken, table, n)
    assert torch.isnan(got[0, 2:]).all() and torch.equal(got[0, :2], out[0, :2]) and torch.equal(got[1], out[1])
    broken = [t.clone() for t in cache]
    broken[1][page, 0, 1, place, 1] = 255
    got = cache_attention(q, *broken, table, n)
    assert torch.isnan(got[0, :2, 32:]).all() and torch.equal(got[0, :2, :32], out[0, :2, :32])
    assert torch.equal(got[0, 2:], out[0, 2:]) and torch.equal(got[1], out[1])
    q[1, 3, 7] = float("nan")
    got = cache_attention(q, *cache, table, n)
    assert torch.isnan(got[1, 3]).all() and torch.equal(got[1, :3], out[1, :3]) and torch.equal(got[0], out[0])


def test_large_scores_and_scales():
    for dtype in DTYPES:
        q, cache, table, n, _ = _attend(8, [300, 70], 4, 1, 128, 16, dtype, scale=4.0)
        zero = cache_attention(q, *cache, table, n, scale=0.0)
        kv = decoder.cache_values(*(t.cpu().numpy() for t in cache))[:, 0, 1]
        for b, count in enumerate((300, 70)):
            t = np.arange(count)
            want = np.broadcast_to(kv[table[b].cpu().numpy()[t // 16], t % 16].mean(0), (4, 128))
            assert_within(zero[b], want, (half(dtype) + 400 * U) * np.abs(want) + half(dtype) * 1.0, "mean")


def test_attention_layouts():
    q, cache, table, n, out = _attend(9, [70, 33, 5, 90], 4, 2, 64, 16, torch.bfloat16)
    wide = torch.nn.functional.pad(q, (3, 2))[..., 3:-2]
    across = q.transpose(0, 1).contiguous().transpose(0, 1)
    for t in (wide, across):
        assert torch.equal(cache_attention(t, *cache, table, n), out)
    two = cache_attention(q.unflatten(0, (2, 2)), *cache, table.unflatten(0, (2, 2)), n.unflatten(0, (2, 2)))
    assert torch.equal(two.flatten(0, 1), out)
    one = cache_attention(q[3], *cache, table[3], n[3])
    assert one.shape == (4, 64)
    torch.testing.assert_close(one, out[3], rtol=4 * half(torch.bfloat16), atol=2.0**-12)  # (other parts of the length)
    assert torch.equal(cache_attention(q, *cache, table.repeat_interleave(2, 1)[:, ::2], n), out)
    none = cache_attention(q[:0], *cache, table[:0], n[:0])
    assert none.shape == (0, 4, 64)
    assert not cache_attention(q, *cache, table[:, :0], n).any()
    empty = quantized_cache(0, 2, 64, device=DEV)
    assert not cache_attention(q, *empty, table, n).any()


def test_cache_past_32_bits():
    """A cache of more than 2^32 bytes: its last pages."""

    cache = quantized_cache(2**25 // 64 * 2 + 3, 1, 128, device=DEV)
    pages = cache[0].shape[0]
    assert cache[0].numel() > 2**32
    g = torch.Generator().manual_seed(10)
    key, value = (_randn(g, 1, 200, 128, dtype=torch.bfloat16) for _ in range(2))
    slots = (pages - 4) * 64 + torch.arange(200, device=DEV)
    cache_write(*cache, key, value, slots)
    small = quantized_cache(4, 1, 128, device=DEV)
    cache_write(*small, key, value, torch.arange(200, device=DEV))
    for a, b in zip(cache_read(*cache, slots), cache_read(*small, torch.arange(200, device=DEV))):
        assert torch.equal(a, b)
    q = _randn(g, 1, 4, 128, dtype=torch.bfloat16)
    table = torch.arange(4, device=DEV, dtype=torch.int32)[None]
    n = torch.tensor([200], device=DEV)
    assert torch.equal(cache_attention(q, *cache, table + pages - 4, n), cache_attention(q, *small, table, n))


def test_refusals():
    q, cache, table, n, _ = _attend(11, [20], 4, 2, 64, 16, torch.bfloat16)
    codes, scales = cache
    key = torch.zeros(2, 5, 64, dtype=torch.bfloat16, device=DEV)
    slots = torch.arange(5, device=DEV)
    for call in (lambda: cache_write(codes, scales, key.double(), key.double(), slots), lambda: cache_write(codes, scales, key, key.float(), slots),
                 lambda: cache_write(codes, scales, key, key, slots.float()), lambda: cache_write(codes, scales, key.requires_grad_(True), key, slots),
                 lambda: cache_write(codes[::2], scales[::2], key.detach(), key.detach(), slots), lambda: quantized_cache(3, 2, 48, device=DEV),
                 lambda: quantized_cache(3, 2, 64, page_size=24, device=DEV), lambda: cache_read(codes, scales, slots, dtype=torch.float64),
                 lambda: cache_attention(q.requires_grad_(True), *cache, table, n), lambda: cache_attention(q.detach(), *cache, table.long(), n),
                 lambda: cache_attention(q.detach(), codes.int(), scales, table, n)):  # fmt: skip
        with pytest.raises(OOpsUnsupportedError):
            call()
    key, q = key.detach(), q.detach()
    for call in (lambda: cache_write(codes, scales, key[:1], key[:1], slots), lambda: cache_write(codes, scales, key, key[:, :4], slots),
                 lambda: cache_write(codes, scales, key, key, slots[:4]), lambda: cache_write(codes, scales[..., :1], key, key, slots),
                 lambda: cache_attention(q[:, :3], *cache, table, n), lambda: cache_attention(q[..., :32], *cache, table, n),
                 lambda: cache_attention(q, *cache, table[0], n), lambda: cache_attention(q, *cache, table, n[0]),
                 lambda: quantized_cache(-1, 2, 64, device=DEV), lambda: cache_attention(q, *cache, table.cpu(), n)):  # fmt: skip
        with pytest.raises(ValueError):
            call()


def test_write_counts_as_a_change_of_the_cache():
    cache = quantized_cache(2, 1, 32, page_size=16, device=DEV)
    version = [t._version for t in cache]
    cache_write(*cache, torch.ones(1, 3, 32, device=DEV), torch.ones(1, 3, 32, device=DEV), torch.arange(3, device=DEV))
    assert all(t._version > v for t, v in zip(cache, version))


def test_compile_with_sizes_that_change():
    def f(codes, scales, key, value, slots, q, table, n):
        cache_write(codes, scales, key * 1.0, value, slots)
        return cache_attention(q, codes, scales, table, n), *cache_read(codes, scales, slots)

    g = torch.compile(f, dynamic=True, fullgraph=True)
    for n in (20, 33, 47):
        rng = torch.Generator().manual_seed(n)
        key, value = (_randn(rng, 2, n, 64, dtype=torch.bfloat16) for _ in range(2))
        args = (key, value, torch.arange(n, device=DEV), _randn(rng, 1, 4, 64, dtype=torch.bfloat16),
                torch.tensor([[0, 1, 2]], dtype=torch.int32, device=DEV), torch.tensor([n], device=DEV))  # fmt: skip
        results = []
        for fn in (f, g):
            cache = quantized_cache(3, 2, 64, page_size=16, device=DEV)
            results.append((*fn(*cache, *args), *cache))
        assert all(torch.equal(a, b) for a, b in zip(*results))


def test_graph_replays_and_streams():
    """A decoding step captured (write, then attend, split over the length), replayed as the sequences grow; two graphs."""

    g = torch.Generator().manual_seed(12)
    d, kv, page = 128, 2, 16
    table = torch.randperm(40, generator=g).view(2, 20).int().to(DEV)
    cache = quantized_cache(40, kv, d, page_size=page, device=DEV)
    eager = [t.clone() for t in cache]
    q, key, value = _randn(g, 2, 8, d), _randn(g, 2, kv, 1, d), _randn(g, 2, kv, 1, d)
    lengths = torch.tensor([0, 250], device=DEV)

    def step(c):
        slots = table.long().gather(1, (lengths[:, None]) // page) * page + lengths[:, None] % page
        cache_write(*c, key, value, slots)
        return cache_attention(q, *c, table, lengths + 1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step([t.clone() for t in cache])
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(cache))
    for i in range(40):
        q.copy_(_randn(g, 2, 8, d))
        key.copy_(_randn(g, 2, kv, 1, d))
        value.copy_(_randn(g, 2, kv, 1, d))
        graphs[i % 2].replay()
        want = step(eager)
        torch.cuda.synchronize()
        assert torch.equal(outs[i % 2], want), i
        assert all(torch.equal(a, b) for a, b in zip(cache, eager))
        lengths += 1
