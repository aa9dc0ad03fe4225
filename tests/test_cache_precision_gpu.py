"""cache_attention where its result must have the precision of the query's type (oracle/decoder.py, float64).

h: half a step of the query's type, U of float32.  Weights enter the second product with at least 16 bits (2^-16 of
themselves), their sum and the products' sums of n terms are float32 (n U each).
"""

import numpy as np
import pytest
import torch

from layer_tolerance import U, assert_within, f64, half, smallest
from oops_amd import cache_attention, cache_write, quantized_cache
from oracle import decoder

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _filled(key, value):
    """A cache of pages of 64 with key and value (1, T, D), which the codes hold exactly, and its page table."""

    n, d = key.shape[1:]
    cache = quantized_cache(n // 64, 1, d, device=DEV)
    cache_write(*cache, key, value, torch.arange(n, device=DEV))
    kv = decoder.cache_values(*(t.cpu().numpy() for t in cache))
    assert np.array_equal(kv[:, 0, 0].reshape(n, d), f64(key)[0]) and np.array_equal(kv[:, 0, 1].reshape(n, d), f64(value)[0])
    return cache, torch.arange(n // 64, dtype=torch.int32, device=DEV)[None], kv


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [256, 2048])
def test_a_rounding_that_many_weights_share(dtype, n):
    """Half the tokens have weight 1, the others all the same one, a little above: 1 + a part of a step of 16-bit types."""

    d = 64
    key, value = torch.zeros(1, n, d, device=DEV), torch.zeros(1, n, d, device=DEV)
    key[0, n // 2 :, 0] = 1
    value[0, n // 2 :] = torch.tensor([0.5, 1, 1.5, 2, 3, 4, 6, -6] * (d // 8), device=DEV)
    cache, table, kv = _filled(key, value)
    lengths = torch.tensor([n], device=DEV)
    q = torch.zeros(1, 1, d, dtype=dtype, device=DEV)
    q[..., 0] = 1
    for part in np.linspace(0.05, 0.95, 19):
        scale = float(np.log1p(part * 2.0**-7))
        out = cache_attention(q, *cache, table, lengths, scale=scale)
        want = decoder.cache_attention(f64(q), kv, table.cpu().numpy(), [n], scale)
        bound = half(dtype) * np.abs(want) * (1 + 2.0**-8) + (2.0**-16 if dtype != torch.float32 else 0) * np.abs(want)
        assert_within(out, want, bound + 2 * (n + 16) * U * np.abs(want), f"part {part:.2f}")


def test_queries_above_the_largest_bfloat16():
    """float32 numbers that bfloat16 would round to infinity: scores that float32 holds, and zeros, are what they are."""

    d, n = 32, 64
    key, value = torch.zeros(1, n, d, device=DEV), torch.zeros(1, n, d, device=DEV)
    key[0, :, 0] = torch.tensor([0, 0.5, 1, -1] * (n // 4), device=DEV)
    value[0] = (torch.arange(n, device=DEV) % 4)[:, None].float()
    cache, table, kv = _filled(key, value)
    q = torch.zeros(2, 1, d, device=DEV)
    q[0, 0, 0], q[1, 0, 0] = 3.4e38, -3.3999e38
    out = cache_attention(q, *cache, table.expand(2, 1), torch.tensor([n, n], device=DEV), scale=1e-38)
    want = decoder.cache_attention(f64(q), kv, table.cpu().numpy().repeat(2, 0), [n, n], 1e-38)
    # a score of up to 3.4: 100 U of it as in the other tests; 64 terms
    assert_within(out, want, (np.expm1(2 * 104 * U * 3.4) + 200 * U) * 3 + smallest(torch.float32), "out")
