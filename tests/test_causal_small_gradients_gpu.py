"""causal_attention in float32 with gradients far below 1: where the lower terms of the operands leave bfloat16's range.

An operand is three bfloat16 terms.  They share float32's exponents, and their smallest number is 2^-133: a number above 2^-110
has them all, of a smaller one 2^-134 may be missing.  The bounds are those for gradients of size 1, scaled with them, and
2^-134 for each element of dO (to dP, dV) and of dS (to dQ, dK).
"""

import numpy as np
import pytest
import torch

from layer_tolerance import U, assert_within, f64
from oops_amd import causal_attention
from oracle import decoder

pytestmark = pytest.mark.gpu

LOST = 2.0**-134


@pytest.mark.parametrize("power", [0, -60, -100, -115])
def test_gradients(power):
    n, d = 150, 64
    g = torch.Generator().manual_seed(9)
    q, k, v, do = (torch.randn(1, 2, n, d, generator=g).cuda() for _ in range(4))
    do = do * 2.0**power
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(causal_attention(*leaves), leaves, do)
    Q, K, V, DO = (f64(t) for t in (q, k, v, do))
    t, a, scale = (lambda m: np.swapaxes(m, -1, -2)), np.abs, d**-0.5
    p = decoder.causal_weights(Q, K, scale)
    want = decoder.causal_backward(Q, K, V, DO, scale)
    lost = LOST if power < -90 else 0.0
    # a probability: its score and its row's sum; products of n, d terms; delta from the float32 output
    score = scale * (d + 8) * U * (a(Q) @ t(a(K)) * decoder.causal_pairs(n))
    rel = np.expm1(score + score.max(-1, keepdims=True) + (n + 16) * U)
    dp, out = DO @ t(V), p @ V
    delta = (a(DO) * a(out)).sum(-1, keepdims=True)
    err_dp = (d + 2) * U * (a(DO) @ t(a(V))) + lost * a(V).sum(-1)[:, :, None, :]
    err_delta = (a(DO) * ((p * (rel + n * U)) @ a(V) + 4 * U * a(out))).sum(-1, keepdims=True) + (d + 4) * U * delta
    size = a(dp - (p * dp).sum(-1, keepdims=True))
    err_ds = p * ((rel + 4 * U) * size + err_dp + err_delta)
    sized = err_ds * (1 + n * U) + n * U * p * size + lost * decoder.causal_pairs(n)
    w = p * (rel + n * U)
    bound = (scale * sized @ a(K), scale * t(sized) @ a(Q), t(w) @ a(DO) + lost * p.sum(-2)[..., None])
    for name, x, y, b in zip(("dq", "dk", "dv"), got, want, bound):
        assert_within(x, y, b + U * a(y) + 2.0**-149, name)
