"""Compiled causal_attention over operands whose results take another order of dimensions than theirs."""

import pytest
import torch

from oops_amd import causal_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dynamic", [False, True])
def test_tokens_far_apart(dynamic):
    """Token-outermost memory, tokens 2^24 bytes apart: eager results, outputs and gradients."""

    def f(q, k, v):
        return causal_attention(q * 1.0, k, v) * 2.0

    compiled = torch.compile(f, dynamic=dynamic, fullgraph=True)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = [torch.randn(3, 64, 1024, 128, generator=g, device="cuda", dtype=torch.bfloat16).permute(1, 2, 0, 3) for _ in range(4)]
    results = []
    for fn in (f, compiled):
        leaves = [t.detach().requires_grad_(True) for t in x[:3]]
        out = fn(*leaves)
        results.append((out, *torch.autograd.grad(out, leaves, x[3])))
    for a, b in zip(*results):
        assert torch.equal(a, b)
