"""Wrapper tensors (no storage of their own, as quantised and distributed ones) and lazily negated views in the place of each
operand and gradient of the decoder's operators: the bits of the call with what they stand for."""

import pytest
import torch

import oops_amd
from test_layer_wrappers_gpu import _same, _tuple, _Wrapped

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _randn(seed, *shapes):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(*shape, generator=g).to(DEV) for shape in shapes]


def _causal():
    return [*_randn(1, (1, 4, 40, 16), (1, 2, 40, 16), (1, 2, 40, 8)), torch.tensor([0, 30, 40], device=DEV)]


def _rotary():
    q, k, wq, wk = _randn(2, (2, 4, 9, 32), (2, 1, 9, 32), (32,), (32,))
    return [q, k, oops_amd.rotary_table(20, 32, device=DEV), torch.arange(9, device=DEV) + 3, wq, wk]


def _cache():
    cache = oops_amd.quantized_cache(4, 2, 32, page_size=16, device=DEV)
    slots = torch.arange(64, device=DEV)
    key, value = _randn(3, (2, 64, 32), (2, 64, 32))
    oops_amd.cache_write(*cache, key, value, slots)
    return cache, key, value, slots


def _read():
    cache, _, _, slots = _cache()
    return [*cache, slots]


def _attend():
    cache, _, _, _ = _cache()
    pages = torch.tensor([[1, 3], [0, 2]], device=DEV, dtype=torch.int32)
    return [*_randn(4, (2, 4, 32)), *cache, pages, torch.tensor([30, 9], device=DEV)]


CALLS = {
    "causal_attention": (oops_amd.causal_attention, _causal),
    "rms_norm_rotary": (oops_amd.rms_norm_rotary, _rotary),
    "cache_read": (oops_amd.cache_read, _read),
    "cache_attention": (oops_amd.cache_attention, _attend),
}


def _negated(t):
    return torch._neg_view(-t)


@pytest.mark.parametrize("name", CALLS)
def test_operands(name):
    call, make = CALLS[name]
    operands = make()
    with torch.no_grad():
        want = _tuple(call(*operands))
        for i, t in enumerate(operands):
            for other in (_Wrapped(t), *([_negated(t)] if t.dtype != torch.uint8 else [])):
                _same(_tuple(call(*[other if i == j else u for j, u in enumerate(operands)])), want)


def test_write():
    cache, key, value, slots = _cache()
    slots = slots.flip(0)
    oops_amd.cache_write(*cache, key, value, slots)
    for i in range(5):
        for f in (_Wrapped, _negated):
            again = oops_amd.quantized_cache(4, 2, 32, page_size=16, device=DEV)
            args = [*again, key, value, slots]
            if f is _negated and i < 2:
                continue
            args[i] = f(args[i])
            oops_amd.cache_write(*args)
            _same(again, cache)


@pytest.mark.parametrize("f", [_Wrapped, _negated])
@pytest.mark.parametrize("which", [0, 1])
def test_gradients(which, f):
    q, k, v, offsets = _causal()
    rq, rk, table, positions, wq, wk = _rotary()
    for leaves, call in (([q, k, v], lambda *t: oops_amd.causal_attention(*t, offsets)),
                         ([rq, rk, wq, wk], lambda q, k, wq, wk: oops_amd.rms_norm_rotary(q, k, table, positions, wq, wk))):  # fmt: skip
        leaves = [t.requires_grad_(True) for t in leaves]
        outs = _tuple(call(*leaves))
        if which >= len(outs):
            continue
        grads = [torch.randn_like(t) for t in outs]
        want = torch.autograd.grad(outs, leaves, grads, retain_graph=True)
        _same(torch.autograd.grad(outs, leaves, [f(g) if i == which else g for i, g in enumerate(grads)]), want)


@pytest.mark.parametrize("name", ["causal_attention", "rms_norm_rotary"])
def test_broadcast_operands_and_gradients(name):
    """Operands expanded over batch, heads or tokens (strides of zero) have gradients of their own shape."""

    if name == "causal_attention":
        q, k, v, offsets = _causal()
        base = [q[:, :1].clone(), k[:, :, :1].clone(), v.clone()]
        shapes = [(3, 4, 40, 16), (3, 2, 40, 16), (3, 2, 40, 8)]
        call = lambda q, k, v: oops_amd.causal_attention(q, k, v, offsets)  # noqa: E731
    else:
        q, k, table, positions, wq, wk = _rotary()
        base = [q[:1, :1].clone(), k[:, :, :1].clone(), wq[:1].clone(), wk.clone()]
        shapes = [(2, 4, 9, 32), (2, 1, 9, 32), (32,), (32,)]
        call = lambda q, k, wq, wk: oops_amd.rms_norm_rotary(q, k, table, positions, wq, wk)  # noqa: E731
    leaves = [t.requires_grad_(True) for t in base]
    wide = [t.expand(*s) for t, s in zip(leaves, shapes)]
    full = [t.detach().clone(memory_format=torch.contiguous_format).requires_grad_(True) for t in wide]
    outs, want = _tuple(call(*wide)), _tuple(call(*full))
    _same([t.detach() for t in outs], [t.detach() for t in want])
    got = torch.autograd.grad(outs, leaves, [torch.ones(1, device=DEV).expand_as(t) for t in outs])
    ref = torch.autograd.grad(want, full, [torch.ones_like(t) for t in want])
    for a, b, leaf in zip(got, ref, leaves):
        torch.testing.assert_close(a, b.double().sum_to_size(leaf.shape).float(), rtol=0, atol=b.numel() * 2.0**-24 * float(b.abs().max()))
