"""Wrapper tensors (no storage of their own, as quantised and distributed ones) in the place of each operand and
gradient of the layer operators: the bits of the call with what they wrap."""

import pytest
import torch

import oops_amd

pytestmark = pytest.mark.gpu

DEV = "cuda"


class _Wrapped(torch.Tensor):
    @staticmethod
    def __new__(cls, inner):
        out = torch.Tensor._make_wrapper_subclass(cls, inner.shape, strides=inner.stride(), dtype=inner.dtype,
                                                  device=inner.device)  # fmt: skip
        out.inner = inner
        return out

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        unwrap = lambda t: t.inner if isinstance(t, cls) else t  # noqa: E731
        return func(*torch.utils._pytree.tree_map(unwrap, args), **(kwargs or {}))


def _tuple(x):
    return x if isinstance(x, tuple) else (x,)


def _same(got, want):
    for a, b in zip(got, want, strict=True):
        assert torch.equal(a.inner if isinstance(a, _Wrapped) else a, b)


def _norm_operands():
    g = torch.Generator().manual_seed(1)
    return [torch.randn(*shape, generator=g).to(DEV) for shape in ((9, 64), (64,), (9, 64))]


def _linear_operands():
    g = torch.Generator().manual_seed(2)
    q, k, v, s0 = (torch.randn(*shape, generator=g).to(DEV) for shape in ((2, 3, 40, 16), (2, 3, 40, 16), (2, 3, 40, 8), (2, 3, 16, 8)))
    return [q, k, v, torch.tensor([-0.1, -0.5, 0.0], device=DEV), s0, torch.tensor([40, 11], device=DEV)]


def _int8_operands():
    g = torch.Generator().manual_seed(3)
    x, w = (torch.randint(-128, 128, (n, 48), generator=g, dtype=torch.int8).to(DEV) for n in (7, 20))
    return [x, torch.rand(7, device=DEV), w, torch.rand(20, device=DEV), torch.randn(20, device=DEV)]


CALLS = {
    "rms_norm": (lambda x, w, r: oops_amd.rms_norm(x, 64, w, residual=r), _norm_operands),
    "rms_norm_int8": (lambda x, w, r: oops_amd.rms_norm_int8(x, 64, w, residual=r), _norm_operands),
    "quantize_int8": (oops_amd.quantize_int8, lambda: _norm_operands()[:1]),
    "int8_linear": (oops_amd.int8_linear, _int8_operands),
    "linear_attention": (lambda *t: oops_amd.linear_attention(*t, return_state=True), _linear_operands),
}


@pytest.mark.parametrize("name", CALLS)
def test_operands(name):
    call, make = CALLS[name]
    operands = make()
    with torch.no_grad():
        want = _tuple(call(*operands))
        for i in range(len(operands)):
            _same(_tuple(call(*[_Wrapped(t) if i == j else t for j, t in enumerate(operands)])), want)


def test_step():
    q, k, v, ld, s0, _ = _linear_operands()
    operands = [q[:, :, 0], k[:, :, 0], v[:, :, 0], ld]
    state = s0.clone()
    want = oops_amd.linear_attention_step(*operands, state)
    for i in range(5):
        again = s0.clone()
        args = [_Wrapped(t) if i == j else t for j, t in enumerate((*operands, again))]
        _same([oops_amd.linear_attention_step(*args), again], [want, state])


@pytest.mark.parametrize("which", [0, 1])
def test_gradients(which):
    x, w, r = (t.requires_grad_(True) for t in _norm_operands())
    q, k, v, ld, s0, n = _linear_operands()
    leaves = [t.requires_grad_(True) for t in (q, k, v, s0)]
    for outs, inputs in ((oops_amd.rms_norm(x, 64, w, residual=r), [x, w, r]),
                         (oops_amd.linear_attention(q, k, v, ld, s0, n, return_state=True), leaves)):  # fmt: skip
        grads = [torch.randn_like(t) for t in outs]
        want = torch.autograd.grad(outs, inputs, grads, retain_graph=True)
        _same(torch.autograd.grad(outs, inputs, [_Wrapped(g) if i == which else g for i, g in enumerate(grads)]), want)
