"""The layer operators' front-ends on the host: what they hand to the kernels.  No kernel is launched."""

import importlib

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.symbolic_shapes import DimDynamic, ShapeEnv, StatelessSymbolicContext

import oops_amd
from layer_tolerance import U, assert_within, f64, half
from oops_amd import RMSNorm
from oops_amd.attention import linear
from oops_amd.linear import int8
from oops_amd.normalization import modules
from oracle import layers

rms_norm = importlib.import_module("oops_amd.normalization.rms_norm")  # (the package's name is the function)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scale", [1e-4, 1e-3, 0.02, 1.0])
def test_default_eps_of_the_module_is_pytorchs(dtype, scale, monkeypatch):
    """Rows small enough that the eps decides the result: the definition with the eps that the module passes, against
    torch.nn.RMSNorm (one rounding to the type, and float32 arithmetic: 64 terms a row, 64 U)."""

    passed = []
    monkeypatch.setattr(modules, "rms_norm", lambda x, shape, weight, eps, residual: passed.append(eps))
    x = (torch.randn(5, 64, generator=torch.Generator().manual_seed(1)) * scale).to(dtype)
    RMSNorm(64, dtype=dtype)(x)
    want = layers.rms_norm_forward(f64(x), None, passed[0])
    assert_within(torch.nn.RMSNorm(64, dtype=dtype)(x), want, (half(dtype) + 64 * U) * abs(want), "y")
    RMSNorm(64, eps=1e-3, dtype=dtype)(x)
    assert passed[1] == 1e-3


def _symbolic_mode():
    """A fake-tensor mode and two sizes that are symbols, as torch.compile traces sizes that change."""

    mode = FakeTensorMode(shape_env=ShapeEnv())
    context = StatelessSymbolicContext([DimDynamic.DYNAMIC] * 2)
    return mode, mode.from_tensor(torch.empty(3, 70), symbolic_context=context).shape


def test_symbolic_sizes():
    """Every layer operator traces with symbolic batch and length; shapes and dimension orders are the eager ones."""

    mode, (b, n) = _symbolic_mode()
    with mode, torch.no_grad():
        new = lambda *shape, dtype=torch.bfloat16: torch.empty(*shape, dtype=dtype, device="cuda")  # noqa: E731
        x, w = new(b, n, 64), new(64, dtype=torch.float32)
        y, summed = oops_amd.rms_norm(x, 64, w, residual=x)
        assert y.shape == summed.shape == (b, n, 64)
        for values, scales in (oops_amd.rms_norm_int8(x, 64, w), oops_amd.quantize_int8(x)):
            assert values.shape == (b, n, 64) and scales.shape == (b, n)
        wq, ws = new(96, 64, dtype=torch.int8), new(96, dtype=torch.float32)
        assert oops_amd.int8_linear(values, scales, wq, ws).shape == (b, n, 96)
        q, v, ld = new(b, n, 4, 32).transpose(1, 2), new(b, n, 4, 16).transpose(1, 2), new(4, dtype=torch.float32)
        s0, lengths = new(b, 4, 32, 16, dtype=torch.float32), new(b, dtype=torch.int32)
        out, state = oops_amd.linear_attention(q, q, v, ld, s0, lengths, return_state=True)
        assert out.shape == (b, 4, n, 16) and out.transpose(1, 2).is_contiguous() and state.shape == (b, 4, 32, 16)
        grads = linear.linear_attention_backward(out, state, q, q, v, ld, lengths, s0, 1.0, [True] * 4)
        assert [g.shape for g in grads] == [q.shape, q.shape, v.shape, s0.shape]
        assert all(g.transpose(1, 2).is_contiguous() for g in grads[:3])
        assert oops_amd.linear_attention_step(q[:, :, 0], q[:, :, 0], v[:, :, 0], ld, s0).shape == (b, 4, 16)


class _Dispatched(Exception):
    pass


class _Wrapped(torch.Tensor):
    """A wrapper without storage of its own, as quantised and distributed tensors are; an operator of the framework
    that it is given to is reported."""

    @staticmethod
    def __new__(cls, inner):
        out = torch.Tensor._make_wrapper_subclass(cls, inner.shape, strides=inner.stride(), dtype=inner.dtype,
                                                  device=inner.device)  # fmt: skip
        out.inner = inner
        return out

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        if func.namespace == "oops_amd":
            raise _Dispatched(func._schema.name)
        if func in (torch.ops.aten.view.default, torch.ops.aten.detach.default):
            return cls(func(args[0].inner, *args[1:]))
        unwrap = lambda t: t.inner if isinstance(t, cls) else t  # noqa: E731
        return func(*torch.utils._pytree.tree_map(unwrap, args), **(kwargs or {}))


@pytest.fixture
def no_launches(monkeypatch):
    """Checks see device tensors; a launch is an error."""

    def launched(*args):
        raise AssertionError("a launch with a wrapper's address")

    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))
    for module, names in ((rms_norm, ("_forward_impl", "_int8_impl", "_quantize_impl", "_backward_impl")),
                          (int8, ("_forward_impl",)),
                          (linear, ("_forward_impl", "_forward_with_workspace", "_backward_impl", "_step_impl"))):  # fmt: skip
        for name in names:
            monkeypatch.setattr(module, name, launched)
    return launched


def _each_wrapped(call, operands):
    """``call`` with each operand in turn as a wrapper has to reach the dispatcher."""

    for i in range(len(operands)):
        wrapped = [_Wrapped(t) if i == j else t for j, t in enumerate(operands)]
        with torch.no_grad(), pytest.raises(_Dispatched):
            call(*wrapped)


def test_wrappers_in_the_place_of_any_operand_are_dispatched(no_launches):
    x, r, w = torch.randn(3, 8), torch.randn(3, 8), torch.randn(8)
    for norm in (oops_amd.rms_norm, oops_amd.rms_norm_int8):
        _each_wrapped(lambda x, w, r, norm=norm: norm(x, 8, w, residual=r), [x, w, r])
    _each_wrapped(oops_amd.quantize_int8, [x])
    i8, w8 = torch.zeros(3, 8, dtype=torch.int8), torch.zeros(5, 8, dtype=torch.int8)
    _each_wrapped(oops_amd.int8_linear, [i8, torch.ones(3), w8, torch.ones(5), torch.ones(5)])
    q, v, ld, s0 = torch.randn(2, 3, 7, 8), torch.randn(2, 3, 7, 4), torch.zeros(3), torch.zeros(2, 3, 8, 4)
    lengths = torch.tensor([7, 5], dtype=torch.int32)
    _each_wrapped(oops_amd.linear_attention, [q, q.clone(), v, ld, s0, lengths])
    _each_wrapped(oops_amd.linear_attention_step, [q[:, :, 0], q[:, :, 1], v[:, :, 0], ld, s0])
    with pytest.raises(AssertionError, match="launch"):  # (a parameter is no wrapper)
        oops_amd.rms_norm(x, 8, torch.nn.Parameter(w), residual=r)


def test_lazily_negated_operands_are_resolved(no_launches, monkeypatch):
    """Addresses cannot carry a lazy negation: the launch of each operator gets the negated values."""

    def launched(*args):
        raise _Dispatched(*args)

    for module, name in ((rms_norm, "_int8_impl"), (int8, "_forward_impl"), (linear, "_forward_impl"), (linear, "_step_impl")):
        monkeypatch.setattr(module, name, launched)
    i8, w8 = torch.arange(24, dtype=torch.int8).view(3, 8), torch.arange(40, dtype=torch.int8).view(5, 8)
    x, q, v, ld, s0 = torch.randn(3, 8), torch.randn(2, 3, 7, 8), torch.randn(2, 3, 7, 4), torch.rand(3), torch.randn(2, 3, 8, 4)
    calls = [(lambda x, w, r: oops_amd.rms_norm_int8(x, 8, w, residual=r), [x, torch.randn(8), torch.randn(3, 8)]),
             (oops_amd.int8_linear, [i8, torch.rand(3), w8, torch.rand(5), torch.rand(5)]),
             (oops_amd.linear_attention, [q, q + 1, v, ld, s0, torch.tensor([-7, -5])]),
             (lambda *t: oops_amd.linear_attention_step(*t, s0), [q[:, :, 0], q[:, :, 1], v[:, :, 0], ld])]  # fmt: skip
    for call, operands in calls:
        for i, negated in enumerate(operands):
            with pytest.raises(_Dispatched) as launch:
                call(*[torch._neg_view(t) if i == j else t for j, t in enumerate(operands)])
            passed = [t for t in launch.value.args if isinstance(t, torch.Tensor)]
            assert not any(t.is_neg() for t in passed)
            assert any(t.shape == negated.shape and torch.equal(t, -negated) for t in passed)


@pytest.mark.parametrize("which", [0, 1])
def test_wrapped_gradients_are_dispatched(no_launches, monkeypatch, which):
    monkeypatch.setattr(rms_norm, "_forward_impl", lambda x, w, r, eps, save: (x + 0, x + r, torch.ones(3)))
    monkeypatch.setattr(linear, "_forward_with_workspace", lambda q, k, v, ld, n, s0, scale, state: (
        q + 0, torch.zeros(2, 3, 8, 8), torch.zeros(4)))  # fmt: skip
    x, w, q = (torch.randn(*shape, requires_grad=True) for shape in ((3, 8), (8,), (2, 3, 7, 8)))
    for leaf, outs in ((x, oops_amd.rms_norm(x, 8, w, residual=x.detach())),
                       (q, oops_amd.linear_attention(q, q, q, torch.zeros(3), return_state=True))):  # fmt: skip
        grads = [_Wrapped(torch.randn(t.shape)) if i == which else torch.randn(t.shape) for i, t in enumerate(outs)]
        with pytest.raises(_Dispatched):
            torch.autograd.grad(outs, leaf, grads)
