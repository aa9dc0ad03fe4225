"""The layer operators' front-ends on the host: what they hand to the kernels.  No kernel is launched."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.symbolic_shapes import DimDynamic, ShapeEnv, StatelessSymbolicContext

import oops_amd
from layer_tolerance import U, assert_within, f64, half
from oops_amd import RMSNorm
from oops_amd.attention import linear
from oops_amd.normalization import modules
from oracle import layers


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
