"""The layer operators' front-ends on the host: what they hand to the kernels.  No kernel is launched."""

import pytest
import torch

from layer_tolerance import U, assert_within, f64, half
from oops_amd import RMSNorm
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
