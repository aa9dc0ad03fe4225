"""What the decoder's operators announce to traced code: the strides that the real calls allocate (meta tensors, no GPU)."""

import pytest
import torch

from oops_amd.attention import causal

# (B, H, L, D), its memory's order of dimensions, the type
LAYOUTS = [
    ((2, 4, 5, 64), (0, 2, 1, 3), torch.bfloat16),
    ((2, 4, 5, 64), (0, 1, 2, 3), torch.float32),
    ((64, 1024, 3, 128), (2, 0, 1, 3), torch.bfloat16),  # tokens outermost, 2^24 bytes apart
    ((64, 1023, 3, 128), (2, 0, 1, 3), torch.bfloat16),  # a little less
    ((64, 1024, 1, 128), (2, 0, 1, 3), torch.bfloat16),  # one token
    ((64, 512, 3, 128), (2, 1, 0, 3), torch.float32),
]


def _meta(shape, order, dtype):
    t = torch.empty([shape[i] for i in order], dtype=dtype, device="meta")
    return t.permute([order.index(i) for i in range(4)])


@pytest.mark.parametrize("shape,order,dtype", LAYOUTS)
def test_causal_attention_strides(shape, order, dtype):
    q, k, v = (_meta(shape, order, dtype) for _ in range(3))
    out, low, lse = torch.ops.oops_amd.causal_attention_forward(q, k, v, None, 1.0, True)
    real = causal._result_like(q, v.shape[-1])
    assert out.shape == real.shape and out.stride() == real.stride()
    if dtype != torch.float32:
        assert low.stride() == torch.empty_like(real).stride()
    grads = torch.ops.oops_amd.causal_attention_backward(out, q, k, v, None, out, low, lse, 1.0, [True] * 3)
    for g, t in zip(grads, (q, k, v)):
        real = causal._result_like(t, t.shape[-1])
        assert g.shape == real.shape and g.stride() == real.stride()
