"""The layer operators together, as a block of a model uses them: the residual's addition and norm, projections, linear
attention, the gated output stage; trained in bfloat16, and served in 8 bits from a prompt to single tokens.

Training is compared with the same block in float64 PyTorch operations.  Every tensor that the bfloat16 block
writes is rounded once (at most half a step, 2^-8), a path crosses at most twelve of them, and a rounding reaches
the next tensor multiplied by at most the ratio of the sums' magnitudes: errors are compared in the 2-norm, where
roundings of independent terms do not grow, with 12 half steps.
"""

import pytest
import torch

import oops_amd

pytestmark = pytest.mark.gpu

DEV = "cuda"
H, D, C = 4, 32, 128


def _weights(seed):
    g = torch.Generator().manual_seed(seed)
    lin = lambda n, k: (torch.randn(n, k, generator=g) * k**-0.5).bfloat16().to(DEV)  # noqa: E731
    w = {"qkv": lin(3 * H * D, C), "gate": lin(H * D, C), "out": lin(C, H * D)}
    w["norm"] = (1 + 0.1 * torch.randn(C, generator=g)).to(DEV)
    return w


def _heads(t):
    q, k, v = t.unflatten(-1, (3, H, D)).unbind(-3)
    return [x.transpose(1, 2) for x in (q, k, v)]  # token-major views


def _block(x, residual, w, ld, state=None):
    y, stream = oops_amd.rms_norm(x, C, w["norm"], residual=residual)
    q, k, v = _heads(torch.nn.functional.linear(y, w["qkv"]))
    att, last = oops_amd.linear_attention(q, k, v, ld, state, return_state=True)
    return oops_amd.gate_attention_output(att, y, w["gate"], w["out"]), stream, last


def _plain(x, residual, w, ld):
    stream = x + residual
    y = stream * torch.rsqrt(stream.square().mean(-1, keepdim=True) + 1e-6) * w["norm"]
    q, k, v = _heads(y @ w["qkv"].t())
    t = torch.arange(x.shape[1], device=DEV)
    lag = (t[:, None] - t[None]).double()
    decay = torch.where(lag >= 0, torch.exp(ld.double()[:, None, None] * lag.clamp(min=0)), 0.0)
    att = (q @ k.transpose(-1, -2) * decay * D**-0.5) @ v
    gate = torch.sigmoid(y @ w["gate"].t())
    return (gate * att.transpose(1, 2).flatten(2)) @ w["out"].t(), stream


@pytest.mark.parametrize("n", [1, 70, 300])
def test_training(n):
    g = torch.Generator().manual_seed(n)
    x, r, dy, ds = ((torch.randn(2, n, C, generator=g)).bfloat16().to(DEV) for _ in range(4))
    ld = -torch.exp2(-torch.arange(1.0, H + 1)).to(DEV)
    w = _weights(1)
    leaves = [t.clone().requires_grad_(True) for t in (x, r, *w.values())]
    out, stream, _ = _block(leaves[0], leaves[1], dict(zip(w, leaves[2:])), ld)
    got = [out, stream, *torch.autograd.grad((out, stream), leaves, (dy, ds))]
    exact = [t.detach().double().requires_grad_(True) for t in leaves]
    ref, ref_stream = _plain(exact[0], exact[1], dict(zip(w, exact[2:])), ld)
    want = [ref, ref_stream, *torch.autograd.grad((ref, ref_stream), exact, (dy.double(), ds.double()))]
    for name, a, b in zip(("out", "stream", "dx", "dresidual", *w), got, want):
        off = ((a.double() - b).norm() / b.norm()).item()
        assert off <= 12 * 2.0**-8, f"{name}: {off:.3g}"


def test_serving_in_8_bits():
    """A prompt through the 8-bit block, then token by token from its state: the same as the whole sequence at once,
    to the rounding of bfloat16 activations that meet the same 8-bit values (a step of 8 bits where they do not)."""

    n, more = 130, 9
    g = torch.Generator().manual_seed(5)
    x, r = (torch.randn(2, n + more, C, generator=g).bfloat16().to(DEV) for _ in range(2))
    ld = -torch.exp2(-torch.arange(1.0, H + 1)).to(DEV)
    w = _weights(2)
    qkv, out = (oops_amd.quantize_int8(w[name]) for name in ("qkv", "out"))

    def project(x, r):
        q8, s8, stream = oops_amd.rms_norm_int8(x, C, w["norm"], residual=r)
        return oops_amd.int8_linear(q8, s8, *qkv), stream

    def finish(att):
        return oops_amd.int8_linear(*oops_amd.quantize_int8(att), *out)

    with torch.no_grad():
        t, stream = project(x, r)
        whole, last = oops_amd.linear_attention(*_heads(t), ld, return_state=True)
        whole = finish(whole.transpose(1, 2).flatten(2))
        t, _ = project(x[:, :n], r[:, :n])
        att, state = oops_amd.linear_attention(*_heads(t), ld, return_state=True)
        pieces = [finish(att.transpose(1, 2).flatten(2))]
        for i in range(n, n + more):
            t, s = project(x[:, i], r[:, i])
            assert torch.equal(s, stream[:, i])
            q, k, v = t.unflatten(-1, (3, H, D)).unbind(-3)
            pieces.append(finish(oops_amd.linear_attention_step(q, k, v, ld, state).flatten(1))[:, None])
    got = torch.cat(pieces, 1)
    # projections are the same bits; the attention's outputs may differ by its bfloat16 roundings (2 half steps), and an
    # 8-bit step (1/127 of a row's largest value, itself below 4 of its norms over the root of its 128 values)
    off = ((got.double() - whole.double()).norm() / whole.double().norm()).item()
    assert off <= 2 * 2.0**-8 + 4 / 127 / 2, off
    torch.testing.assert_close(state, last, rtol=0, atol=float(last.abs().max()) * 2.0**-15)
