"""The decoder's operators together, as a block of a model uses them: the residual's addition and norm, projections, the
heads' norm and rotation, causal attention over packed sequences, the gated output stage; trained in bfloat16, and served from
prompts to single tokens over the 4-bit cache, eagerly and as a replayed graph.

Training is compared with the same block in float64 PyTorch operations.  A path crosses at most sixteen roundings to bfloat16
(the normed stream, projections, rotated heads, weights, attention, gate, gated values and output; their gradients on the way
back), a rounding reaches the next tensor multiplied by at most the ratio of the sums' magnitudes, and in the 2-norm
independent roundings do not add up: 16 half steps.

Serving has two ways to one result: the steps' attention reads codes, and causal attention over what they stand for (exact in
bfloat16) gives the same rows.  Either is off by its weights' and its result's rounding, each at most half a step in the
2-norm, so they differ by at most 4 half steps.
"""

import pytest
import torch

import oops_amd
from layer_tolerance import half

pytestmark = pytest.mark.gpu

DEV = "cuda"
H, G, D, C, PAGE = 4, 2, 32, 128, 16


def _weights(seed):
    g = torch.Generator().manual_seed(seed)
    lin = lambda n, k: (torch.randn(n, k, generator=g) * k**-0.5).bfloat16().to(DEV)  # noqa: E731
    one = lambda n: (1 + 0.1 * torch.randn(n, generator=g)).to(DEV)  # noqa: E731
    w = {"qkv": lin((H + 2 * G) * D, C), "gate": lin(H * D, C), "out": lin(C, H * D)}
    return w | {"norm": one(C), "wq": one(D), "wk": one(D)}


def _heads(t):
    return [x.transpose(-2, -3) for x in t.unflatten(-1, (H + 2 * G, D)).split((H, G, G), -2)]  # token-major views


def _block(x, residual, w, table, positions, offsets):
    y, stream = oops_amd.rms_norm(x, C, w["norm"], residual=residual)
    q, k, v = _heads(torch.nn.functional.linear(y, w["qkv"]))
    q, k = oops_amd.rms_norm_rotary(q, k, table, positions, w["wq"], w["wk"])
    att = oops_amd.causal_attention(q, k, v, offsets)
    return oops_amd.gate_attention_output(att, y, w["gate"], w["out"]), stream


def _plain(x, residual, w, table, positions, sequence):
    norm = lambda t: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6)  # noqa: E731
    stream = x + residual
    y = norm(stream) * w["norm"]
    q, k, v = _heads(y @ w["qkv"].t())
    cos, sin = table.double()[positions][None, None].unbind(-2)

    def turn(t):
        a, b = t.chunk(2, -1)
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    q, k = turn(norm(q) * w["wq"]), turn(norm(k) * w["wk"])
    k, v = (t.repeat_interleave(H // G, 1) for t in (k, v))
    pair = (sequence[:, None] == sequence[None]).tril()
    p = torch.softmax((q @ k.transpose(-1, -2) * D**-0.5).masked_fill(~pair, -torch.inf), -1)
    gate = torch.sigmoid(y @ w["gate"].t())
    return (gate * (p @ v).transpose(1, 2).flatten(2)) @ w["out"].t(), stream


@pytest.mark.parametrize("lengths", [[1], [70], [130, 1, 0, 169]])
def test_training(lengths):
    n = sum(lengths)
    g = torch.Generator().manual_seed(n)
    x, r, dy, ds = ((torch.randn(2, n, C, generator=g)).bfloat16().to(DEV) for _ in range(4))
    positions = torch.cat([torch.arange(m) for m in lengths]).to(DEV)
    sequence = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(lengths)).to(DEV)
    offsets = torch.tensor([0, *lengths]).cumsum(0).to(DEV)
    table, w = oops_amd.rotary_table(200, D, device=DEV), _weights(1)
    leaves = [t.clone().requires_grad_(True) for t in (x, r, *w.values())]
    outs = _block(leaves[0], leaves[1], dict(zip(w, leaves[2:])), table, positions, offsets)
    got = [*outs, *torch.autograd.grad(outs, leaves, (dy, ds))]
    exact = [t.detach().double().requires_grad_(True) for t in leaves]
    ref = _plain(exact[0], exact[1], dict(zip(w, exact[2:])), table, positions, sequence)
    want = [*ref, *torch.autograd.grad(ref, exact, (dy.double(), ds.double()))]
    for name, a, b in zip(("out", "stream", "dx", "dresidual", *w), got, want):
        if n == 1 and name in ("wq", "wk"):  # (one key has the whole weight, whatever its score)
            assert a.double().norm() <= 16 * half(torch.bfloat16) * dy.double().norm()
            continue
        off = ((a.double() - b).norm() / b.norm()).item()
        assert off <= 16 * half(torch.bfloat16), f"{name}: {off:.3g}"


class _Server:
    """A decoder's attention in 8-bit projections and a 4-bit cache of pages in any order."""

    def __init__(self, lengths, room):
        g = torch.Generator().manual_seed(9)
        self.w = _weights(2)
        self.qkv = oops_amd.quantize_int8(self.w["qkv"])
        self.table = oops_amd.rotary_table(room, D, device=DEV)
        width = -(-room // PAGE)
        self.pages = torch.randperm(len(lengths) * width + 1, generator=g)[: len(lengths) * width].view(len(lengths), width).int().to(DEV)
        self.cache = oops_amd.quantized_cache(len(lengths) * width + 1, G, D, page_size=PAGE, device=DEV)

    def slots(self, sequence, positions):
        return self.pages[sequence, positions // PAGE] * PAGE + positions % PAGE

    def project(self, x, residual, positions):
        values, scales, _ = oops_amd.rms_norm_int8(x, C, self.w["norm"], residual=residual)
        q, k, v = _heads(oops_amd.int8_linear(values, scales, *self.qkv))
        return *oops_amd.rms_norm_rotary(q, k, self.table, positions, self.w["wq"], self.w["wk"]), v

    def prompts(self, x, residual, sequence, positions, offsets):
        """Packed prompts (1, L, C): their attention, and their keys and values in the cache."""

        q, k, v = self.project(x, residual, positions)
        oops_amd.cache_write(*self.cache, k[0], v[0], self.slots(sequence, positions))
        return oops_amd.causal_attention(q, k, v, offsets), q

    def step(self, x, residual, positions):
        """One token (B, 1, C) of every sequence."""

        q, k, v = self.project(x, residual, positions[:, None])
        row = torch.arange(len(positions), device=DEV)
        oops_amd.cache_write(*self.cache, k, v, self.slots(row, positions)[:, None])
        return oops_amd.cache_attention(q[:, :, 0], *self.cache, self.pages, positions + 1), q


@pytest.mark.parametrize("graph", [False, True])
@torch.no_grad()
def test_serving(graph):
    lengths, more = [130, 57, 0], 20
    g = torch.Generator().manual_seed(5)
    s = _Server(lengths, max(lengths) + more)
    n = sum(lengths)
    x, r = (torch.randn(1, n, C, generator=g).bfloat16().to(DEV) for _ in range(2))
    sequence = torch.repeat_interleave(torch.arange(3), torch.tensor(lengths)).to(DEV)
    positions = torch.cat([torch.arange(m) for m in lengths]).to(DEV)
    att, prompt_q = s.prompts(x, r, sequence, positions, torch.tensor([0, *lengths]).cumsum(0).to(DEV))
    assert att.shape == (1, H, n, D)
    steps = [(torch.randn(3, 1, C, generator=g).bfloat16().to(DEV), torch.randn(3, 1, C, generator=g).bfloat16().to(DEV)) for _ in range(more)]
    at = torch.tensor(lengths, device=DEV)
    bx, br, bp = steps[0][0].clone(), steps[0][1].clone(), at.clone()
    if graph:
        # (the warm-up writes the first step's tokens, which the first replay writes again)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            s.step(bx, br, bp)
        torch.cuda.current_stream().wait_stream(side)
        recorded = torch.cuda.CUDAGraph()
        with torch.cuda.graph(recorded):
            static = s.step(bx, br, bp)
    outs, queries = [], []
    for i, (tx, tr) in enumerate(steps):
        if graph:
            bx.copy_(tx), br.copy_(tr), bp.copy_(at + i)
            recorded.replay()
            out, q = (t.clone() for t in static)
        else:
            out, q = s.step(tx, tr, at + i)
        outs.append(out), queries.append(q[:, :, 0])
    for b, m in enumerate(lengths):
        p = torch.arange(m + more, device=DEV)
        k, v = oops_amd.cache_read(*s.cache, s.slots(torch.full_like(p, b), p))
        first = sum(lengths[:b])
        q = torch.cat((prompt_q[0, :, first : first + m], torch.stack([q[b] for q in queries], 1)), 1)
        want = oops_amd.causal_attention(q, k, v)[:, m:].double()
        got = torch.stack([o[b] for o in outs], 1).double()
        off = ((got - want).norm() / want.norm()).item()
        assert off <= 4 * half(torch.bfloat16), off
        # and the prompt's own attention to unquantized keys is the step's to the rounding of 4 bits
        if m:
            stood = oops_amd.causal_attention(q, k, v)[:, :m].double()
            own = att[0, :, first : first + m].double()
            assert torch.nn.functional.cosine_similarity(own.flatten(), stood.flatten(), 0) > 0.95
