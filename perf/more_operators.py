"""Performance cases of softmax attention in a decoder: norm and rotation of queries and keys, attention over whole
prompts, and the key/value cache in 4 bits.

A case is a dict of plain values; ``kind`` names the operator it times:

* ``rotary``: ``rms_norm_rotary``, queries and keys of ``batch`` x ``length`` tokens; ``train`` runs the forward and the
  backward of both and of their weights;
* ``attend``: ``causal_attention``; ``sequences`` > 0 packs that many sequences of different lengths into ``length``
  tokens (``batch`` 1), else every batch element is one sequence; ``train`` runs the forward and the backward;
* ``write``: ``cache_write`` of ``length`` tokens and ``cache_read`` of the same ones;
* ``decode``: ``cache_attention``, one token of each of ``batch`` sequences of up to ``length`` cached tokens.

Operands are token-major views, as projections leave them.  Queries and keys are unit normal (what a norm leaves), with
some channels of the keys larger than others, as trained models have them; values are unit normal.  Cached blocks of 32
channels hold 4-bit floating point codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign) and one exponent.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6
BASE = 500000.0
BLOCK = 32  # channels that share an exponent


def listed():
    return [
        # decoding: four sequences, one token each; latency counts
        dict(name="rotary_decode", kind="rotary", batch=4, length=1, heads=32, kv_heads=8, d=128, rotary=128, train=False,
             dtype="bf16"),
        # a training step's queries and keys
        dict(name="rotary_train", kind="rotary", batch=1, length=8192, heads=32, kv_heads=8, d=128, rotary=128, train=True,
             dtype="bf16"),
        # a head size that is no power of two, half of it rotated, float32
        dict(name="rotary_odd", kind="rotary", batch=3, length=333, heads=6, kv_heads=2, d=80, rotary=40, train=True,
             dtype="f32"),
        # a training step: documents of different lengths packed into one row of 8192 tokens
        dict(name="attend_train", kind="attend", batch=1, length=8192, sequences=5, mix=1, heads=32, kv_heads=8, d=128,
             train=True, dtype="bf16"),
        # one long prompt
        dict(name="attend_prompt", kind="attend", batch=1, length=16384, sequences=0, mix=0, heads=16, kv_heads=2, d=128,
             train=False, dtype="bf16"),
        # odd sizes everywhere, float32, fine-tuned
        dict(name="attend_odd", kind="attend", batch=2, length=777, sequences=0, mix=0, heads=6, kv_heads=3, d=40,
             train=True, dtype="f32"),
        # many short sequences packed, a head of keys for each head of queries, half precision
        dict(name="attend_ragged", kind="attend", batch=1, length=5000, sequences=24, mix=2, heads=8, kv_heads=8, d=64,
             train=True, dtype="f16"),
        # decoding: a batch's new tokens
        dict(name="write_decode", kind="write", length=64, kv_heads=8, d=128, page=64, dtype="bf16"),
        # a long prompt's keys and values
        dict(name="write_prompt", kind="write", length=30011, kv_heads=8, d=128, page=64, dtype="bf16"),
        # decoding: one long sequence; the length has to be split
        dict(name="decode_one", kind="decode", batch=1, length=32768, heads=32, kv_heads=8, d=128, page=64, mix=0,
             dtype="bf16"),
        # decoding: a full batch of ragged lengths, bound by the cache's bytes
        dict(name="decode_batch", kind="decode", batch=64, length=16384, heads=32, kv_heads=8, d=128, page=64, mix=3,
             dtype="bf16"),
        # odd sizes, float32, small pages, sequences of no and of one token among them
        dict(name="decode_odd", kind="decode", batch=5, length=999, heads=9, kv_heads=3, d=96, page=16, mix=4, dtype="f32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "attend", "attend", "write", "decode", "decode"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 5, 8])
    if kind == "rotary":
        d = rng.choice([64, 128, 128, 2 * _log_int(rng, 4, 128)])
        rotary = d if rng.random() < 0.7 else 2 * rng.randint(1, d // 2)
        batch = _log_int(rng, 1, 64)
        length = 1 if rng.random() < 0.3 else _log_int(rng, 1, max(1, min(8192, (1 << 25) // (batch * heads * d))))
        return dict(kind=kind, batch=batch, length=length, heads=heads, kv_heads=kv_heads, d=d, rotary=rotary,
                    train=rng.random() < 0.5, dtype=dtype)
    if kind == "attend":
        d = rng.choice([64, 128, 128, 128, 96, _log_int(rng, 8, 128)])
        batch = _log_int(rng, 1, 16)
        sequences = 0
        if rng.random() < 0.5:
            batch, sequences = 1, _log_int(rng, 1, 64)
        top = min(16384, math.isqrt((1 << 29) // (batch * heads)))
        return dict(kind=kind, batch=batch, length=_log_int(rng, 1, top), sequences=sequences, mix=rng.randrange(1 << 20),
                    heads=heads, kv_heads=kv_heads, d=d, train=rng.random() < 0.5, dtype=dtype)
    d = rng.choice([32, 64, 64, 96, 128, 128, 128])
    page = rng.choice([16, 32, 64, 64, 128])
    if kind == "write":
        return dict(kind=kind, length=_log_int(rng, 1, 30011), kv_heads=kv_heads, d=d, page=page, dtype=dtype)
    batch = _log_int(rng, 1, 64)
    length = _log_int(rng, 1, min(65536, (1 << 20) // batch))
    return dict(kind=kind, batch=batch, length=length, heads=heads, kv_heads=kv_heads, d=d, page=page,
                mix=rng.randrange(1 << 20), dtype=dtype)


# ----------------------------------------------------------------- inputs


def _bounds(case):
    """Where the packed sequences begin and the last one ends: ``sequences`` lengths that fill ``length``."""

    n, s = case["length"], case["sequences"]
    if not s:
        return [0, n]
    rng = random.Random(case["mix"])
    return [0, *sorted(rng.randint(0, n) for _ in range(s - 1)), n]


def _cached(case):
    """Tokens in the cache for each sequence: the first has them all; in a mix others have any number, 1 and 0 too."""

    n, b = case["length"], case["batch"]
    if not case["mix"]:
        return [n] * b
    rng = random.Random(case["mix"])
    counts = [n] + [rng.randint(n // 4, n) for _ in range(b - 1)]
    if b > 3:
        counts[1], counts[2] = 0, 1
    return counts


class _Maker:
    def __init__(self, seed, dtype):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.dtype = dtype

    def randn(self, *shape, dtype=None):
        return torch.randn(*shape, generator=self.gen, device="cuda").to(dtype or self.dtype)

    def heads(self, b, n, h, d, gain=None):
        """(b, h, n, d), token-major memory; ``gain`` weighs the channels."""

        t = torch.randn(b, n, h, d, generator=self.gen, device="cuda")
        return (t if gain is None else t * gain).to(self.dtype).transpose(1, 2)

    def gain(self, d):
        return torch.exp(0.5 * torch.randn(d, generator=self.gen, device="cuda"))


def _angles(length, rotary):
    """(length, 2, rotary / 2) cosines and sines, angles in float64."""

    freq = BASE ** (-torch.arange(rotary // 2, device="cuda", dtype=torch.float64) * 2 / rotary)
    a = torch.arange(length, device="cuda", dtype=torch.float64)[:, None] * freq
    return torch.stack((a.cos(), a.sin()), 1).float()


def _quantized(x):
    """4-bit codes and exponents of float32 x (..., d): the smallest scale 2^e with max|block| <= 6 * 2^e, values rounded
    to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the even code).  Returns the codes (0..15) and e + 127."""

    b = x.unflatten(-1, (-1, BLOCK))
    m, e = torch.frexp(b.abs().amax(-1))
    e = torch.where(m > 0.75, e - 2, e - 3).clamp(-126, 125)
    e = torch.where(m == 0, -126, e)
    q = torch.ldexp(b.abs(), -e[..., None]).clamp(max=6.0)
    low, mid = torch.round(q * 2), torch.round(q) + 2
    code = torch.where(q < 2, low, torch.where(q < 4, mid, torch.round(q * 0.5) + 4))
    code = code.to(torch.uint8) | (torch.signbit(b).to(torch.uint8) << 3)
    return code.flatten(-2), (e + 127).to(torch.uint8)


def _values(code, exponent):
    """What codes (..., d) and exponents (..., d / 32) stand for, float32."""

    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=code.device)
    v = table[(code & 7).long()]
    v = torch.where(code >= 8, -v, v).unflatten(-1, (-1, BLOCK))
    return torch.ldexp(v, exponent.int()[..., None] - 127).flatten(-2)


def _inputs(case, seed):
    m = _Maker(seed, DTYPES[case["dtype"]])
    kind, d, n = case["kind"], case["d"], case["length"]
    if kind == "rotary":
        b, h, g = case["batch"], case["heads"], case["kv_heads"]
        gain = m.gain(d)
        x = {"query": m.heads(b, n, h, d, gain), "key": m.heads(b, n, g, d, gain), "table": _angles(32768, case["rotary"])}
        x["query_weight"], x["key_weight"] = (1 + 0.1 * m.randn(d, dtype=torch.float32) for _ in range(2))
        start = torch.randint(0, 32768 - n, (b, 1), generator=m.gen, device="cuda")
        x["positions"] = (start + torch.arange(n, device="cuda")).int()
        if case["train"]:
            x["dquery"], x["dkey"] = m.heads(b, n, h, d), m.heads(b, n, g, d)
        return x
    if kind == "attend":
        b, h, g = case["batch"], case["heads"], case["kv_heads"]
        x = {"query": m.heads(b, n, h, d), "key": m.heads(b, n, g, d, m.gain(d)), "value": m.heads(b, n, g, d)}
        if case["train"]:
            x["dout"] = m.heads(b, n, h, d)
        if case["sequences"]:
            x = {name: t[0] for name, t in x.items()}
            x["offsets"] = torch.tensor(_bounds(case), dtype=torch.int32, device="cuda")
        return x
    g, page = case["kv_heads"], case["page"]
    if kind == "write":
        x = {"key": m.heads(1, n, g, d, m.gain(d))[0], "value": m.heads(1, n, g, d)[0]}
        pages = n // page + 3
        order = torch.randperm(pages, generator=m.gen, device="cuda")
        t = torch.arange(n, device="cuda") + page // 2  # (a sequence is continued inside a page)
        x["slots"] = order[t // page] * page + t % page
        x["codes"] = torch.zeros(pages, g, 2, page, d // 2, dtype=torch.uint8, device="cuda")
        x["scales"] = torch.zeros(pages, g, 2, page, d // BLOCK, dtype=torch.uint8, device="cuda")
        return x
    counts, b = _cached(case), case["batch"]
    width = max(1, -(-n // page))
    used = sum(-(-c // page) for c in counts)
    pages = used + 2
    codes = torch.empty(pages, g, 2, page, d // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(pages, g, 2, page, d // BLOCK, dtype=torch.uint8, device="cuda")
    gain = torch.stack((m.gain(d), torch.ones(d, device="cuda")))[:, None]
    step = max(1, (1 << 25) // (g * 2 * page * d))
    for i in range(0, pages, step):
        k = min(step, pages - i)
        code, exponent = _quantized(m.randn(k, g, 2, page, d, dtype=torch.float32) * gain)
        codes[i : i + k] = code[..., 0::2] | (code[..., 1::2] << 4)
        scales[i : i + k] = exponent
    order = torch.randperm(pages, generator=m.gen, device="cuda").int()
    table, at = torch.zeros(b, width, dtype=torch.int32, device="cuda"), 0
    for i, c in enumerate(counts):
        k = -(-c // page)
        table[i, :k] = order[at : at + k]
        at += k
    lengths = torch.tensor(counts, dtype=torch.int32, device="cuda")
    return {"query": m.randn(b, case["heads"], d), "codes": codes, "scales": scales, "pages": table, "lengths": lengths}


def _leaf_names(case):
    if not case.get("train"):
        return []
    if case["kind"] == "rotary":
        return ["query", "key", "query_weight", "key_weight"]
    return ["query", "key", "value"]


def prepare(case, seed):
    x = _inputs(case, seed)
    for name in _leaf_names(case):
        x[name].requires_grad_(True)
    return case, x


# ----------------------------------------------------------------- plain forms


def _turn(x, cos, sin, back=False):
    """Channels i and i + R / 2 of x (b, h, n, d) turned by their token's angle; those behind R stay."""

    half = cos.shape[-1]
    a, b = x[..., :half], x[..., half : 2 * half]
    sin = -sin if back else sin
    return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., 2 * half :]), -1)


def _plain_rotary(case, x):
    rows = x["table"][x["positions"].long()][:, None]  # (b, 1, n, 2, R / 2)
    cos, sin = rows[..., 0, :], rows[..., 1, :]
    outs, grads, wgrads = [], [], []
    for name in ("query", "key"):
        t, w = x[name].float(), x[name + "_weight"]
        rstd = torch.rsqrt((t * t).mean(-1, keepdim=True) + EPS)
        n = t * rstd
        outs.append(_turn(n * w, cos, sin).to(x[name].dtype))
        if case["train"]:
            g = _turn(x["d" + name].float(), cos, sin, back=True)
            wgrads.append((g * n).sum((0, 1, 2)))
            g = g * w
            grads.append((rstd * (g - n * (g * n).mean(-1, keepdim=True))).to(x[name].dtype))
    return (*outs, *grads, *wgrads)


ROWS = 2048  # queries at once in the plain form


def _plain_sequence(case, q, k, v, do):
    """One sequence: q (g, r, n, d), k and v (g, n, d), float32.  Returns out and, with do, the gradients."""

    n, scale = q.shape[2], case["d"] ** -0.5
    out = torch.zeros_like(q)
    dq, dk, dv = (torch.zeros_like(t) for t in (q, k, v)) if do is not None else (None, None, None)
    for i in range(0, n, ROWS):
        j = min(n, i + ROWS)
        kj, vj = k[:, None, :j], v[:, None, :j]
        s = (q[:, :, i:j] @ kj.transpose(2, 3)) * scale
        t = torch.arange(j, device=q.device)
        s = s.masked_fill(t > t[i:j, None], -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        out[:, :, i:j] = p @ vj
        if do is not None:
            w = do[:, :, i:j]
            dv[:, :j] += (p.transpose(2, 3) @ w).sum(1)
            dp = w @ vj.transpose(2, 3)
            ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
            dq[:, :, i:j] = ds @ kj
            dk[:, :j] += (ds.transpose(2, 3) @ q[:, :, i:j]).sum(1)
    return (out,) if do is None else (out, dq, dk, dv)


def _plain_attend(case, x):
    dt, h, g = DTYPES[case["dtype"]], case["heads"], case["kv_heads"]
    packed = bool(case["sequences"])
    names = ("query", "key", "value", "dout") if case["train"] else ("query", "key", "value")
    q, k, v, *do = ((x[name][None] if packed else x[name]).float() for name in names)
    q, *do = (t.unflatten(1, (g, h // g)) for t in (q, *do))
    outs = [torch.zeros_like(t) for t in ((q, q, k, v) if case["train"] else (q,))]
    bounds = _bounds(case)
    for b in range(q.shape[0]):
        for lo, hi in zip(bounds, bounds[1:]):
            parts = [t[b, ..., lo:hi, :] for t in (q, k, v, *do)]
            for to, part in zip(outs, _plain_sequence(case, *parts, *([] if do else [None]))):
                to[b, ..., lo:hi, :] = part
    outs = [t.flatten(1, 2) if t.dim() == 5 else t for t in outs]
    return tuple((t[0] if packed else t).to(dt) for t in outs)


def _plain_write(case, x):
    return tuple(_values(*_quantized(x[name].float())).to(x[name].dtype) for name in ("key", "value"))


def _plain_decode(case, x):
    d, g, page = case["d"], case["kv_heads"], case["page"]
    q = x["query"].float().unflatten(1, (g, -1))
    out = torch.zeros_like(q)
    for b, count in enumerate(_cached(case)):
        if not count:
            continue
        ids = x["pages"][b, : -(-count // page)].long()
        code = x["codes"][ids]
        code = torch.stack((code & 15, code >> 4), -1).flatten(-2)
        kv = _values(code, x["scales"][ids]).permute(2, 1, 0, 3, 4).flatten(2, 3)[:, :, :count]  # (2, g, count, d)
        s = (q[b] @ kv[0].transpose(1, 2)) * d**-0.5
        p = torch.exp(s - s.amax(-1, keepdim=True))
        out[b] = (p @ kv[1]) / p.sum(-1, keepdim=True)
    return out.flatten(1, 2).to(x["query"].dtype)


# ----------------------------------------------------------------- the framework's calls


def _own(case, x):
    import oops_amd

    kind = case["kind"]
    if kind == "rotary":
        q, k = oops_amd.rms_norm_rotary(x["query"], x["key"], x["table"], x["positions"], x["query_weight"],
                                        x["key_weight"], EPS)
        if not case["train"]:
            return q, k
        leaves = [x[name] for name in _leaf_names(case)]
        return (q.detach(), k.detach(), *torch.autograd.grad((q, k), leaves, (x["dquery"], x["dkey"])))
    if kind == "attend":
        out = oops_amd.causal_attention(x["query"], x["key"], x["value"], x.get("offsets"))
        if not case["train"]:
            return (out,)
        leaves = [x[name] for name in _leaf_names(case)]
        return (out.detach(), *torch.autograd.grad(out, leaves, x["dout"]))
    if kind == "write":
        oops_amd.cache_write(x["codes"], x["scales"], x["key"], x["value"], x["slots"])
        return oops_amd.cache_read(x["codes"], x["scales"], x["slots"], dtype=x["key"].dtype)
    return oops_amd.cache_attention(x["query"], x["codes"], x["scales"], x["pages"], x["lengths"])


def run(state):
    case, x = state
    if own:
        return _own(case, x)
    with torch.no_grad():
        plain = {"rotary": _plain_rotary, "attend": _plain_attend, "write": _plain_write, "decode": _plain_decode}
        return plain[case["kind"]](case, x)


# ----------------------------------------------------------------- what a pass cannot do without


def work(case):
    kind, d = case["kind"], case["d"]
    el = 4 if case["dtype"] == "f32" else 2
    if kind == "rotary":
        tokens = case["batch"] * case["length"]
        cells = tokens * (case["heads"] + case["kv_heads"]) * d
        # forward: read and written; backward: input and gradient read, gradient written
        passes = 5 if case["train"] else 2
        return {"bytes": cells * el * passes + tokens * case["rotary"] * 4, "flops": 5 * passes * cells}
    if kind == "attend":
        bounds = _bounds(case)
        pairs = case["batch"] * sum((b - a) * (b - a + 1) // 2 for a, b in zip(bounds, bounds[1:]))
        q = case["batch"] * case["length"] * case["heads"] * d
        kv = case["batch"] * case["length"] * case["kv_heads"] * d
        flops, cells = 4 * pairs * case["heads"] * d, 2 * q + 2 * kv
        if case["train"]:
            # scores and their gradient, and the products of dv, dq and dk; q, k, v, out, dout read, three written
            flops += 10 * pairs * case["heads"] * d
            cells += 4 * q + 4 * kv
        return {"bytes": cells * el, "flops": flops}
    cached = 2 * case["kv_heads"] * (d // 2 + d // BLOCK)  # bytes of a token
    if kind == "write":
        cells = 2 * case["length"] * case["kv_heads"] * d
        # keys and values read, their codes written, read again, and the values they stand for written
        return {"bytes": 2 * cells * el + 2 * case["length"] * cached, "flops": 8 * cells}
    tokens = sum(_cached(case))
    return {"bytes": tokens * cached + 2 * case["batch"] * case["heads"] * d * el, "flops": 4 * tokens * case["heads"] * d}


# ----------------------------------------------------------------- float64 definition


def _exact_rotary(case, x):
    """Pairs (i, i + R / 2) as complex numbers, multiplied by the token's unit number (or its conjugate, backwards)."""

    half = case["rotary"] // 2
    row = x["table"].double()[x["positions"].long()]
    unit = torch.complex(row[..., 0, :], row[..., 1, :])[:, None]

    def rotated(t, by):
        z = torch.complex(t[..., :half].contiguous(), t[..., half : 2 * half].contiguous()) * by
        return torch.cat((z.real, z.imag, t[..., 2 * half :]), -1)

    ys, dxs, dws = [], [], []
    for name in ("query", "key"):
        t, w = x[name].detach().double(), x[name + "_weight"].detach().double()
        rms = (t.square().sum(-1, keepdim=True) / case["d"] + EPS).sqrt()
        ys.append(rotated(t / rms * w, unit))
        if case["train"]:
            dn = rotated(x["d" + name].double(), unit.conj())
            dws.append((dn * (t / rms)).flatten(0, 2).sum(0))
            dn = dn * w
            dxs.append(dn / rms - t * (dn * t).sum(-1, keepdim=True) / (case["d"] * rms**3))
    return (*ys, *dxs, *dws)


def _exact_attend(case, x):
    h, r = case["heads"], case["heads"] // case["kv_heads"]
    lift = lambda t: t.detach().double()[None] if case["sequences"] else t.detach().double()  # noqa: E731
    q, k, v = lift(x["query"]), lift(x["key"]), lift(x["value"])
    do = lift(x["dout"]) if case["train"] else None
    out = torch.zeros_like(q)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    bounds = _bounds(case)
    for lo, hi in zip(bounds, bounds[1:]):
        at = slice(lo, hi)
        mask = torch.ones(hi - lo, hi - lo, dtype=torch.bool, device=q.device).tril()
        for b in range(q.shape[0]):
            for i in range(h):
                if hi == lo:
                    continue
                s = q[b, i, at] @ k[b, i // r, at].T / math.sqrt(case["d"])
                p = torch.softmax(torch.where(mask, s, -math.inf), -1)
                del s
                out[b, i, at] = p @ v[b, i // r, at]
                if do is None:
                    continue
                w = do[b, i, at]
                dv[b, i // r, at] += p.T @ w
                # dS = P (dP - o . do): the softmax's gradient
                ds = p * (w @ v[b, i // r, at].T - (out[b, i, at] * w).sum(-1, keepdim=True)) / math.sqrt(case["d"])
                dq[b, i, at] = ds @ k[b, i // r, at]
                dk[b, i // r, at] += ds.T @ q[b, i, at]
    outs = (out,) if do is None else (out, dq, dk, dv)
    return tuple(t[0] if case["sequences"] else t for t in outs)


def _exact_values(t):
    """The nearest point of the block's grid, by distance; a tie goes to the point with the even code."""

    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=t.device)
    b = t.detach().double().unflatten(-1, (-1, BLOCK))
    top = b.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(top / 6))
    e = e + (top > 6 * torch.exp2(e)).double() - (top <= 3 * torch.exp2(e)).double()
    unit = torch.where(top > 0, torch.exp2(e.clamp(-126, 125)), torch.ones_like(top))
    a = (b.abs() / unit).clamp(max=6.0)
    far = torch.full_like(a, math.inf)
    value = torch.zeros_like(a)
    for code in (0, 2, 4, 6, 1, 3, 5, 7):  # even codes first: an odd one has to be strictly nearer
        dist = (a - grid[code]).abs()
        value = torch.where(dist < far, grid[code], value)
        far = torch.minimum(dist, far)
    return (value * unit * torch.sign(b)).flatten(-2)


def _exact_decode(case, x):
    d, r, page = case["d"], case["heads"] // case["kv_heads"], case["page"]
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")
    grid = torch.cat((grid, -grid))
    out = torch.zeros(case["batch"], case["heads"], d, dtype=torch.float64, device="cuda")
    for b, count in enumerate(_cached(case)):
        t = torch.arange(count, device="cuda")
        ids = x["pages"][b].long()[t // page]
        for i in range(case["kv_heads"] if count else 0):
            kv = []
            for which in (0, 1):
                byte = x["codes"][ids, i, which, t % page].long()
                val = torch.stack((grid[byte % 16], grid[byte // 16]), -1).flatten(1)
                unit = torch.exp2(x["scales"][ids, i, which, t % page].double() - 127)
                kv.append(val * unit.repeat_interleave(BLOCK, 1))
            heads = slice(i * r, (i + 1) * r)
            p = torch.softmax(x["query"][b, heads].double() @ kv[0].T / math.sqrt(d), -1)
            out[b, heads] = p @ kv[1]
    return out


def exact(case, seed):
    """``run``'s outputs by the definition, in float64."""

    x = _inputs(case, seed)
    if case["kind"] == "rotary":
        return _exact_rotary(case, x)
    if case["kind"] == "attend":
        return _exact_attend(case, x)
    if case["kind"] == "write":
        return tuple(_exact_values(x[name]) for name in ("key", "value"))
    return _exact_decode(case, x)
