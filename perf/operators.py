"""Performance cases of the layer operators: root-mean-square norm, 8-bit linear layers, linear attention.

A case is a dict of plain values; ``kind`` names the operator it times:

* ``norm``: ``rms_norm``, with or without the residual's addition; forward and backward of a training step;
* ``norm8``: ``rms_norm_int8``, the norm in front of an 8-bit projection, with the residual's addition;
* ``int8``: ``int8_linear``; with ``quantize`` the call starts from activations (``quantize_int8`` before it);
* ``linear``: ``linear_attention``; ``train`` runs the forward and the backward of every operand, ``state`` starts
  from a state and returns the last one, ``ragged`` is a padded batch with lengths (a length of zero among them);
* ``step``: ``linear_attention_step``, one token of every sequence of a batch.

Queries and keys are non-negative features (SiLU of unit normals), as linear attention takes them; the decays of the
heads fall from exp(-1/2) to exp(-1/256) geometrically.  q, k and v are token-major views, as projections leave
them.  Residual streams and values are unit normal, weights of 8-bit layers are quantized normal rows.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6
CHUNK = 128  # tokens of a chunk in the plain form


def listed():
    return [
        # the pair representation of a 256-residue crop, normalized without a residual, training
        dict(name="norm_pair_train", kind="norm", rows=65536, width=128, residual=False, dtype="bf16"),
        # a block's input in training: the residual stream of 8192 tokens
        dict(name="norm_wide_train", kind="norm", rows=8192, width=4096, residual=True, dtype="bf16"),
        # decoding: four sequences, one token each; latency counts
        dict(name="norm8_decode", kind="norm8", rows=4, width=4096, residual=True, dtype="bf16"),
        # a prompt's residual stream in front of an 8-bit projection
        dict(name="norm8_prompt", kind="norm8", rows=8192, width=8192, residual=True, dtype="f16"),
        # decoding: four tokens through an 8-bit layer, bound by the weight's bytes
        dict(name="int8_decode", kind="int8", rows=4, k=4096, n=16384, bias=False, quantize=True, dtype="bf16"),
        # odd sizes everywhere, float32 results with a bias
        dict(name="int8_odd", kind="int8", rows=333, k=1001, n=777, bias=True, quantize=False, dtype="f32"),
        # a prompt of 8192 tokens through an 8-bit layer
        dict(name="int8_prompt", kind="int8", rows=8192, k=4096, n=16384, bias=False, quantize=True, dtype="bf16"),
        # a training step's token mixing
        dict(name="linear_train", kind="linear", batch=4, heads=16, length=4096, d=128, e=128, train=True, state=False,
             ragged=False, dtype="bf16"),
        # one long prompt continued from a state, its last state kept for decoding
        dict(name="linear_prompt", kind="linear", batch=1, heads=16, length=30011, d=128, e=128, train=False,
             state=True, ragged=False, dtype="bf16"),
        # a padded batch of ragged lengths in half precision, fine-tuned from a learned state
        dict(name="linear_ragged", kind="linear", batch=6, heads=8, length=777, d=64, e=64, train=True, state=True,
             ragged=True, dtype="f16"),
        # decoding: one sequence; latency counts
        dict(name="step_one", kind="step", batch=1, heads=16, d=128, e=128, dtype="bf16"),
        # decoding: a full batch, bound by the states' bytes
        dict(name="step_batch", kind="step", batch=256, heads=32, d=128, e=128, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm8", "int8", "linear", "linear", "step"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind in ("norm", "norm8"):
        # (8-bit values are returned in the input's type: 16 bits, where one step at a border is a rounding)
        dtype = "bf16" if kind == "norm8" and dtype == "f32" else dtype
        width = rng.choice([_log_int(rng, 17, 8192), 8 * _log_int(rng, 2, 1024)])
        rows = _log_int(rng, 1, min(65536, (1 << 26) // width))
        return dict(kind=kind, rows=rows, width=width, residual=rng.random() < 0.6, dtype=dtype)
    if kind == "int8":
        k = rng.choice([_log_int(rng, 33, 8192), 64 * _log_int(rng, 1, 128)])
        n = rng.choice([_log_int(rng, 17, 16384), 64 * _log_int(rng, 1, 256)])
        rows = _log_int(rng, 1, min(8192, (1 << 38) // (k * n)))
        quantize = rng.random() < 0.5
        # quantized activations may differ by one step at a border: float32 results only from given ones
        dtype = "bf16" if quantize and dtype == "f32" else dtype
        return dict(kind=kind, rows=rows, k=k, n=n, bias=rng.random() < 0.5, quantize=quantize, dtype=dtype)
    d = rng.choice([32, 64, 64, 96, 128, 128, _log_int(rng, 8, 128)])
    e = d if rng.random() < 0.7 else rng.choice([32, 64, 128, _log_int(rng, 8, 128)])
    if kind == "step":
        batch = _log_int(rng, 1, 256)
        return dict(kind=kind, batch=batch, heads=rng.choice([1, 4, 8, 16, 32]), d=d, e=e, dtype=dtype)
    heads = rng.choice([1, 2, 4, 8, 12, 16])
    batch = _log_int(rng, 1, 8)
    length = _log_int(rng, 1, min(32768, (1 << 18) // (heads * batch)))
    return dict(kind=kind, batch=batch, heads=heads, length=length, d=d, e=e, train=rng.random() < 0.5,
                state=rng.random() < 0.4, ragged=rng.random() < 0.4, dtype=dtype)


# ----------------------------------------------------------------- inputs


class _Maker:
    def __init__(self, seed, dtype):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.dtype = dtype

    def randn(self, *shape, scale=1.0, dtype=None):
        t = torch.randn(*shape, generator=self.gen, device="cuda")
        return (t * scale).to(dtype or self.dtype)

    def silu(self, *shape):
        t = torch.randn(*shape, generator=self.gen, device="cuda")
        return (t * torch.sigmoid(t)).to(self.dtype)

    def int8_rows(self, rows, width):
        t = torch.randn(rows, width, generator=self.gen, device="cuda")
        return (t * 32).round().clamp(-127, 127).to(torch.int8)


def _inputs(case, seed):
    m = _Maker(seed, DTYPES[case["dtype"]])
    kind = case["kind"]
    if kind in ("norm", "norm8"):
        rows, width = case["rows"], case["width"]
        x = {"input": m.randn(rows, width), "weight": 1.0 + m.randn(width, scale=0.1, dtype=torch.float32)}
        if case["residual"]:
            x["residual"] = m.randn(rows, width, scale=2.0)
        if kind == "norm":
            x["dout"] = m.randn(rows, width)
            if case["residual"]:
                x["dsum"] = m.randn(rows, width)
        return x
    if kind == "int8":
        rows, k, n = case["rows"], case["k"], case["n"]
        x = {"weight": m.int8_rows(n, k), "weight_scale": (0.5 + torch.rand(n, generator=m.gen, device="cuda")) / 32 / k**0.5}
        if case["quantize"]:
            x["input"] = m.randn(rows, k)
        else:
            x["input"] = m.int8_rows(rows, k)
            x["input_scale"] = (0.5 + torch.rand(rows, generator=m.gen, device="cuda")) / 32
        if case["bias"]:
            x["bias"] = m.randn(n, dtype=torch.float32)
        return x
    b, h, d, e = case["batch"], case["heads"], case["d"], case["e"]
    # exp(log_decay) from exp(-1/2) to exp(-1/256)
    expo = torch.linspace(1.0, 8.0, h, device="cuda") if h > 1 else torch.full((1,), 4.0, device="cuda")
    x = {"log_decay": -torch.exp2(-expo)}
    if kind == "step":
        x |= {"query": m.silu(b, h, d), "key": m.silu(b, h, d), "value": m.randn(b, h, e),
              "state": m.randn(b, h, d, e, scale=4.0, dtype=torch.float32)}
        return x
    n = case["length"]
    x["query"], x["key"] = (m.silu(b, n, h, d).transpose(1, 2) for _ in range(2))
    x["value"] = m.randn(b, n, h, e).transpose(1, 2)
    if case["state"]:
        x["initial_state"] = m.randn(b, h, d, e, dtype=torch.float32)
    if case["ragged"]:
        lengths = torch.randint(0, n + 1, (b,), generator=m.gen, device="cuda", dtype=torch.int32)
        lengths[0] = n
        if b > 1:
            lengths[1] = 0
        x["lengths"] = lengths
    if case["train"]:
        x["dout"] = m.randn(b, n, h, e).transpose(1, 2)
        if case["state"]:
            x["dstate"] = m.randn(b, h, d, e, dtype=torch.float32)
    return x


def _leaf_names(case):
    if case["kind"] == "norm":
        return ["input", "weight"] + (["residual"] if case["residual"] else [])
    if case["kind"] == "linear" and case["train"]:
        return ["query", "key", "value"] + (["initial_state"] if case["state"] else [])
    return []


def prepare(case, seed):
    x = _inputs(case, seed)
    for name in _leaf_names(case):
        x[name].requires_grad_(True)
    return case, x


# ----------------------------------------------------------------- plain forms


def _plain_norm(x):
    h = x["input"]
    if "residual" in x:
        h = (h.float() + x["residual"].float()).to(h.dtype)
    hf = h.float()
    rstd = torch.rsqrt((hf * hf).mean(-1, keepdim=True) + EPS)
    return h, hf * rstd, rstd


def _plain_norm_step(x):
    h, n, rstd = _plain_norm(x)
    dt = h.dtype
    y = (n * x["weight"]).to(dt)
    dy = x["dout"].float()
    g = dy * x["weight"]
    dx = rstd * (g - n * (g * n).mean(-1, keepdim=True))
    dw = (dy * n).sum(0)
    if "residual" not in x:
        return y, dx.to(dt), dw
    dx = (dx + x["dsum"].float()).to(dt)
    return y, h, dx, dw, dx.clone()


def _plain_quantize(y):
    amax = y.abs().amax(-1)
    scales = amax / 127.0
    q = torch.where(scales[:, None] > 0, torch.round(y / scales[:, None]), 0.0)
    return q.to(torch.int8), scales


def _plain_norm8(x):
    h, n, _ = _plain_norm(x)
    q, scales = _plain_quantize(n * x["weight"])
    values = torch.mul(q, scales[:, None], out=torch.empty_like(h))
    return (values, scales, h) if "residual" in x else (values, scales)


def _plain_int8(case, x):
    q, scales = _plain_quantize(x["input"].float()) if case["quantize"] else (x["input"], x["input_scale"])
    y = (q.float() @ x["weight"].float().t()) * scales[:, None] * x["weight_scale"]
    if case["bias"]:
        y = y + x["bias"]
    return y.to(DTYPES[case["dtype"]])


def _powers(log_decay, n):
    """exp(log_decay * n) as float32, (H, *n.shape)."""

    ld = log_decay.double().view(-1, *[1] * n.dim())
    return torch.exp(ld * n.double()).float()


def _walk(a, b, c, log_decay):
    """out_i = sum_{j <= i} exp(log_decay (i - j)) (a_i . b_j) c_j, (B, H, L, .) float32, in chunks."""

    length = a.shape[2]
    pad = -length % CHUNK
    chunks = (length + pad) // CHUNK
    a, b, c = (torch.nn.functional.pad(t, (0, 0, 0, pad)).unflatten(2, (chunks, CHUNK)) for t in (a, b, c))
    i = torch.arange(CHUNK, device=a.device)
    lag = i[:, None] - i[None, :]
    inside = torch.where(lag >= 0, _powers(log_decay, lag.clamp(min=0)), 0.0)
    out = ((a @ b.transpose(-1, -2)) * inside[:, None]) @ c
    update = (b * _powers(log_decay, CHUNK - 1 - i)[:, None, :, None]).transpose(-1, -2) @ c
    n = torch.arange(chunks, device=a.device)
    lag = (n[:, None] - n[None, :] - 1) * CHUNK
    between = torch.where(lag >= 0, _powers(log_decay, lag.clamp(min=0)), 0.0)
    state = (between @ update.flatten(-2)).view(update.shape)
    out = out + (a @ state) * _powers(log_decay, i + 1)[:, None, :, None]
    return out.flatten(2, 3)[:, :, :length]


def _plain_linear(case, x):
    ld, n = x["log_decay"], case["length"]
    q, k, v = (x[name].float() for name in ("query", "key", "value"))
    scale = case["d"] ** -0.5
    dt = DTYPES[case["dtype"]]
    t = torch.arange(n, device=q.device)
    lengths = x["lengths"].long() if case["ragged"] else torch.full((case["batch"],), n, device=q.device)
    keep = (t < lengths[:, None])[:, None, :, None]  # (B, 1, L, 1)
    # exp(log_decay (length - 1 - t)): (B, H, L, 1)
    to_end = torch.where(keep, _powers(ld, (lengths[:, None] - 1 - t).clamp(min=0)).transpose(0, 1)[..., None], 0.0)
    from_start = _powers(ld, t + 1)[:, :, None]  # (H, L, 1)
    whole = _powers(ld, lengths).t()[:, :, None, None]
    k, v = k * keep, v * keep
    out = _walk(q, k, v, ld)
    if case["state"]:
        out = out + (q * from_start) @ x["initial_state"]
    out = (scale * out * keep).to(dt)
    outs = [out]
    if case["state"]:
        outs.append(whole * x["initial_state"] + (k * to_end).transpose(-1, -2) @ v)
    if not case["train"]:
        return tuple(outs)
    do = x["dout"].float() * keep
    dq = scale * _walk(do, v, k, ld)
    qf, kf, vf, dof = (a.flip(2) for a in (q, k, v, do))
    dk = scale * _walk(vf, dof, qf, ld).flip(2)
    dv = scale * _walk(kf, qf, dof, ld).flip(2)
    if case["state"]:
        s0, ds = x["initial_state"], x["dstate"]
        dq = dq + scale * (do * from_start) @ s0.transpose(-1, -2)
        dk = dk + (v * to_end) @ ds.transpose(-1, -2)
        dv = dv + (k * to_end) @ ds
        outs += [(dq * keep).to(dt), (dk * keep).to(dt), (dv * keep).to(dt)]
        outs.append(scale * (q * from_start).transpose(-1, -2) @ do + whole * ds)
    else:
        outs += [(dq * keep).to(dt), (dk * keep).to(dt), (dv * keep).to(dt)]
    return tuple(outs)


def _plain_step(case, x):
    q, k, v = (x[name].float() for name in ("query", "key", "value"))
    state = x["state"]
    state.mul_(torch.exp(x["log_decay"])[:, None, None]).add_(k[..., None] * v[..., None, :])
    out = (q[..., None, :] @ state)[..., 0, :] * case["d"] ** -0.5
    return out.to(DTYPES[case["dtype"]]), state


# ----------------------------------------------------------------- the framework's calls


def _own(case, x):
    import oops_amd

    kind = case["kind"]
    if kind == "norm":
        width = case["width"]
        if not case["residual"]:
            y = oops_amd.rms_norm(x["input"], width, x["weight"], EPS)
            return (y.detach(), *torch.autograd.grad(y, (x["input"], x["weight"]), x["dout"]))
        y, h = oops_amd.rms_norm(x["input"], width, x["weight"], EPS, residual=x["residual"])
        leaves = (x["input"], x["weight"], x["residual"])
        return (y.detach(), h.detach(), *torch.autograd.grad((y, h), leaves, (x["dout"], x["dsum"])))
    if kind == "norm8":
        q, scales, *h = oops_amd.rms_norm_int8(x["input"], case["width"], x["weight"], EPS, residual=x.get("residual"))
        return (torch.mul(q, scales[:, None], out=torch.empty_like(x["input"])), scales, *h)
    if kind == "int8":
        q, scales = oops_amd.quantize_int8(x["input"]) if case["quantize"] else (x["input"], x["input_scale"])
        return oops_amd.int8_linear(q, scales, x["weight"], x["weight_scale"], x.get("bias"), dtype=DTYPES[case["dtype"]])
    if kind == "step":
        out = oops_amd.linear_attention_step(x["query"], x["key"], x["value"], x["log_decay"], x["state"])
        return out, x["state"]
    res = oops_amd.linear_attention(x["query"], x["key"], x["value"], x["log_decay"], x.get("initial_state"),
                                    x.get("lengths"), return_state=case["state"])
    outs = res if case["state"] else (res,)
    if not case["train"]:
        return outs
    grads = (x["dout"], x["dstate"]) if case["state"] else (x["dout"],)
    leaves = [x[name] for name in _leaf_names(case)]
    return (*(t.detach() for t in outs), *torch.autograd.grad(outs, leaves, grads))


def run(state):
    case, x = state
    if own:
        return _own(case, x)
    with torch.no_grad():
        kind = case["kind"]
        if kind == "norm":
            return _plain_norm_step(x)
        if kind == "norm8":
            return _plain_norm8(x)
        if kind == "int8":
            return _plain_int8(case, x)
        return _plain_step(case, x) if kind == "step" else _plain_linear(case, x)


# ----------------------------------------------------------------- what a pass cannot do without


def work(case):
    kind = case["kind"]
    el = 4 if case["dtype"] == "f32" else 2
    if kind in ("norm", "norm8"):
        cells, res = case["rows"] * case["width"], int(case["residual"])
        if kind == "norm8":
            # input (residual) read, values (sum) written, and the values read as what they stand for
            return {"bytes": cells * (el * (1 + 2 * res) + 2 + el) + 8 * case["rows"], "flops": 8 * cells}
        # forward: input (residual) read, y (sum) written; backward: the summed rows, dy (dsum) read, dx written
        return {"bytes": cells * el * (2 + 2 * res + 3 + res), "flops": 20 * cells}
    if kind == "int8":
        rows, k, n = case["rows"], case["k"], case["n"]
        nbytes = rows * k + n * k + rows * n * el + 4 * (rows + n)
        if case["quantize"]:
            nbytes += rows * k * (el + 1)
        return {"bytes": nbytes, "flops": 2 * rows * n * k}
    b, h, d, e = case["batch"], case["heads"], case["d"], case["e"]
    if kind == "step":
        return {"bytes": b * h * (8 * d * e + el * (2 * d + 2 * e)), "flops": 6 * b * h * d * e}
    tokens = b * h * case["length"]
    states = 8 * b * h * d * e if case["state"] else 0
    # a token: the update of the state and its reading (the recurrence is the least work there is)
    nbytes, flops = tokens * el * (2 * d + 2 * e) + states, 4 * tokens * d * e
    if case["train"]:
        # q, k, v, do read, dq, dk, dv written; two states walked, dq, dk, dv read from them
        nbytes += tokens * el * (4 * d + 3 * e) + states
        flops += 10 * tokens * d * e
    return {"bytes": nbytes, "flops": flops}


# ----------------------------------------------------------------- float64 definition


def _exact_norm(case, x):
    """Rows in float64; the sum of input and residual is rounded to the input's type, as the operator defines."""

    h = x["input"].double()
    if case["residual"]:
        h = (h + x["residual"].double()).to(x["input"].dtype).double()
    rms = ((h**2).sum(-1, keepdim=True) / case["width"] + EPS) ** 0.5
    return h, rms


def _exact_recurrence(case, x):
    """The recurrence token by token: outputs, last state and, for training, every gradient."""

    b, h, d, e, n = (case[name] for name in ("batch", "heads", "d", "e", "length"))
    q, k, v = (x[name].double().permute(2, 0, 1, 3).contiguous() for name in ("query", "key", "value"))
    decay = x["log_decay"].double().exp()[None, :, None, None].expand(b, h, 1, 1)
    scale = d**-0.5
    s = x["initial_state"].double().clone() if case["state"] else q.new_zeros(b, h, d, e)
    live = None
    if case["ragged"]:
        live = (torch.arange(n, device=q.device)[:, None] < x["lengths"][None]).double()[:, :, None, None, None]
    ragged = case["ragged"]
    out = q.new_zeros(n, b, h, e)
    do = dq = None
    if case["train"]:
        do = x["dout"].double().permute(2, 0, 1, 3).contiguous()
        dq = torch.zeros_like(q)
    for t in range(n):
        if ragged:
            on = live[t]
            s = s * (on * decay + (1 - on)) + on * k[t][..., :, None] * v[t][..., None, :]
            out[t] = scale * on[..., 0] * (q[t][..., None, :] @ s)[..., 0, :]
        else:
            s.mul_(decay).addcmul_(k[t][..., :, None], v[t][..., None, :])
            out[t] = scale * (q[t][..., None, :] @ s)[..., 0, :]
        if dq is not None:
            dq[t] = scale * (s @ do[t][..., :, None])[..., 0]
            if ragged:
                dq[t] *= live[t][..., 0]
    back = lambda a: a.permute(1, 2, 0, 3)  # noqa: E731
    outs = [back(out)] + ([s] if case["state"] else [])
    if not case["train"]:
        return tuple(outs)
    r = x["dstate"].double().clone() if case["state"] else torch.zeros_like(s)
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    for t in reversed(range(n)):
        # r: the gradient of the state behind token t
        on = live[t] if ragged else 1.0
        r = r + on * scale * q[t][..., :, None] * do[t][..., None, :]
        dk[t] = (r @ v[t][..., :, None])[..., 0] * (on[..., 0] if ragged else 1.0)
        dv[t] = (k[t][..., None, :] @ r)[..., 0, :] * (on[..., 0] if ragged else 1.0)
        r = r * (on * decay + (1 - on)) if ragged else r * decay
    outs += [back(dq), back(dk), back(dv)] + ([r] if case["state"] else [])
    return tuple(outs)


def exact(case, seed):
    """``run``'s outputs by the definition, in float64."""

    x = _inputs(case, seed)
    kind = case["kind"]
    if kind == "norm":
        h, rms = _exact_norm(case, x)
        n, w, dy = h / rms, x["weight"].double(), x["dout"].double()
        dn = dy * w
        dh = (dn - n * ((dn * n).sum(-1, keepdim=True) / case["width"])) / rms
        if not case["residual"]:
            return n * w, dh, (dy * n).sum(0)
        dh = dh + x["dsum"].double()
        return n * w, h, dh, (dy * n).sum(0), dh
    if kind == "norm8":
        h, rms = _exact_norm(case, x)
        y = h / rms * x["weight"].double()
        top = y.abs().amax(-1, keepdim=True)
        values = torch.round(y * 127 / top) * (top / 127)
        return (values, top[:, 0] / 127, h) if case["residual"] else (values, top[:, 0] / 127)
    if kind == "int8":
        a = x["input"].double()
        if case["quantize"]:
            top = a.abs().amax(-1, keepdim=True)
            a = torch.round(a * 127 / top) * (top / 127)
        else:
            a = a * x["input_scale"].double()[:, None]
        y = a @ (x["weight"].double() * x["weight_scale"].double()[:, None]).t()
        return y + x["bias"].double() if case["bias"] else y
    if kind == "linear":
        return _exact_recurrence(case, x)
    s = x["state"].double() * x["log_decay"].double().exp()[:, None, None]
    s = s + x["key"].double()[..., :, None] * x["value"].double()[..., None, :]
    return (x["query"].double()[..., None, :] @ s)[..., 0, :] * case["d"] ** -0.5, s
