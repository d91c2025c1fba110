"""The performance cases of the operators of a token network's layers in 8 bits: the norm with the
residual's addition (its backward pass among them), activations as 8-bit rows, int8 products with
a scale for each token and channel, and the same grouped by expert.

A case is a dict of plain values.  Its "path" names the entry points a pass goes through:

  norm     rms_row8, then row8_expand: the norm of a sum as 8-bit rows, and what they stand for
  train    rms_fprop, then rms_bprop: the norm of a sum and its gradients
  gate     act_row8, then row8_expand: an activation (gated: times its second half) as 8-bit rows
  linear   row8_linear: an int8 product, a bias and rows added to it
  experts  experts_plan, row8_experts, act_row8, row8_experts, experts_join: a layer of gated
           networks, each token through some of them

The 8-bit form of a row v: m = max(max |v|, 2^-110), scale = m / 127, codes round(v * 127 / m) to
nearest even.  What lies between two operators is a tensor of the type that the first one returns:
the sum of norm and train (rounded to the type, then normed) and the bf16 rows between the experts'
product and its activation.

Fields: "type" (inputs) and "out" are f32 or bf16; rows or tokens, c (channels), k (output
channels), hidden (channels between two experts' products), experts, slots (experts of a token).
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}
EPS = 1e-6
LEAST = 2.0 ** -110


def listed():
    return [
        # a serving step of four sequences: latency
        {"name": "norm_token", "path": "norm", "rows": 4, "c": 4096, "add": True, "type": "bf16"},
        # a long prompt batch: traffic
        {"name": "norm_batch", "path": "norm", "rows": 16384, "c": 4096, "add": True, "type": "bf16"},
        # a training batch's norm and its gradients
        {"name": "train_batch", "path": "train", "rows": 16384, "c": 2048, "add": True, "type": "bf16"},
        # odd sizes, fp32, no residual
        {"name": "train_ragged", "path": "train", "rows": 5003, "c": 1001, "add": False, "type": "f32"},
        # the gated activation of a long prompt batch: the largest traffic
        {"name": "gate_batch", "path": "gate", "rows": 16384, "c": 8192, "act": "silu", "gated": True, "type": "bf16"},
        # odd sizes: rows at every alignment
        {"name": "gate_ragged", "path": "gate", "rows": 4099, "c": 1003, "act": "gelu", "gated": False, "type": "f32"},
        # one token: the weights' traffic
        {"name": "linear_token", "path": "linear", "rows": 1, "c": 4096, "k": 4096, "bias": False, "add": True,
         "out": "bf16"},
        # a serving step of 64 sequences: the weights' traffic, more rows than one matrix tile
        {"name": "linear_step", "path": "linear", "rows": 64, "c": 4096, "k": 8192, "bias": False, "add": False,
         "out": "bf16"},
        # a long prompt batch: the largest product
        {"name": "linear_batch", "path": "linear", "rows": 16384, "c": 4096, "k": 8192, "bias": False, "add": False,
         "out": "bf16"},
        # odd sizes: rows at every alignment, edges in every direction
        {"name": "linear_ragged", "path": "linear", "rows": 1003, "c": 2051, "k": 1537, "bias": True, "add": False,
         "out": "f32"},
        # a serving step of eight sequences: few rows on few of the experts
        {"name": "experts_token", "path": "experts", "tokens": 8, "slots": 2, "experts": 64, "c": 2048, "hidden": 1024},
        # a prompt batch: every expert has rows, in ragged numbers
        {"name": "experts_batch", "path": "experts", "tokens": 8192, "slots": 2, "experts": 32, "c": 2048,
         "hidden": 2048},
    ]


# ---- drawn cases ----------------------------------------------------------------------------

def _log(rng, lo, hi):
    """An integer spread over [lo, hi] by its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _channels(rng, lo, hi):
    """A channel count: half of them multiples of 64, the rest anything."""
    c = _log(rng, lo, hi)
    return max(64, c // 64 * 64) if rng.random() < 0.5 else c


def draw(rng):
    path = rng.choice(["norm", "train", "gate", "linear", "experts"])
    if path in ("norm", "train"):
        c = _channels(rng, 48, 8192)
        return {"path": path, "rows": min(_log(rng, 1, 65536), (1 << 25) // c), "c": c, "add": rng.random() < 0.7,
                "type": rng.choice(["f32", "bf16"])}
    if path == "gate":
        c = _channels(rng, 48, 8192)
        return {"path": path, "rows": min(_log(rng, 1, 65536), (1 << 25) // c), "c": c,
                "act": rng.choice(["none", "relu", "silu", "gelu"]), "gated": rng.random() < 0.6,
                "type": rng.choice(["f32", "bf16"])}
    if path == "linear":
        c, k = _channels(rng, 48, 8192), _channels(rng, 48, 16384)
        return {"path": path, "rows": min(_log(rng, 1, 16384), (1 << 38) // (c * k)), "c": c, "k": k,
                "bias": rng.random() < 0.5, "add": rng.random() < 0.5, "out": rng.choice(["f32", "bf16"])}
    c, hidden = _channels(rng, 64, 4096), _channels(rng, 64, 2048)
    experts = min(_log(rng, 4, 128), (1 << 27) // (c * hidden))
    return {"path": path, "tokens": min(_log(rng, 1, 8192), (1 << 34) // (c * hidden)),
            "slots": rng.choice([1, 2, 4]), "experts": experts, "c": c, "hidden": hidden}


# ---- inputs -----------------------------------------------------------------------------------

def _normal(g, shape, spread=1.0):
    return torch.randn(shape, generator=g, device="cuda") * spread


def _activations(g, rows, c):
    """Rows of different sizes, channels of different scales, a few large values."""
    x = _normal(g, (rows, c)) * torch.exp(0.2 * _normal(g, (c,))) * torch.exp(0.3 * _normal(g, (rows, 1)))
    return torch.where(torch.rand((rows, c), generator=g, device="cuda") < 0.001, x * 4, x)


def _codes(g, shape, spread=40.0):
    return _normal(g, shape, spread).round().clamp(-127, 127).to(torch.int8)


def _scales(g, shape, size):
    return torch.exp(0.2 * _normal(g, shape)) * size


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 2 + 1)
    s, path = dict(case), case["path"]
    c = case["c"]
    if path in ("norm", "train"):
        rows, kind = case["rows"], TYPES[case["type"]]
        s["x"] = _activations(g, rows, c).to(kind)
        s["more"] = _activations(g, rows, c).to(kind) if case["add"] else None
        s["gain"] = torch.exp(0.2 * _normal(g, (c,))).to(kind)
        if path == "train":
            s["dy"] = _normal(g, (rows, c), 1e-3).to(kind)
            s["dsum"] = _normal(g, (rows, c), 1e-3).to(kind) if case["add"] else None
    elif path == "gate":
        s["x"] = _activations(g, case["rows"], c * (2 if case["gated"] else 1)).to(TYPES[case["type"]])
    elif path == "linear":
        rows, k = case["rows"], case["k"]
        s["codes"], s["scales"] = _codes(g, (rows, c)), _scales(g, (rows,), 0.02)
        s["w"], s["w_scales"] = _codes(g, (k, c)), _scales(g, (k,), 0.02 / math.sqrt(c) / 16)
        s["b"] = _normal(g, (k,)) if case["bias"] else None
        s["more"] = _normal(g, (rows, k)).to(TYPES[case["out"]]) if case["add"] else None
    else:
        tokens, slots, experts, hidden = case["tokens"], case["slots"], case["experts"], case["hidden"]
        s["codes"], s["scales"] = _codes(g, (tokens, c)), _scales(g, (tokens,), 0.02)
        s["w"], s["w_scales"] = _codes(g, (experts, 2 * hidden, c)), _scales(g, (experts, 2 * hidden), 0.03 / math.sqrt(c))
        s["v"], s["v_scales"] = _codes(g, (experts, c, hidden)), _scales(g, (experts, c), 0.03 / math.sqrt(hidden))
        # some experts are wanted more than others; padded positions (id -1) go to none
        score = _normal(g, (tokens, experts)) + 0.3 * _normal(g, (experts,))
        top, ids = torch.topk(score, slots, dim=1)
        pad = torch.rand((tokens, 1), generator=g, device="cuda") < 0.02
        s["ids"] = torch.where(pad, -1, ids).to(torch.int32)
        s["share"] = torch.softmax(top, 1)
        # of the plain form: the rows of the fullest expert, which a program that pads to it knows
        s["most"] = int(torch.bincount(s["ids"].flatten().long() + 1, minlength=experts + 1)[1:].max())
    return s


# ---- the plain forms ----------------------------------------------------------------------------

def _row8(v):
    """(codes as fp32, scales) of fp32 rows."""
    m = v.abs().amax(-1, keepdim=True).clamp(min=LEAST)
    return torch.round(v * (127 / m)), m / 127


def _act(x, act):
    if act == "relu":
        return torch.where(x < 0, torch.zeros_like(x), x)
    if act == "silu":
        return x / (1 + torch.exp(-x))
    if act == "gelu":
        return 0.5 * x * torch.erfc(x * -math.sqrt(0.5))
    return x


def _total(s):
    """The rows that are normed, in the type's values."""
    x = s["x"].float()
    return x if s["more"] is None else (x + s["more"].float()).to(s["x"].dtype).float()


def _grouped(x, w, experts, most, offsets):
    """Products of sorted fp32 rows x (n, c) with their expert's fp32 weights w (experts, k, c), each
    expert's rows padded to the fullest one's."""
    at = torch.arange(most, device=x.device)
    count = (offsets[1:] - offsets[:-1])[:, None]
    index = torch.where(at[None] < count, offsets[:-1, None] + at[None], x.shape[0])
    padded = torch.cat([x, x.new_zeros((1, x.shape[1]))])[index]
    y = torch.bmm(padded, w.transpose(1, 2).contiguous())
    out = x.new_zeros((x.shape[0] + 1, w.shape[1]))
    out[index.flatten()] = y.flatten(0, 1)
    return out[:-1]


def _plain(s):
    path = s["path"]
    if path == "norm":
        t = _total(s)
        r = torch.rsqrt((t * t).mean(1, keepdim=True) + EPS)
        codes, scales = _row8(t * r * s["gain"].float())
        values = (codes * scales).to(torch.bfloat16)
        return values if s["more"] is None else (values, t.to(s["x"].dtype))
    if path == "train":
        t, gain, dy, kind = _total(s), s["gain"].float(), s["dy"].float(), s["x"].dtype
        r = torch.rsqrt((t * t).mean(1, keepdim=True) + EPS)
        n = t * r
        d = dy * gain
        dx = r * (d - n * (d * n).mean(1, keepdim=True))
        dgain = (dy * n).sum(0)
        if s["more"] is None:
            return (n * gain).to(kind), dx.to(kind), dgain
        return (n * gain).to(kind), t.to(kind), (dx + s["dsum"].float()).to(kind), dgain
    if path == "gate":
        x, c = s["x"].float(), s["c"]
        v = _act(x[:, :c], s["act"]) * x[:, c:] if s["gated"] else _act(x, s["act"])
        codes, scales = _row8(v)
        return (codes * scales).to(torch.bfloat16)
    if path == "linear":
        y = torch.matmul(s["codes"].float(), s["w"].float().t()) * s["scales"][:, None] * s["w_scales"]
        if s["b"] is not None:
            y = y + s["b"]
        if s["more"] is not None:
            y = y + s["more"].float()
        return y.to(TYPES[s["out"]])
    ids, experts, slots, hidden = s["ids"].flatten().long(), s["experts"], s["slots"], s["hidden"]
    n = ids.numel()
    key = torch.where(ids < 0, experts, ids)
    order = torch.argsort(key, stable=True)
    expert = key[order]
    offsets = torch.searchsorted(expert, torch.arange(experts + 1, device=ids.device))
    there = expert < experts
    rows = torch.where(there, order // slots, -1)
    places = torch.empty_like(order)
    places[order] = torch.where(there, torch.arange(n, device=ids.device), -1)
    at = expert.clamp(max=experts - 1)
    x_rows = rows.clamp(min=0)
    h = _grouped(s["codes"].float()[x_rows], s["w"].float(), experts, s["most"], offsets)
    h = (h * s["scales"][x_rows, None] * s["w_scales"][at]).to(torch.bfloat16).float()
    codes, scales = _row8(_act(h[:, :hidden], "silu") * h[:, hidden:])
    y = _grouped(codes, s["v"].float(), experts, s["most"], offsets)
    y = (y * scales * s["v_scales"][at]).to(torch.bfloat16).float()
    y = torch.where((places >= 0)[:, None], y[places.clamp(min=0)], torch.zeros(1, device=ids.device))
    y = (y.reshape(-1, slots, s["c"]) * s["share"][:, :, None]).sum(1)
    return (y.to(torch.bfloat16), offsets.to(torch.int32), rows.to(torch.int32),
            places.reshape(-1, slots).to(torch.int32))


def run(state):
    if not own:
        return _plain(state)
    import my_own_cnn_amd as M

    s, path = state, state["path"]
    if path == "norm":
        if s["more"] is None:
            return M.row8_expand(M.rms_row8(s["x"], s["gain"], eps=EPS), dtype=torch.bfloat16)
        kept, total = M.rms_row8(s["x"], s["gain"], add=s["more"], eps=EPS)
        return M.row8_expand(kept, dtype=torch.bfloat16), total
    if path == "train":
        if s["more"] is None:
            y = M.rms_fprop(s["x"], s["gain"], eps=EPS)
            return (y, *M.rms_bprop(s["dy"], s["x"], s["gain"], eps=EPS))
        y, total = M.rms_fprop(s["x"], s["gain"], add=s["more"], eps=EPS)
        return (y, total, *M.rms_bprop(s["dy"], total, s["gain"], dsum=s["dsum"], eps=EPS))
    if path == "gate":
        return M.row8_expand(M.act_row8(s["x"], s["act"], gated=s["gated"]), dtype=torch.bfloat16)
    if path == "linear":
        return M.row8_linear(M.Row8(s["codes"], s["scales"]), M.Row8(s["w"], s["w_scales"]), bias=s["b"], add=s["more"],
                             dtype=TYPES[s["out"]])
    plan = M.experts_plan(s["ids"], s["experts"])
    h = M.row8_experts(M.Row8(s["codes"], s["scales"]), M.Row8(s["w"], s["w_scales"]), plan.offsets, rows=plan.rows,
                       dtype=torch.bfloat16)
    y = M.row8_experts(M.act_row8(h, "silu", gated=True), M.Row8(s["v"], s["v_scales"]), plan.offsets,
                       dtype=torch.bfloat16)
    return M.experts_join(y, plan.places, s["share"]), plan.offsets, plan.rows, plan.places


# ---- what a pass cannot do without ----------------------------------------------------------------

def work(case):
    path, c = case["path"], case["c"]
    if path in ("norm", "train", "gate"):
        rows, size = case["rows"], SIZE[case["type"]]
        if path == "gate":
            wide = 2 if case["gated"] else 1
            # x and the codes; the codes and the values
            return {"bytes": rows * (c * (wide * size + 2 + 2) + 8), "flops": 12 * rows * c * wide}
        add = 2 if case["add"] else 0
        if path == "norm":
            # x, the sum and the codes; the codes and the values
            return {"bytes": rows * (c * (size * (1 + add) + 2 + 2) + 8) + c * size, "flops": 8 * rows * c}
        # x, y and the sum; dy, the sum and its gradients
        return {"bytes": rows * c * size * (2 + add + 3 + add // 2) + 2 * c * size + 4 * c, "flops": 14 * rows * c}
    if path == "linear":
        rows, k, size = case["rows"], case["k"], SIZE[case["out"]]
        return {"bytes": rows * c + k * c + rows * k * size * (2 if case["add"] else 1) + 4 * (rows + k),
                "flops": 2 * rows * c * k}
    tokens, slots, experts, hidden = case["tokens"], case["slots"], case["experts"], case["hidden"]
    n = tokens * slots
    # the experts that at least one token names, were they drawn evenly
    named = experts * -math.expm1(tokens * math.log1p(-min(slots / experts, 1 - 1e-9)))
    return {"bytes": int(named) * (3 * hidden * c + 4 * (2 * hidden + c)) + tokens * (c + 4) + n * (2 * 4 * hidden + hidden)
            + n * (hidden + 2 * 2 * c) + tokens * c * 2 + n * 16, "flops": 2 * n * 3 * hidden * c}


# ---- the definitions in 64 bits ---------------------------------------------------------------------

def _stands_for(v):
    """What float64 rows stand for once they are 8-bit rows."""
    step = torch.maximum(v.abs().max(-1).values, torch.tensor(LEAST, device=v.device).double())[..., None] / 127
    return torch.round(v / step) * step


def _activated(x, act, gated):
    c = x.shape[1] // 2 if gated else x.shape[1]
    gate = x[:, :c]
    if act == "relu":
        gate = gate.clamp(min=0)
    elif act == "silu":
        gate = gate * torch.sigmoid(gate)
    elif act == "gelu":
        gate = gate * torch.special.ndtr(gate)
    return gate * x[:, c:] if gated else gate


def exact(case, seed):
    s = prepare(case, seed)
    path, c = case["path"], case["c"]
    if path in ("norm", "train"):
        kind = s["x"].dtype
        t = s["x"].double()
        if case["add"]:
            t = (t + s["more"].double()).to(kind).double()
        spread = torch.sqrt(t.square().sum(1) / c + EPS)[:, None]
        n, gain = t / spread, s["gain"].double()
        if path == "norm":
            values = _stands_for(n * gain)
            return (values, t) if case["add"] else values
        dn = s["dy"].double() * gain
        # the part of dn along n has no way through the norm
        dx = (dn - n * ((dn * n).sum(1) / c)[:, None]) / spread
        dgain = torch.einsum("rc,rc->c", s["dy"].double(), n)
        return (n * gain, t, dx + s["dsum"].double(), dgain) if case["add"] else (n * gain, dx, dgain)
    if path == "gate":
        return _stands_for(_activated(s["x"].double(), case["act"], case["gated"]))
    if path == "linear":
        y = (s["codes"].double() * s["scales"].double()[:, None]) @ (s["w"].double() * s["w_scales"].double()[:, None]).t()
        y = y if s["b"] is None else y + s["b"].double()
        return y if s["more"] is None else y + s["more"].double()
    x = s["codes"].double() * s["scales"].double()[:, None]
    y = torch.zeros((case["tokens"], c), dtype=torch.float64, device=x.device)
    for e in range(case["experts"]):
        token, slot = torch.nonzero(s["ids"] == e, as_tuple=True)
        if token.numel():
            w, v = s["w"][e].double() * s["w_scales"][e].double()[:, None], s["v"][e].double() * s["v_scales"][e].double()[:, None]
            h = (x[token] @ w.t()).to(torch.bfloat16).double()
            h = (_stands_for(_activated(h, "silu", True)) @ v.t()).to(torch.bfloat16).double()
            y[token] += h * s["share"][token, slot].double()[:, None]
    return y, None, None, None
