"""The performance cases of the operators of a token network's training step: the first layer
and what the step keeps between its forward and backward passes.

A case is a dict of plain values.  Its "path" names the entry points a pass goes through:

  lookup  embed_fprop: rows of a table by token, scaled
  egrad   embed_grad: the table's gradient, tokens sorted
  act     act8_fprop, then act8_bprop: an activation whose input is kept in 8 bits, and its
          backward pass from what was kept
  keep    act8_keep, then act8_expand: a tensor kept in 8 bits and expanded again
  wgrad   act8_grad: a linear (1x1) layer's weight gradient from its kept input

The 8-bit form: each group of 32 channels of a row (the last one may be shorter; the two halves
of a gated row are grouped apart) has one exponent byte b, and a value stands for
code * 2^(b - 127), -127 <= code <= 127.  With E and m the exponent and mantissa fields of the
group's largest magnitude as fp32, b = E - 6, one more where m >= 0x7F0000 (the code would round
to 128), held to 1 .. 248; codes round to nearest even.  A group that holds an infinity or a
NaN has b = 255, codes 0, and stands for NaN.

Fields: "type" and "out" are f32 or bf16; tokens, vocab, rows, c (channels), k (output channels).
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}
GROUP = 32


def listed():
    return [
        # a serving step of eight sequences: latency
        {"name": "lookup_step", "path": "lookup", "tokens": 8, "vocab": 65536, "c": 2048, "type": "bf16",
         "out": "bf16", "ids": "i64"},
        # a training batch from the fp32 master table to bf16 rows
        {"name": "lookup_batch", "path": "lookup", "tokens": 65536, "vocab": 65536, "c": 2048, "type": "f32",
         "out": "bf16", "ids": "i64"},
        # a short batch on a small network: the gradient's launches and its zero rows
        {"name": "egrad_short", "path": "egrad", "tokens": 1024, "vocab": 16384, "c": 512, "type": "f32",
         "out": "f32", "ids": "i64"},
        # a training batch: frequent tokens come thousands of times
        {"name": "egrad_batch", "path": "egrad", "tokens": 65536, "vocab": 65536, "c": 2048, "type": "bf16",
         "out": "f32", "ids": "i64"},
        # odd sizes: rows at every alignment
        {"name": "egrad_ragged", "path": "egrad", "tokens": 20011, "vocab": 50021, "c": 1001, "type": "f32",
         "out": "f32", "ids": "i32"},
        # four tokens through a gated activation: latency
        {"name": "act_token", "path": "act", "rows": 4, "c": 4096, "act": "silu", "gated": True, "type": "bf16"},
        # a training batch's gated activation: the largest traffic
        {"name": "act_gated", "path": "act", "rows": 16384, "c": 8192, "act": "silu", "gated": True, "type": "bf16"},
        # the input of an expanding pointwise convolution layer, 64 images of 28x28
        {"name": "keep_layer", "path": "keep", "rows": 64 * 28 * 28, "c": 128, "type": "f32"},
        # odd sizes: the last group of a row is short
        {"name": "keep_ragged", "path": "keep", "rows": 8191, "c": 1003, "type": "bf16"},
        # a short batch's weight gradient: few output tiles, the rows split
        {"name": "wgrad_short", "path": "wgrad", "rows": 512, "c": 1024, "k": 1024, "type": "bf16", "out": "f32"},
        # a training batch's: the largest product
        {"name": "wgrad_batch", "path": "wgrad", "rows": 16384, "c": 4096, "k": 4096, "type": "bf16", "out": "f32"},
        # the expanding pointwise convolution layer's, in fp32: a long sum into a small filter
        {"name": "wgrad_layer", "path": "wgrad", "rows": 64 * 28 * 28, "c": 128, "k": 512, "type": "f32",
         "out": "f32"},
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
    path = rng.choice(["lookup", "egrad", "act", "keep", "wgrad"])
    kind = rng.choice(["f32", "bf16"])
    if path in ("lookup", "egrad"):
        c = _channels(rng, 48, 4096)
        tokens = min(_log(rng, 1, 65536), (1 << 27) // c)
        vocab = min(_log(rng, 64, 131072), (1 << 27) // c)
        return {"path": path, "tokens": tokens, "vocab": vocab, "c": c, "type": kind,
                "out": rng.choice(["f32", "bf16"]), "ids": rng.choice(["i32", "i64"])}
    if path == "act":
        gated = rng.random() < 0.5
        c = _channels(rng, 32, 8192)
        rows = min(_log(rng, 1, 131072), (1 << 26) // c)
        return {"path": path, "rows": rows, "c": c, "act": rng.choice(["relu", "silu", "gelu"]), "gated": gated,
                "type": kind}
    if path == "keep":
        c = _channels(rng, 32, 8192)
        return {"path": path, "rows": min(_log(rng, 1, 131072), (1 << 26) // c), "c": c, "type": kind}
    c, k = _channels(rng, 32, 4096), _channels(rng, 32, 4096)
    rows = min(_log(rng, 1, 65536), (1 << 36) // (c * k))
    return {"path": path, "rows": rows, "c": c, "k": k, "type": kind,
            "out": rng.choice(["f32", "bf16"]) if kind == "bf16" else "f32"}


# ---- inputs -----------------------------------------------------------------------------------

def _normal(g, shape, spread=1.0):
    return torch.randn(shape, generator=g, device="cuda") * spread


def _activations(g, rows, c):
    """Values before an activation: channels of different scales, a few large values, some rows
    of zeros (padded positions)."""
    x = _normal(g, (rows, c)) * torch.exp(0.5 * _normal(g, (c,)))
    x = torch.where(torch.rand((rows, c), generator=g, device="cuda") < 0.001, x * 16, x)
    return x * (torch.rand((rows, 1), generator=g, device="cuda") > 0.02)


def _gradients(g, rows, c):
    return _normal(g, (rows, c), 1e-3) * (torch.rand((rows, 1), generator=g, device="cuda") > 0.02)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 2 + 1)
    s = dict(case)
    kind = TYPES[case["type"]]
    if case["path"] in ("lookup", "egrad"):
        tokens, vocab, c = case["tokens"], case["vocab"], case["c"]
        # token frequencies fall as 1 / rank; -1 is a position without a token
        u = torch.rand((tokens,), generator=g, device="cuda", dtype=torch.float64)
        ids = (torch.exp(u * math.log(vocab + 1)) - 1).long().clamp(0, vocab - 1)
        ids = torch.where(torch.rand((tokens,), generator=g, device="cuda") < 0.02, -1, ids)
        s["idx"] = ids.to(torch.int32 if case["ids"] == "i32" else torch.int64)
        s["scale"] = math.sqrt(c)
        if case["path"] == "lookup":
            s["table"] = _normal(g, (vocab, c), 0.02).to(kind)
        else:
            s["dy"] = _gradients(g, tokens, c).to(kind)
    elif case["path"] == "act":
        s["x"] = _activations(g, case["rows"], case["c"] * (2 if case["gated"] else 1)).to(kind)
        s["dy"] = _gradients(g, case["rows"], case["c"]).to(kind)
    elif case["path"] == "keep":
        s["x"] = _activations(g, case["rows"], case["c"]).to(kind)
    else:
        s["codes"], s["scales"] = _keep(_activations(g, case["rows"], case["c"]), 1)
        s["dy"] = _gradients(g, case["rows"], case["k"]).to(kind)
    return s


# ---- the plain forms ----------------------------------------------------------------------------

def _grouped(x, halves):
    """(rows, halves, groups, 32) of a row-major x, short groups filled with zeros."""
    rows, c = x.shape[0], x.shape[1] // halves
    pad = -c % GROUP
    x = x.reshape(rows, halves, c)
    if pad:
        x = torch.cat([x, x.new_zeros((rows, halves, pad))], 2)
    return x.reshape(rows, halves, -1, GROUP)


def _keep(x, halves):
    """int8 codes, shaped as x, and exponent bytes (rows, halves * groups)."""
    rows, width = x.shape
    x = _grouped(x.float(), halves)
    top = x.abs().amax(3).view(torch.int32)
    byte = ((top >> 23) - 6 + ((top & 0x7FFFFF) >= 0x7F0000).int()).clamp(1, 248)
    inverse = ((254 - byte) << 23).view(torch.float32)
    bad = ~torch.isfinite(x).all(3)
    codes = torch.where(bad[..., None], torch.zeros_like(x), torch.round(x * inverse[..., None]).clamp(-127, 127))
    byte = torch.where(bad, torch.full_like(byte, 255), byte)
    codes = codes.reshape(rows, halves, -1)[:, :, : width // halves].reshape(rows, width)
    return codes.to(torch.int8).contiguous(), byte.reshape(rows, -1).to(torch.uint8).contiguous()


def _expand(codes, scales, halves):
    rows, width = codes.shape
    each = (scales.int() << 23).view(torch.float32).reshape(rows, halves, -1, 1)
    x = _grouped(codes.float(), halves) * each
    return x.reshape(rows, halves, -1)[:, :, : width // halves].reshape(rows, width)


def _act(x, act):
    if act == "relu":
        return torch.where(x < 0, torch.zeros_like(x), x)
    if act == "silu":
        return x / (1 + torch.exp(-x))
    return 0.5 * x * torch.erfc(x * -math.sqrt(0.5))


def _slope(x, act):
    if act == "relu":
        return torch.where(x > 0, torch.ones_like(x), torch.where(x <= 0, torch.zeros_like(x), x))
    if act == "silu":
        s = 1 / (1 + torch.exp(-x))
        return s * (1 + x * (1 - s))
    return 0.5 * torch.erfc(x * -math.sqrt(0.5)) + x * torch.exp(-0.5 * x * x) * (1 / math.sqrt(2 * math.pi))


def _plain(s):
    path, kind = s["path"], TYPES[s["type"]]
    if path == "lookup":
        ids = s["idx"].long()
        there = (ids >= 0) & (ids < s["vocab"])
        y = s["table"][torch.where(there, ids, 0)].float() * s["scale"]
        return torch.where(there[:, None], y, torch.zeros_like(y)).to(TYPES[s["out"]])
    if path == "egrad":
        ids = s["idx"].long()
        there = (ids >= 0) & (ids < s["vocab"])
        sums = torch.zeros((s["vocab"] + 1, s["c"]), device=ids.device)
        sums.index_add_(0, torch.where(there, ids, s["vocab"]), s["dy"].float())
        return (sums[: s["vocab"]] * s["scale"]).to(TYPES[s["out"]])
    if path == "act":
        halves = 2 if s["gated"] else 1
        x, dy, c = s["x"].float(), s["dy"].float(), s["c"]
        y = _act(x[:, :c], s["act"])
        back = _expand(*_keep(x, halves), halves)
        if not s["gated"]:
            return y.to(kind), (dy * _slope(back, s["act"])).to(kind)
        gate, up = back[:, :c], back[:, c:]
        dx = torch.cat([dy * up * _slope(gate, s["act"]), dy * _act(gate, s["act"])], 1)
        return (y * x[:, c:]).to(kind), dx.to(kind)
    if path == "keep":
        return _expand(*_keep(s["x"], 1), 1).to(kind)
    return torch.matmul(s["dy"].float().t(), _expand(s["codes"], s["scales"], 1)).to(TYPES[s["out"]])


def run(state):
    if not own:
        return _plain(state)
    import my_own_cnn_amd as M

    path = state["path"]
    if path == "lookup":
        return M.embed_fprop(state["table"], state["idx"], scale=state["scale"], dtype=TYPES[state["out"]])
    if path == "egrad":
        return M.embed_grad(state["dy"], state["idx"], state["vocab"], scale=state["scale"], dtype=TYPES[state["out"]])
    if path == "act":
        y, kept = M.act8_fprop(state["x"], state["act"], gated=state["gated"])
        return y, M.act8_bprop(state["dy"], kept)
    if path == "keep":
        return M.act8_expand(M.act8_keep(state["x"]), dtype=TYPES[state["type"]])
    return M.act8_grad(state["dy"], M.Act8(state["codes"], state["scales"]), dtype=TYPES[state["out"]])


# ---- what a pass cannot do without ----------------------------------------------------------------

def work(case):
    path, size = case["path"], SIZE[case["type"]]
    if path == "lookup":
        tokens, c = case["tokens"], case["c"]
        # the rows that at least one token names, on average over the draws of prepare()
        rank = np.arange(case["vocab"], dtype=np.float64)
        share = 0.98 * np.log1p(1 / (rank + 1)) / math.log(case["vocab"] + 1)
        rows = int(-np.expm1(tokens * np.log1p(-share)).sum())
        return {"bytes": rows * c * size + tokens * c * SIZE[case["out"]] + tokens * int(case["ids"][1:]) // 8,
                "flops": tokens * c}
    if path == "egrad":
        tokens, c = case["tokens"], case["c"]
        return {"bytes": tokens * c * size + case["vocab"] * c * SIZE[case["out"]] + tokens * int(case["ids"][1:]) // 8,
                "flops": tokens * c}
    rows, c = case["rows"], case["c"]
    kept = rows * (c + -(-c // GROUP))
    if path == "act":
        wide = 2 if case["gated"] else 1
        # x, y and the codes; dy, the codes and dx
        return {"bytes": 2 * (rows * c * (wide + 1) * size + wide * kept), "flops": 20 * rows * c * wide}
    if path == "keep":
        return {"bytes": 2 * (rows * c * size + kept), "flops": 4 * rows * c}
    k = case["k"]
    return {"bytes": rows * k * size + kept + k * c * SIZE[case["out"]], "flops": 2 * rows * k * c}


# ---- the definitions in 64 bits ---------------------------------------------------------------------

def _power(e):
    """2 to the integers of a tensor, as float64 (pow and ldexp may be a rounding off)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _stands_for(x, halves):
    """What the 8-bit form of x (float64) stands for, by its arithmetic definition."""
    rows, width = x.shape
    c = width // halves
    out = torch.empty_like(x)
    for half in range(halves):
        for g in range(0, c, GROUP):
            lo, hi = half * c + g, half * c + min(g + GROUP, c)
            part = x[:, lo:hi]
            top = part.abs().amax(1, keepdim=True)
            # the least power of two that leaves every code within 127 after rounding
            step = _power(torch.frexp(top)[1] - 7)
            step = torch.where(torch.round(top / step) > 127, 2 * step, step)
            step = torch.where(top > 0, step, torch.ones_like(step))
            out[:, lo:hi] = torch.round(part / step) * step
    return out


def exact(case, seed):
    s = prepare(case, seed)
    path = case["path"]
    if path == "lookup":
        table = torch.cat([s["table"].double() * s["scale"], torch.zeros((1, case["c"]), device="cuda").double()])
        return table[torch.where(s["idx"] < 0, case["vocab"], s["idx"].long())]
    if path == "egrad":
        # running sums along the sorted tokens, and their differences at the rows' ends
        ids, order = torch.sort(s["idx"].long())
        sums = torch.cumsum(s["dy"][order].double(), 0)
        sums = torch.cat([torch.zeros_like(sums[:1]), sums])
        rows = torch.arange(case["vocab"], device="cuda")
        return (sums[torch.searchsorted(ids, rows, right=True)] - sums[torch.searchsorted(ids, rows)]) * s["scale"]
    if path == "keep":
        return _stands_for(s["x"].double(), 1)
    if path == "wgrad":
        power = _power(s["scales"].int() - 127).repeat_interleave(GROUP, 1)[:, : case["c"]]
        return torch.matmul(s["dy"].double().t(), s["codes"].double() * power)
    c, halves = case["c"], 2 if case["gated"] else 1
    x, dy = s["x"].double(), s["dy"].double()

    def both(v):
        """The activation and its derivative."""
        if case["act"] == "relu":
            return v.clamp(min=0), (v > 0).double()
        if case["act"] == "silu":
            p = torch.sigmoid(v)
            return v * p, p + v * p * torch.sigmoid(-v)
        p = torch.special.ndtr(v)
        return v * p, p + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)

    y = both(x[:, :c])[0]
    back = _stands_for(x, halves)
    value, slope = both(back[:, :c])
    if halves == 1:
        return y, dy * slope
    return y * x[:, c:], torch.cat([dy * back[:, c:] * slope, dy * value], 1)
