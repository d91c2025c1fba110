"""Layers on 8-bit rows on the GPU (miq_rms_*, miq_act_row8, miq_row8_*, miq_experts_*).

What the definitions give exactly is compared exactly: sums of integer products, codes of given values,
sorted pairs, and every fp32 operation after them in its order (numpy rounds as fp32 does).  With
u = 2^-24 (half a unit of fp32) the rest is held to:
  - a sum of c squares in a tree of runs: at most c / 1024 + 60 additions one after another, so
    (c / 1024 + 60) u of it, half of that of its root, and 8 u for the operations around it;
  - an activation: (16 + 4 v^2) u of its value (exp and erfc are good to a few units, gelu's argument is
    rounded, which moves erfc by v^2 u in relative terms);
  - a code: half a step, and 127 times the relative errors of the value, of the row's largest and of 3
    operations;
  - a gradient: the number of additions times u of the sum of magnitudes.
A bf16 result is the rounding of a value within these bounds, 2^-8 of it."""
import math

import numpy as np
import pytest
import torch

import my_own_cnn_amd as M

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24
INF, NAN = float("inf"), float("nan")
LEAST = np.float32(2.0 ** -110)


def _half_step(kind):
    return 2.0 ** -8 if kind == BF16 else U


def _values(seed, shape, kind, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * spread * torch.exp(torch.randn((1, shape[-1]), generator=g))
    return x.to(kind)


def _row8_32(v):
    """(codes, scales) of float32 rows, in float32 operations."""
    v = v.astype(np.float32)
    m = np.maximum(np.abs(v).max(-1, initial=0), LEAST).astype(np.float32)
    with np.errstate(invalid="ignore", over="ignore"):
        codes = np.rint(v * (np.float32(127) / m)[..., None])
        scales = m / np.float32(127)
    bad = ~np.isfinite(v).all(-1)
    return np.where(bad[..., None], 0, np.nan_to_num(codes)).astype(np.int8), np.where(bad, np.float32(NAN), scales)


def _codes(seed, shape):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-128, 128, shape, generator=g, dtype=torch.int32).to(torch.int8)


def _reals(seed, shape, low=0.01):
    return torch.rand(shape, generator=torch.Generator().manual_seed(seed)) + low


# ---- 8-bit rows -------------------------------------------------------------------------------

SHAPES = [(1, 1), (1, 31), (3, 32), (2, 33), (5, 64), (7, 100), (33, 257), (4, 1003), (3, 2048), (200, 8), (64, 96),
          (1100, 1500), (3, 5000), (2, 12001), (2, 20011), (1, 70001)]


@pytest.mark.parametrize("rows,c", SHAPES)
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("act", ["none", "relu"])
def test_codes_and_scales_are_the_definition(device, rows, c, kind, act):
    x = _values(rows + c, (rows, c), kind)
    if rows > 2:
        x[rows // 2] = 0
    v = x.float().numpy()
    codes, scales = _row8_32(np.maximum(v, 0) if act == "relu" else v)
    got = M.act_row8(x.to(device), act)
    np.testing.assert_array_equal(got.codes.cpu().numpy(), codes)
    np.testing.assert_array_equal(got.scales.cpu().numpy(), scales)
    for out in (F32, BF16):
        want = torch.from_numpy(codes.astype(np.float32) * scales[:, None]).to(out)
        assert torch.equal(M.row8_expand(got, dtype=out).cpu(), want)


def test_codes_of_extreme_rows(device):
    big, tiny = 3.4028234663852886e38, 2.0 ** -126
    rows = [[127.5, -127.5, 63.75, 0.5], [1.0, 0.5, -0.5, 0.25], [big, -big, big / 2, 1.0], [tiny, -tiny, 0.0, 2.0 ** -149],
            [2.0 ** -110, -(2.0 ** -111), 2.0 ** -117, 0.0], [0.0, -0.0, 0.0, 0.0], [INF, 1.0, 2.0, 3.0],
            [1.0, -INF, 2.0, 3.0], [NAN, 1.0, 2.0, 3.0], [INF, NAN, 0.0, 1.0], [254.0, 1.0, 3.0, -5.0]]
    for width in (4, 7, 600, 5000, 20000):
        x = np.zeros((len(rows), width), np.float32)
        x[:, -4:] = rows
        codes, scales = _row8_32(x)
        got = M.act_row8(torch.from_numpy(x).to(device))
        np.testing.assert_array_equal(got.codes.cpu().numpy(), codes)
        np.testing.assert_array_equal(got.scales.cpu().numpy(), scales)
        assert np.isnan(scales[6:10]).all() and (codes[6:10] == 0).all() and np.isfinite(scales[:6]).all()
        assert torch.isnan(M.row8_expand(got)[6:10]).all()


def _act64(v, act):
    if act == "silu":
        return v / (1 + np.exp(-v))
    if act == "gelu":
        return 0.5 * v * np.vectorize(math.erfc)(-v / math.sqrt(2))
    return np.maximum(v, 0) if act == "relu" else v


@pytest.mark.parametrize("rows,c", [(1, 1), (3, 33), (5, 100), (1030, 600), (2, 4096), (3, 9001), (2, 18001)])
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("gated", [False, True])
def test_activations_as_rows(device, rows, c, kind, act, gated):
    if rows * c > 10000 and act == "gelu":
        rows = min(rows, 8)
    x = _values(c, (rows, 2 * c if gated else c), kind, 1.5)
    v = x.double().numpy()
    gate = v[:, :c]
    want = _act64(gate, act) * (v[:, c:] if gated else 1)
    off = (18 + 4 * gate ** 2) * U * np.abs(want)  # of each value
    m = np.maximum(np.abs(want).max(1), float(LEAST))
    m_off = (off.max(1) / m)[:, None]
    got = M.act_row8(x.to(device), act, gated=gated)
    codes, scales = got.codes.cpu().double().numpy(), got.scales.cpu().double().numpy()
    near = 0.5 + 127 * (off / m[:, None] + m_off + 4 * U)
    assert (np.abs(codes - want * 127 / m[:, None]) <= near).all()
    assert (np.abs(scales - m / 127) <= (m_off[:, 0] + 2 * U) * m / 127).all()


# ---- the norm -----------------------------------------------------------------------------------

NORMS = [(1, 1), (1, 3), (4, 33), (7, 64), (5, 100), (1100, 1500), (9, 1001), (4, 4096), (3, 8191), (2, 12001), (2, 33001)]


def _norm64(s, gain, eps):
    r = 1 / np.sqrt((s ** 2).mean(1, keepdims=True) + eps)
    return s * r, s * r * gain, r


@pytest.mark.parametrize("rows,c", NORMS)
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("gain_kind", [F32, BF16])
@pytest.mark.parametrize("added", [False, True])
def test_norm(device, rows, c, kind, gain_kind, added):
    x, gain = _values(rows, (rows, c), kind), (1 + 0.2 * _values(c, (1, c), F32)[0]).to(gain_kind)
    add = _values(rows + 1, (rows, c), kind) if added else None
    s = (x.float() + add.float()).to(kind) if added else x
    eps = 1e-5
    _, want, r = _norm64(s.double().numpy(), gain.double().numpy(), eps)
    off = (c / 2048 + 40) * U
    held = x.to(device), gain.to(device)
    more = add.to(device) if added else None
    y = M.rms_fprop(*held, add=more, eps=eps)
    kept = M.rms_row8(*held, add=more, eps=eps)
    if added:
        assert torch.equal(y[1].cpu(), s) and torch.equal(kept[1].cpu(), s)
        y, kept = y[0], kept[0]
    assert (np.abs(y.cpu().double().numpy() - want) <= (off + _half_step(kind)) * np.abs(want) + 2.0 ** -130).all()
    m = np.abs(want).max(1)
    codes, scales = kept.codes.cpu().double().numpy(), kept.scales.cpu().double().numpy()
    assert (np.abs(codes - want * (127 / m)[:, None]) <= 0.5 + 127 * 5 * U).all()
    assert (np.abs(scales - m / 127) <= (off + 4 * U) * m / 127).all()


@pytest.mark.parametrize("c", [5, 700, 2500, 20000])
def test_norm_of_extreme_rows(device, c):
    """Squares that overflow, rows of zeros, infinities and NaN, values far below eps."""
    x = torch.zeros((7, c))
    g = torch.Generator().manual_seed(c)
    part = torch.randn((5,), generator=g)
    x[0, :5] = part * 1e30
    x[1, :5] = part * 1e-30
    x[2, :5] = torch.tensor([3e38, -3e38, 1.0, 0.0, 2e38])
    x[4, 2] = INF
    x[5, 1] = NAN
    x[6, :5] = part * 1e18
    gain = torch.full((c,), 0.5)
    n, want, _ = _norm64(x[:, :].double().numpy(), 0.5, 1e-6)
    y = M.rms_fprop(x.to(device), gain.to(device)).cpu().double().numpy()
    kept = M.rms_row8(x.to(device), gain.to(device))
    fine = [0, 1, 2, 3, 6]
    assert (np.abs(y - want)[fine] <= (c / 2048 + 40) * U * np.abs(want)[fine] + 2.0 ** -126).all()
    assert np.isnan(y[5]).all() and np.isnan(y[4, 2]) and (y[4, 3:] == 0).all()
    scales = kept.scales.cpu().numpy()
    assert np.isnan(scales[4]) and np.isnan(scales[5]) and (kept.codes[4:6] == 0).all()
    m = np.abs(want).max(1)
    for i in (0, 2, 6):
        assert abs(scales[i] * 127 / m[i] - 1) <= (c / 2048 + 44) * U
        assert (np.abs(kept.codes[i].cpu().double().numpy() - want[i] * 127 / m[i]) <= 0.5 + 127 * 5 * U).all()
    assert (kept.codes[3] == 0).all() and scales[3] >= 0
    dy = torch.randn((7, c), generator=g)
    dx, dgain = M.rms_bprop(dy[:4].to(device), x[:4].to(device), gain.to(device))
    d = dy[:4].double().numpy()
    dn = d * 0.5
    n, _, r = _norm64(x[:4].double().numpy(), 0.5, 1e-6)
    back = r * (dn - n * (dn * n).mean(1, keepdims=True))
    size = r * (np.abs(dn) + np.abs(n) * (np.abs(dn * n)).mean(1, keepdims=True))
    assert (np.abs(dx.cpu().double().numpy() - back) <= (c / 512 + 200) * U * size + 2.0 ** -126).all()
    assert (np.abs(dgain.cpu().double().numpy() - (d * n).sum(0)) <= (c / 2048 + 150) * U * np.abs(d * n).sum(0)).all()


@pytest.mark.parametrize("rows,c", NORMS + [(0, 40), (4500, 257)])
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("more", [False, True])
def test_norm_backward(device, rows, c, kind, more):
    x, dy = _values(rows, (rows, c), kind), _values(rows + 2, (rows, c), kind)
    gain = 1 + 0.2 * _values(c, (1, c), F32)[0]
    dsum = _values(rows + 3, (rows, c), kind) if more else None
    start = _values(5, (1, c), F32)[0]
    n, _, r = _norm64(x.double().numpy(), 1.0, 1e-6)
    d = dy.double().numpy()
    dn = d * gain.double().numpy()
    want = r * (dn - n * (dn * n).mean(1, keepdims=True)) if rows else d
    size = r * (np.abs(dn) + np.abs(n) * np.abs(dn * n).mean(1, keepdims=True)) if rows else d
    if more:
        want = want + dsum.double().numpy()
        size = size + np.abs(dsum.double().numpy())
    at = dict(dsum=dsum.to(device) if more else None)
    dx, dgain = M.rms_bprop(dy.to(device), x.to(device), gain.to(device), **at)
    off = (c / 512 + 150) * U * size
    assert (np.abs(dx.cpu().double().numpy() - want) <= off + _half_step(kind) * (np.abs(want) + off)).all()
    total, size = (d * n).sum(0), np.abs(d * n).sum(0)
    off = (rows / 500 + c / 2048 + 150) * U * size
    assert dgain.dtype == F32 and (np.abs(dgain.cpu().double().numpy() - total) <= off).all()
    again = M.rms_bprop(dy.to(device), x.to(device), gain.to(device), dtype=BF16, **at)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dgain.to(BF16))
    onto = start.to(device)
    M.rms_bprop(dy.to(device), x.to(device), gain.to(device), dgain=onto, accumulate=True, **at)
    assert (np.abs(onto.cpu().double().numpy() - total - start.double().numpy()) <=
            off + 34 * U * (size + np.abs(start.double().numpy()))).all()


def test_norm_backward_against_differences(device):
    """The gradient of sum(y * dy) by central differences in 64 bits."""
    rows, c, eps, h = 3, 37, 1e-3, 1e-6
    x, gain, dy = _values(1, (rows, c), F32), 1 + 0.2 * _values(2, (1, c), F32)[0], _values(3, (rows, c), F32)
    dx, dgain = M.rms_bprop(dy.to(device), x.to(device), gain.to(device), eps=eps)
    x64, g64, d64 = x.double().numpy(), gain.double().numpy(), dy.double().numpy()

    def loss(s, g):
        return (_norm64(s, g, eps)[1] * d64).sum()

    want_x, want_g = np.zeros_like(x64), np.zeros_like(g64)
    for i in range(rows):
        for j in range(c):
            e = np.zeros_like(x64)
            e[i, j] = h
            want_x[i, j] = (loss(x64 + e, g64) - loss(x64 - e, g64)) / (2 * h)
    for j in range(c):
        e = np.zeros_like(g64)
        e[j] = h
        want_g[j] = (loss(x64, g64 + e) - loss(x64, g64 - e)) / (2 * h)
    # differences: h^2 of third derivatives, and 2^-52 / h of the loss
    near = 1e-8 * (1 + np.abs(d64).sum()) + 300 * U * np.abs(d64).max()
    assert np.abs(dx.cpu().double().numpy() - want_x).max() <= near * 10
    assert np.abs(dgain.cpu().double().numpy() - want_g).max() <= near * 10


# ---- products -------------------------------------------------------------------------------------

def _product32(x, w, xs, ws, bias, add, kind):
    """The product of codes and the fp32 operations after it, in their order."""
    sums = x.double().numpy() @ w.double().numpy().T  # integers below 2^31: exact
    y = sums.astype(np.float32) * xs.numpy()[:, None] * ws.numpy()[None]
    if bias is not None:
        y = y + bias.numpy()[None]
    if add is not None:
        y = y + add.float().numpy()
    return torch.from_numpy(y).to(kind)


PRODUCTS = [(1, 1, 1), (1, 15, 3), (2, 16, 17), (3, 17, 40), (5, 63, 64), (16, 64, 16), (17, 65, 33), (31, 100, 257),
            (64, 128, 64), (65, 129, 100), (100, 1001, 300), (128, 256, 128), (130, 1024, 512), (1, 4096, 1024),
            (4, 2051, 777), (33, 8192, 128), (257, 320, 384), (300, 77, 1030), (513, 640, 520), (70, 131071, 20),
            (1, 131071, 2), (5, 0, 9)]


@pytest.mark.parametrize("rows,c,k", PRODUCTS)
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("with_bias,with_add", [(False, False), (True, True), (False, True)])
def test_linear(device, rows, c, k, kind, with_bias, with_add):
    x, w = _codes(rows, (rows, c)), _codes(k, (k, c))
    xs, ws = _reals(1, (rows,)), _reals(2, (k,)) / 1000
    bias = _values(4, (1, k), F32)[0] if with_bias else None
    add = _values(5, (rows, k), kind) if with_add else None
    want = _product32(x, w, xs, ws, bias, add, kind)
    got = M.row8_linear(M.Row8(x.to(device), xs.to(device)), M.Row8(w.to(device), ws.to(device)),
                        bias=None if bias is None else bias.to(device), add=None if add is None else add.to(device),
                        dtype=kind)
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("rows,c,k", [(3, 100, 70), (1, 4096, 512), (200, 256, 300), (300, 131071, 16)])
def test_linear_of_largest_sums(device, rows, c, k):
    """128 * 128 * c stays in 32 bits; rows whose scale is NaN, infinite or zero keep to themselves."""
    x, w = torch.full((rows, c), -128, dtype=torch.int8), torch.full((k, c), -128, dtype=torch.int8)
    xs = torch.ones((rows,))
    xs[0] = NAN if rows > 1 else 1
    xs[rows // 2] = 0 if rows > 2 else 1
    got = M.row8_linear(M.Row8(x.to(device), xs.to(device)), M.Row8(w.to(device), torch.ones((k,), device=device)), dtype=F32)
    want = (np.float32(16384.0 * c) * xs)[:, None].expand(rows, k)
    torch.testing.assert_close(got.cpu(), want, rtol=0, atol=0, equal_nan=True)


def _experts32(x, w, xs, ws, bias, offsets, index, n, kind):
    y = torch.full((n, w.shape[1]), -7.0).to(kind)
    for e in range(w.shape[0]):
        at = torch.arange(int(offsets[e]), int(offsets[e + 1]))
        if len(at) == 0:
            continue
        of = at if index is None else index[at].long()
        there = (of >= 0) & (of < x.shape[0])
        rows = torch.where(there[:, None], x[of.clamp(0, x.shape[0] - 1)], torch.zeros((), dtype=torch.int8))
        scales = torch.where(there, xs[of.clamp(0, x.shape[0] - 1)], torch.zeros(()))
        y[at] = _product32(rows, w[e], scales, ws[e], None if bias is None else bias[e], None, kind)
    return y


EXPERTS = [([0, 0, 0], 5, 33, 20), ([1], 1, 64, 16), ([3, 0, 5], 8, 17, 33), ([64, 1, 0, 0, 70], 140, 128, 100),
           ([0, 200, 3], 210, 96, 65), ([1] * 70, 70, 256, 48), ([0] * 130 + [2, 0, 9], 11, 100, 130),
           ([300, 0, 17, 129], 450, 512, 260), ([40, 7, 0, 21], 68, 1003, 130), ([600, 513], 1200, 192, 300), ([2, 2], 4, 0, 5)]


@pytest.mark.parametrize("counts,n,c,k", EXPERTS)
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("gathered", [False, True])
@pytest.mark.parametrize("with_bias", [False, True])
def test_experts_products(device, counts, n, c, k, kind, gathered, with_bias):
    experts = len(counts)
    offsets = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32)
    m = 37 if gathered else n
    index = None
    if gathered:  # rows out of order, the same one twice, and some outside
        index = torch.randint(-2, m + 2, (n,), generator=torch.Generator().manual_seed(n), dtype=torch.int32)
        index[-1] = -2 ** 31
    x, w = _codes(1, (m, c)), _codes(2, (experts, k, c))
    xs, ws = _reals(3, (m,)), _reals(4, (experts, k)) / 100
    bias = _values(6, (experts, k), F32) if with_bias else None
    want = _experts32(x, w, xs, ws, bias, offsets, index, n, kind)
    out = torch.full((n, k), -7.0, dtype=kind, device=device)
    got = M.row8_experts(M.Row8(x.to(device), xs.to(device)), M.Row8(w.to(device), ws.to(device)), offsets.to(device),
                         rows=None if index is None else index.to(device),
                         bias=None if bias is None else bias.to(device), out=out)
    assert got is out and torch.equal(got.cpu(), want)  # rows behind the last expert's as they were


def test_experts_offsets_outside_the_rows_are_held_to_them(device):
    x, w = M.Row8(_codes(1, (10, 64)).to(device), _reals(1, (10,)).to(device)), \
        M.Row8(_codes(2, (3, 16, 64)).to(device), _reals(2, (3, 16)).to(device))
    wild = torch.tensor([-5, 4, 100, 2 ** 31 - 1], dtype=torch.int32, device=device)
    held = torch.tensor([0, 4, 10, 10], dtype=torch.int32, device=device)
    assert torch.equal(M.row8_experts(x, w, wild, dtype=F32), M.row8_experts(x, w, held, dtype=F32))


# ---- experts' rows ------------------------------------------------------------------------------------

@pytest.mark.parametrize("tokens,slots,experts", [(0, 2, 3), (1, 1, 1), (5, 2, 4), (64, 1, 7), (100, 4, 64), (1000, 3, 100),
                                                  (4097, 2, 8), (30000, 2, 33), (3, 1, 4096)])
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_plan(device, tokens, slots, experts, kind):
    g = torch.Generator().manual_seed(tokens)
    ids = torch.randint(-1, experts + 1, (tokens, slots), generator=g).to(kind)
    if tokens > 50:
        ids[7, 0] = torch.iinfo(kind).max
        ids[9, 0] = torch.iinfo(kind).min
        ids[ids == experts // 2] = 0  # one without rows
    flat = ids.flatten().numpy()
    there = (flat >= 0) & (flat < experts)
    order = np.argsort(np.where(there, flat, experts), kind="stable")
    total = int(there.sum())
    rows = np.where(np.arange(flat.size) < total, order // slots, -1)
    places = np.full(flat.size, -1)
    places[order[:total]] = np.arange(total)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[there].astype(np.int64), minlength=experts))])
    plan = M.experts_plan(ids.to(device), experts)
    np.testing.assert_array_equal(plan.offsets.cpu().numpy(), offsets)
    np.testing.assert_array_equal(plan.rows.cpu().numpy(), rows)
    np.testing.assert_array_equal(plan.places.cpu().numpy(), places.reshape(tokens, slots))


@pytest.mark.parametrize("tokens,slots,c", [(0, 2, 8), (1, 1, 1), (5, 2, 33), (70, 3, 100), (300, 4, 1030), (9, 8, 4096)])
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("with_add", [False, True])
def test_join(device, tokens, slots, c, kind, with_add):
    n = tokens * slots
    y, share = _values(1, (n, c), kind), _reals(2, (tokens, slots))
    places = torch.randint(-1, n + 1, (tokens, slots), generator=torch.Generator().manual_seed(3), dtype=torch.int32)
    add = _values(4, (tokens, c), kind) if with_add else None
    want = add.float().numpy() if with_add else np.zeros((tokens, c), np.float32)
    for s in range(slots):
        p = places[:, s].numpy()
        there = (p >= 0) & (p < n)
        term = y.float().numpy()[np.where(there, p, 0)] * share[:, s].numpy()[:, None] if n else 0 * want
        want = np.where(there[:, None], want + term, want)
    at = dict(add=add.to(device) if with_add else None)
    got = M.experts_join(y.to(device), places.to(device), share.to(device), **at)
    assert torch.equal(got.cpu(), torch.from_numpy(want).to(kind))
    ones = M.experts_join(y.to(device), places.to(device), torch.ones_like(share).to(device), **at)
    assert torch.equal(M.experts_join(y.to(device), places.to(device), **at), ones)
