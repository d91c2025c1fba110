"""Activations kept in 8 bits on the GPU (miq_act8_fprop, _bprop, _expand, _grad).

Codes and exponent bytes are exact: equal to their definition computed in 64 bits.  With
u = 2^-24 (half a unit of fp32):
  - an activation: exp and erfc are good to a few units, silu is two more operations (16 u of the
    value); gelu's erfc takes a rounded argument z = v / sqrt 2, which moves it by z^2 u more in
    relative terms on the falling side: (16 + 4 v^2) u of the value;
  - a derivative is a sum of terms of at most 1 + |v|: (16 + 4 |v| + 4 v^2) u, absolute;
  - a weight gradient sums `rows` products in fp32 and three pieces a product: (rows + 4) * 2 u of
    the sum of magnitudes (matrix instructions may round by a whole unit).
A bf16 result is the rounding of a value within these bounds."""
import math

import numpy as np
import pytest
import torch

import my_own_cnn_amd as M

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24
INF, NAN = float("inf"), float("nan")


def _keep64(x, halves=1):
    """(codes, bytes, values) of x (rows, halves * c) by the definition, in 64 bits."""
    rows, width = x.shape
    c = width // halves
    groups = -(-c // 32)
    codes = np.zeros((rows, width), np.int8)
    scales = np.zeros((rows, halves * groups), np.uint8)
    values = np.zeros((rows, width))
    for h in range(halves):
        for g in range(groups):
            part = x[:, h * c + g * 32: h * c + min(g * 32 + 32, c)].astype(np.float64)
            at = slice(h * c + g * 32, h * c + g * 32 + part.shape[1])
            top = np.abs(part).max(1)
            bad = ~np.isfinite(part).all(1)
            part, top = np.where(bad[:, None], 0, part), np.where(bad, 0, top)
            e = np.where(top > 0, np.frexp(np.where(top > 0, top, 1))[1] - 1, -2000)  # 2^e <= top
            b = e - 6 + 127
            b = b + (np.rint(top * 2.0 ** np.clip(6 - e, -1000, 1000)) > 127)
            b = np.clip(b, 1, 248)
            step = 2.0 ** (b - 127.0)
            q = np.clip(np.rint(part / step[:, None]), -127, 127)
            codes[:, at] = q
            scales[:, h * groups + g] = np.where(bad, 255, b)
            values[:, at] = np.where(bad[:, None], np.nan, q * step[:, None])
    return codes, scales, values


def _values(seed, rows, c, kind):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, c), generator=g) * torch.exp(2 * torch.randn((1, c), generator=g))
    if rows > 2:
        x[rows // 2] = 0
    return x.to(kind)


SHAPES = [(1, 1), (1, 31), (3, 32), (2, 33), (5, 64), (7, 100), (33, 257), (4, 1003), (3, 2048), (200, 8), (64, 96)]


@pytest.mark.parametrize("rows,c", SHAPES)
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("halves", [1, 2])
def test_codes_bytes_and_values_are_the_definition(device, rows, c, kind, halves):
    x = _values(rows + c, rows, c * halves, kind)
    codes, scales, values = _keep64(x.double().numpy(), halves)
    y, kept = M.act8_fprop(x.to(device), "silu", gated=halves == 2)
    np.testing.assert_array_equal(kept.codes.cpu().numpy(), codes)
    np.testing.assert_array_equal(kept.scales.cpu().numpy(), scales)
    for out in (F32, BF16):  # exact in both
        np.testing.assert_array_equal(M.act8_expand(kept, dtype=out).cpu().double().numpy(), values)
    if halves == 1:
        only = M.act8_keep(x.to(device))
        assert torch.equal(only.codes, kept.codes) and torch.equal(only.scales, kept.scales)


def test_codes_of_extreme_groups(device):
    big, tiny, sub = 3.4028234663852886e38, 2.0 ** -126, 2.0 ** -149
    groups = [
        [127.5, -127.5, 1.0, 0.5], [127.49, 126.5, 2.5, -3.5], [255.0, 254.0, -1.0, 1.0], [64.0, 0.5, 1.5, -0.5],
        [big, -big, big / 2, 1.0], [big * 0.99, 1e30, -1e37, 0.0], [tiny, -tiny, tiny / 2, sub], [sub, -sub, 0.0, 0.0],
        [0.0, -0.0, 0.0, 0.0], [2.0 ** -120, 2.0 ** -127, -(2.0 ** -126), sub], [2.0 ** -121, 1.5 * 2.0 ** -126, 0.0, sub],
        [INF, 1.0, 2.0, 3.0], [1.0, -INF, 2.0, 3.0], [NAN, 1.0, 2.0, 3.0], [INF, NAN, 0.0, 1.0], [1.0, 2.0, 3.0, 4.0],
    ]
    x = np.zeros((2, len(groups) * 32), np.float32)
    for i, g in enumerate(groups):
        x[0, i * 32: i * 32 + 4] = g
        x[1, i * 32 + 28: i * 32 + 32] = g
    codes, scales, values = _keep64(x)
    kept = M.act8_keep(torch.from_numpy(x).to(device))
    np.testing.assert_array_equal(kept.codes.cpu().numpy(), codes)
    np.testing.assert_array_equal(kept.scales.cpu().numpy(), scales)
    assert (kept.codes.cpu().numpy()[:, 11 * 32: 15 * 32] == 0).all() and (scales[:, 11:15] == 255).all()
    for out in (F32, BF16):
        np.testing.assert_array_equal(M.act8_expand(kept, dtype=out).cpu().double().numpy(), values)


# ---- activations ------------------------------------------------------------------------------

def _erfc(v):
    return np.vectorize(math.erfc)(v) if v.size else v


def _sigmoid(v):
    e = np.exp(-np.abs(v))
    return np.where(v >= 0, 1 / (1 + e), e / (1 + e))


def _act(v, act):
    if act == "none":
        return v
    if act == "relu":
        return np.maximum(v, 0)
    if act == "silu":
        return v * _sigmoid(v)
    return 0.5 * v * _erfc(-v / math.sqrt(2))


def _slope(v, act):
    if act == "none":
        return np.ones_like(v)
    if act == "relu":
        return (v > 0).astype(np.float64)
    if act == "silu":
        s = _sigmoid(v)
        return s * (1 + v * _sigmoid(-v))
    return 0.5 * _erfc(-v / math.sqrt(2)) + v * np.exp(-v * v / 2) / math.sqrt(2 * math.pi)


def _value_room(v, act):
    return (16 + (4 * v * v if act == "gelu" else 0)) * U * np.abs(_act(v, act)) + 2.0 ** -125


def _rounded(v):
    return torch.from_numpy(v).float().bfloat16().double().numpy()


def _near(got, want, room, kind):
    got, off = got.cpu().double().numpy(), np.abs(got.cpu().double().numpy() - want)
    if kind == BF16:
        inside = (got >= _rounded(want - room)) & (got <= _rounded(want + room))
    else:
        inside = off <= room
    assert inside.all(), (int((~inside).sum()), float(off.max()))


@pytest.mark.parametrize("rows,c", [(1, 1), (3, 33), (5, 64), (9, 203), (2, 2049)])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("gated", [False, True])
def test_activation_and_backward_against_64_bits(device, rows, c, act, kind, gated):
    h = 2 if gated else 1
    x = (_values(rows * 3 + c, rows, c * h, F32).clamp(-30, 30)).to(kind)
    g = torch.Generator().manual_seed(5)
    dy = torch.randn((rows, c), generator=g).to(kind)
    y, kept = M.act8_fprop(x.to(device), act, gated=gated)
    dx = M.act8_bprop(dy.to(device), kept)
    v, d = x.double().numpy(), dy.double().numpy()
    gate = v[:, :c]
    up = v[:, c:] if gated else 1.0
    _near(y, _act(gate, act) * up, (_value_room(gate, act) + U * np.abs(_act(gate, act))) * np.abs(up), kind)
    back = _keep64(v, h)[2]
    gate = back[:, :c]
    up = back[:, c:] if gated else np.ones_like(gate)
    room = np.abs(d * up) * ((20 + 4 * np.abs(gate) + 4 * gate * gate) * U) + 2.0 ** -125
    if gated:
        want = np.concatenate([d * up * _slope(gate, act), d * _act(gate, act)], 1)
        room = np.concatenate([room, (_value_room(gate, act) + U * np.abs(_act(gate, act))) * np.abs(d) + 2.0 ** -125], 1)
    else:
        want = d * _slope(gate, act)
    _near(dx, want, room, kind)
    again = M.act8_expand(kept, apply=True, dtype=F32)
    _near(again, _act(gate, act) * up, (_value_room(gate, act) + U * np.abs(_act(gate, act))) * np.abs(up), F32)


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("gated", [False, True])
def test_backward_against_differences(device, act, gated):
    """Central differences of the activation at the kept values, in 64 bits: off by h^2 / 6 times the
    third derivative (below 1 here) and the rounding of the difference, 2^-52 / h."""
    c, rows, h = 65, 4, 1e-4
    halves = 2 if gated else 1
    x = _values(8, rows, c * halves, F32).clamp(-8, 8)
    dy = torch.randn((rows, c), generator=torch.Generator().manual_seed(1))
    _, kept = M.act8_fprop(x.to(device), act, gated=gated)
    dx = M.act8_bprop(dy.to(device), kept).cpu().double().numpy()
    back, d = _keep64(x.double().numpy(), halves)[2], dy.double().numpy()

    def f(v):
        return _act(v[:, :c], act) * (v[:, c:] if gated else 1.0)

    for half in range(halves):
        step = np.zeros_like(back)
        step[:, half * c: half * c + c] = h
        slope = (f(back + step) - f(back - step)) / (2 * h)
        scale = np.abs(d) * (1 + np.abs(back[:, c:] if gated else 1.0)) * (1 + np.abs(back[:, :c])) ** 2
        room = scale * (h * h + 1e-11 + 40 * U)
        assert (np.abs(dx[:, half * c: half * c + c] - d * slope) <= room).all()


def test_large_infinite_and_nan_inputs(device):
    x = torch.zeros((3, 64))
    x[0, :4] = torch.tensor([1e30, -1e30, 200.0, -200.0])
    x[1, 3], x[1, 40] = INF, NAN
    x[2, 0] = -INF
    for act in ("relu", "silu", "gelu"):
        y, kept = M.act8_fprop(x.to(device), act)
        y = y.cpu()
        np.testing.assert_array_equal(y[0, :4].numpy(), np.array([1e30, 0, 200, 0], np.float32))
        assert y[1, 3] == INF and torch.isnan(y[1, 40]) and (y[1, 4:32] == 0).all()
        dx = M.act8_bprop(torch.ones((3, 64), device=device), kept).cpu()
        assert dx[0, 0] == 1 and dx[0, 1] == 0 and torch.isfinite(dx[0]).all()
        # a group that held an infinity or a NaN is NaN as a whole, its neighbours are not
        assert torch.isnan(dx[1]).all() and torch.isnan(dx[2, :32]).all() and torch.isfinite(dx[2, 32:]).all()


def test_row_slices_empty_tensors_and_storage(device):
    g = torch.Generator().manual_seed(2)
    wide = torch.randn((3, 7, 150), generator=g).to(device)
    x = wide[..., 5:105]
    out = torch.full((3, 7, 60), -7.0, device=device)
    y, kept = M.act8_fprop(x, "relu", gated=True, out=out[..., 3:53])
    y2, kept2 = M.act8_fprop(x.contiguous(), "relu", gated=True)
    assert torch.equal(y, y2) and torch.equal(kept.codes, kept2.codes) and torch.equal(kept.scales, kept2.scales)
    assert (out[..., :3] == -7).all() and (out[..., 53:] == -7).all()
    dy = torch.randn((3, 7, 50), generator=g).to(device)
    into = torch.full((3, 7, 111), -7.0, device=device)
    M.act8_bprop(dy, kept, out=into[..., 1:101])
    assert torch.equal(into[..., 1:101], M.act8_bprop(dy, kept2))
    assert (into[..., :1] == -7).all() and (into[..., 101:] == -7).all()
    _, same = M.act8_fprop(x + 1, "relu", gated=True, kept=kept)
    assert same.codes.data_ptr() == kept.codes.data_ptr() and not torch.equal(kept.codes, kept2.codes)
    y, kept = M.act8_fprop(x[:0], "silu")
    assert y.shape == (0, 7, 100) and M.act8_bprop(y, kept).shape == (0, 7, 100)


def test_beyond_32_bit_offsets(device):
    rows, c = 70000, 32768  # 2.3e9 values
    x = torch.zeros((rows, c), dtype=BF16, device=device)
    x[-1] = torch.arange(c, device=device).to(BF16)
    x[65600, :64] = 3.0
    kept = M.act8_keep(x)
    tail = M.act8_keep(x[-2:].contiguous())
    assert torch.equal(kept.codes[-2:], tail.codes) and torch.equal(kept.scales[-2:], tail.scales)
    assert int(kept.codes[65600, :64].sum()) == 64 * 96 and int(kept.codes[65600, 64:].abs().sum()) == 0
    back = M.act8_expand(kept, dtype=BF16, out=x)
    assert torch.equal(back[-1], M.act8_expand(tail, dtype=BF16)[-1]) and (back[65600, :64] == 3).all()


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("gated", [False, True])
def test_outputs_beyond_the_caches(device, kind, gated):
    """Outputs of more than 128 MB take other stores: the same bits as of a few rows at a time."""
    rows, c = 50000, 1472
    x = torch.randn((rows, c * (2 if gated else 1)), device=device).to(kind)
    dy = torch.randn((rows, c), device=device).to(kind)
    y, kept = M.act8_fprop(x, "silu", gated=gated)
    dx, back = M.act8_bprop(dy, kept), M.act8_expand(kept, apply=True, dtype=kind)
    for r in (slice(0, 900), slice(31000, 31333), slice(rows - 700, rows)):
        part = M.Act8(kept.codes[r], kept.scales[r], "silu", gated)
        y1, k1 = M.act8_fprop(x[r], "silu", gated=gated)
        assert torch.equal(y[r], y1) and torch.equal(part.codes, k1.codes) and torch.equal(part.scales, k1.scales)
        assert torch.equal(dx[r], M.act8_bprop(dy[r], part))
        assert torch.equal(back[r], M.act8_expand(part, apply=True, dtype=kind))


# ---- weight gradient --------------------------------------------------------------------------

GRADS = [  # rows, c, k
    (1, 1, 1), (1, 33, 5), (2, 32, 64), (31, 128, 128), (32, 127, 129), (33, 130, 70), (64, 257, 200), (257, 64, 300),
    (1000, 96, 513), (513, 1003, 31), (2049, 256, 256), (5000, 65, 40), (300, 512, 384), (20001, 128, 128),
    (24577, 512, 512), (19999, 300, 1001), (1200, 1500, 2000), (290, 4095, 4081),
]


def _kept(device, seed, rows, c, kind=F32):
    x = _values(seed, rows, c, kind)
    return M.act8_keep(x.to(device)), _keep64(x.double().numpy())[2]


@pytest.mark.parametrize("rows,c,k", GRADS)
@pytest.mark.parametrize("dy_type,out_type", [(F32, F32), (BF16, F32), (BF16, BF16)])
def test_weight_gradient_against_64_bits(device, rows, c, k, dy_type, out_type):
    kept, x = _kept(device, rows + c, rows, c)
    dy = (torch.randn((rows, k), generator=torch.Generator().manual_seed(k)) * 1e-3).to(dy_type)
    got = M.act8_grad(dy.to(device), kept, dtype=out_type)
    assert torch.equal(got, M.act8_grad(dy.to(device), kept, dtype=out_type))  # the same bits
    d = dy.double().numpy()
    _near(got, d.T @ x, (rows + 4) * 2 * U * (np.abs(d).T @ np.abs(x)), out_type)


def test_the_shapes_reach_every_tile_split_and_whole():
    for dtype in (F32, BF16):
        plans = {M.plan_act8_grad(*s, dtype) for s in GRADS}
        assert {(t, n > 1) for t, n in plans} == {(t, b) for t in (64, 128, 256) for b in (False, True)}


@pytest.mark.parametrize("rows,c,k", [(1, 40, 3), (700, 129, 131), (9000, 64, 32), (1500, 300, 260)])
@pytest.mark.parametrize("dy_type", [F32, BF16])
def test_weight_gradient_of_integers_is_exact_and_accumulates(device, rows, c, k, dy_type):
    rng = np.random.default_rng(rows)
    x = rng.integers(-3, 4, (rows, c)).astype(np.float64)
    x[:, ::32] = 64  # 2^0 steps: small integers are kept as they are
    d = rng.integers(-3, 4, (rows, k)).astype(np.float64)
    kept = M.act8_keep(torch.from_numpy(x).float().to(device))
    dy = torch.from_numpy(d).to(dy_type).to(device)
    np.testing.assert_array_equal(M.act8_grad(dy, kept).cpu().numpy(), d.T @ x)
    start = torch.full((k, c), 5.0, device=device)
    np.testing.assert_array_equal(M.act8_grad(dy, kept, accumulate=True, out=start).cpu().numpy(), 5 + d.T @ x)


def test_weight_gradient_holds_all_24_bits_of_dy(device):
    """One term each: a product of 24 by 7 bits, rounded once as its three pieces add up."""
    d = np.array([[1 + 2.0 ** -23, -(2 - 2.0 ** -23), 1.0 / 3, 1e-30, -1e30, 2.0 ** -100]], np.float32)
    x = np.array([[1.0, -127 / 64, 33 / 64]], np.float32)
    kept = M.act8_keep(torch.from_numpy(x).to(device))
    np.testing.assert_array_equal(M.act8_expand(kept).cpu().numpy(), x)
    got = M.act8_grad(torch.from_numpy(d).to(device), kept).cpu().double().numpy()
    want = d.astype(np.float64).T @ x.astype(np.float64)
    assert (np.abs(got - want) <= 4 * U * np.abs(want)).all()


def test_weight_gradient_of_row_slices_and_no_rows(device):
    rng = np.random.default_rng(3)
    x = rng.integers(-3, 4, (2, 50, 96)).astype(np.float32)
    x[..., ::32] = 64
    kept = M.act8_keep(torch.from_numpy(x).to(device))
    for kind in (F32, BF16):
        wide = torch.from_numpy(rng.integers(-3, 4, (2, 50, 90)).astype(np.float32)).to(kind).to(device)
        dy = wide[..., 7:72]
        into = torch.full((65, 105), -7.0, device=device)
        M.act8_grad(dy, kept, out=into[:, 4:100])
        want = dy.reshape(100, 65).cpu().double().numpy().T @ x.reshape(100, 96).astype(np.float64)
        np.testing.assert_array_equal(into[:, 4:100].cpu().numpy(), want)
        assert (into[:, :4] == -7).all() and (into[:, 100:] == -7).all()
    none = M.act8_grad(dy[:0], M.Act8(kept.codes[:0], kept.scales[:0]))
    assert none.shape == (65, 96) and (none == 0).all()


@pytest.mark.parametrize("kind", [F32, BF16])
def test_weight_gradient_of_infinities_and_nan(device, kind):
    rows, c, k = 40, 96, 20
    x = torch.zeros((rows, c))
    x[:, ::32], x[:, 1] = 64, 1
    x[7, 33] = NAN  # channels 32 .. 63 of one row
    d = torch.ones((rows, k))
    d[3, 5], d[4, 6], d[2, 9] = INF, NAN, -INF
    got = M.act8_grad(d.to(kind).to(device), M.act8_keep(x.to(device)), dtype=F32).cpu().numpy()
    assert np.isnan(got[:, 32:64]).all()
    plain = [j for j in range(k) if j not in (5, 6, 9)]
    assert (got[plain][:, [0, 64]] == 64 * rows).all() and (got[plain, 1] == rows).all() and (got[plain, 2] == 0).all()
    assert got[5, 0] == INF and got[9, 0] == -INF and np.isnan(got[6, 0])
    assert np.isnan(got[5, 2]) and got[5, 1] == INF  # infinity times a kept zero


def test_weight_gradient_against_differences(device):
    """sum(dy * (x' w^T)) is linear in w: its differences, with values of few bits, are exact."""
    rng = np.random.default_rng(8)
    rows, c, k = 60, 40, 24
    x = rng.integers(-3, 4, (rows, c)).astype(np.float32)
    x[:, ::32] = 64
    kept = M.act8_keep(torch.from_numpy(x).to(device))
    dy = torch.from_numpy(rng.integers(-3, 4, (rows, k)).astype(np.float32)).to(device)
    dw = M.act8_grad(dy, kept).cpu()
    back = M.act8_expand(kept).reshape(1, rows, 1, c)

    def loss(w):
        y = M.conv2d_nhwc_f32(back, w.reshape(k, 1, 1, c).to(device))
        return float((y.reshape(rows, k).double() * dy.double()).sum())

    w = torch.from_numpy(rng.integers(-2, 3, (k, c)).astype(np.float32))
    for j, i in [(0, 0), (3, 33), (23, 39), (11, 5)]:
        up, down = w.clone(), w.clone()
        up[j, i] += 1
        down[j, i] -= 1
        assert (loss(up) - loss(down)) / 2 == float(dw[j, i])


@pytest.mark.parametrize("rows,c,k,kind", [(3000, 64, 100, F32), (700, 2048, 2048, F32), (700, 2048, 4096, BF16)])
def test_other_stream_and_graph_replays(device, rows, c, k, kind):
    kept, _ = _kept(device, 1, rows, c)
    dy = torch.randn((rows, k), device=device).to(kind)
    want = M.act8_grad(dy, kept)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = M.act8_grad(dy, kept, stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    ws = torch.empty(M.act8_grad_workspace_size(rows, c, k, kind), dtype=torch.uint8, device=device)
    out = torch.empty((k, c), device=device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        M.act8_grad(dy, kept, out=out, workspace=ws)
    for seed in range(4):
        dy.copy_(torch.randn((rows, k), generator=torch.Generator().manual_seed(seed)).to(device))
        out.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, M.act8_grad(dy, kept))


def test_refusals(device):
    x = torch.zeros((3, 64), device=device)
    kept = M.act8_keep(x)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        M.act8_keep(x.half())
    with pytest.raises(ValueError, match="act must be"):
        M.act8_fprop(x, "tanh")
    with pytest.raises(ValueError, match="even number"):
        M.act8_fprop(x[:, :63], "silu", gated=True)
    with pytest.raises(ValueError, match="dy must be"):
        M.act8_bprop(x[:2], kept)
    with pytest.raises(ValueError, match="scales must be"):
        M.act8_bprop(x, M.Act8(kept.codes, kept.scales[:, :1].contiguous()))
    with pytest.raises(ValueError, match="contiguous torch.int8"):
        M.act8_bprop(x, M.Act8(kept.codes.float(), kept.scales))
    with pytest.raises(ValueError, match="not gated"):
        M.act8_grad(x[:, :32], M.Act8(kept.codes, kept.scales, "silu", True))
    with pytest.raises(ValueError, match="rows differ"):
        M.act8_grad(x[:2], kept)
    with pytest.raises(M.MiqError, match="dw_type"):
        M.act8_grad(x, kept, dtype=BF16)
    with pytest.raises(M.MiqError, match="workspace is smaller"):
        big = M.act8_keep(torch.zeros((4000, 64), device=device))
        M.act8_grad(torch.zeros((4000, 64), device=device), big, workspace=torch.empty(16, dtype=torch.uint8, device=device))
