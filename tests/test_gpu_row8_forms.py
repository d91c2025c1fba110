"""Forms of the calls on 8-bit rows: row slices, sums in place, other streams, graphs replayed on other
inputs, tensors beyond 32-bit offsets, a layer of experts as it is used.  Each is compared with the plain
call on contiguous tensors (tested against 64 bits elsewhere), bit for bit, or with exact integers."""
import numpy as np
import pytest
import torch

import my_own_cnn_amd as M
from tests.test_gpu_token_forms import _around, _slice

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _real(seed, shape, kind, device):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(kind).to(device)


def _row8(seed, rows, c, device):
    return M.act_row8(_real(seed, rows + (c,), F32, device))


def _same(got, want):
    got, want = (t if isinstance(t, (tuple, list)) else [t] for t in (got, want))
    for a, b in zip(got, want):
        if isinstance(a, tuple):
            _same(a, b)
        else:
            assert torch.equal(a, b)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("c", [1, 7, 33, 100, 1003, 2500, 20001])
def test_row_slices(device, kind, c):
    x, add, dy, dsum = (_real(i, (3, 5, c), kind, device) for i in range(4))
    both = _real(7, (3, 5, 2 * c), kind, device)
    gain = _real(5, (c,), F32, device)
    y, total = M.rms_fprop(x, gain, add=add)
    kept = M.rms_row8(x, gain, add=add)
    dx, dgain = M.rms_bprop(dy, total, gain, dsum=dsum)
    gate = M.act_row8(both, "silu", gated=True)
    real = M.row8_expand(gate, dtype=kind)
    for before, after in [(1, 0), (3, 2), (8, 9)]:
        xs, adds, dys, dsums = (_slice(t, before, after + i)[0] for i, t in enumerate((x, add, dy, dsum)))
        out, wide = _slice(torch.zeros_like(x), before, after)
        s, s_wide = _slice(torch.zeros_like(x), after, before)
        _same(M.rms_fprop(xs, gain, add=adds, out=out, total=s), (y, total))
        assert _around(out, wide, before) and _around(s, s_wide, after)
        assert torch.equal(M.rms_fprop(xs, gain), M.rms_fprop(x, gain))
        _same(M.rms_row8(xs, gain, add=adds), kept)
        out, wide = _slice(torch.zeros_like(x), before, after)
        _same(M.rms_bprop(dys, s, gain, dsum=dsums, out=out), (dx, dgain))
        assert _around(out, wide, before)
        _same(M.act_row8(_slice(both, before, after)[0], "silu", gated=True), gate)
        out, wide = _slice(torch.zeros_like(real), before, after)
        assert torch.equal(M.row8_expand(gate, out=out), real) and _around(out, wide, before)
        # the sum in place of an addend
        mine = _slice(x, before, after)[0]
        _same(M.rms_fprop(mine, gain, add=adds, total=mine), (y, total))
        mine = add.clone()
        _same(M.rms_row8(x, gain, add=mine, total=mine), (kept[0], total))


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("rows,c,k", [(1, 64, 33), (3, 100, 70), (20, 256, 130), (200, 512, 257), (600, 1003, 300)])
def test_products_into_row_slices(device, kind, rows, c, k):
    x, w = _row8(1, (rows,), c, device), _row8(2, (k,), c, device)
    add = _real(3, (rows, k), kind, device)
    want = M.row8_linear(x, w, add=add)
    plain = M.row8_linear(x, w, dtype=kind)
    offsets = torch.tensor([0, rows // 3, rows], dtype=torch.int32, device=device)
    w2 = M.Row8(torch.stack([w.codes, w.codes]), torch.stack([w.scales, w.scales]))
    places = torch.arange(rows, dtype=torch.int32, device=device)
    for before, after in [(1, 0), (3, 2), (8, 9)]:
        adds = _slice(add, after, before)[0]
        out, wide = _slice(torch.zeros_like(add), before, after)
        assert torch.equal(M.row8_linear(x, w, add=adds, out=out), want) and _around(out, wide, before)
        assert torch.equal(M.row8_linear(x, w, add=adds, out=adds), want)
        out, wide = _slice(torch.zeros_like(add), before, after)
        assert torch.equal(M.row8_experts(x, w2, offsets, out=out), plain) and _around(out, wide, before)
        back, wide = _slice(torch.zeros_like(add), after, before)
        assert torch.equal(M.experts_join(out, places, out=back), plain) and _around(back, wide, after)


def test_products_of_codes_at_any_address(device):
    """Codes that start at odd addresses, as slices of a larger buffer do."""
    for c, k, rows in [(64, 40, 9), (256, 130, 100), (1024, 300, 300)]:
        x, w = _row8(1, (rows,), c, device), _row8(2, (k,), c, device)
        want = M.row8_linear(x, w)
        for shift in (1, 4, 8):
            buffer = torch.zeros((rows + k) * c + 64, dtype=torch.int8, device=device)
            xc = buffer[shift: shift + rows * c].view(rows, c)
            wc = buffer[shift + rows * c: shift + (rows + k) * c].view(k, c)
            xc.copy_(x.codes)
            wc.copy_(w.codes)
            assert torch.equal(M.row8_linear(M.Row8(xc, x.scales), M.Row8(wc, w.scales)), want)


def _layer(x, gain, residual, ids, share, w, v, **on):
    """A layer of experts as it is used: norm, plan, products, the gated activation, join."""
    kept, total = M.rms_row8(x, gain, add=residual, **on)
    plan = M.experts_plan(ids, w.codes.shape[0], **on)
    h = M.row8_experts(kept, w, plan.offsets, rows=plan.rows, **on)
    y = M.row8_experts(M.act_row8(h, "silu", gated=True, **on), v, plan.offsets, **on)
    return M.experts_join(y, plan.places, share, add=total, **on), total


def _state(device, tokens, slots, experts, c, hidden, seed):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(experts, generator=g)[:slots] for _ in range(tokens)])
    ids[torch.rand((tokens,), generator=g) < 0.1] = -1
    return [_real(seed, (tokens, c), BF16, device), 1 + 0.1 * _real(seed + 1, (c,), F32, device),
            _real(seed + 2, (tokens, c), BF16, device), ids.to(torch.int32).to(device),
            torch.softmax(torch.randn((tokens, slots), generator=g), 1).to(device)]


def _weights(device, experts, c, hidden):
    return (_row8(11, (experts, 2 * hidden), c, device), _row8(12, (experts, c), hidden, device))


@pytest.mark.parametrize("tokens,slots,experts,c,hidden", [(1, 2, 8, 64, 32), (5, 2, 16, 128, 96), (150, 2, 4, 256, 160),
                                                           (700, 3, 5, 320, 100)])
def test_a_layer_of_experts(device, tokens, slots, experts, c, hidden):
    """Against the same layer in 64 bits from the same norm's codes: the rows between two operators are
    rounded to bf16 and to codes, so a rounding that falls the other way moves a value of h by a bf16
    step (2^-8 of it) and one of the activation by a code."""
    x, gain, residual, ids, share = _state(device, tokens, slots, experts, c, hidden, 3)
    w, v = _weights(device, experts, c, hidden)
    got, total = _layer(x, gain, residual, ids, share, w, v)
    kept, _ = M.rms_row8(x, gain, add=residual)

    def real(r):
        return r.codes.double().cpu() * r.scales.double().cpu()[..., None]

    a, w64, v64 = real(kept), real(w), real(v)
    want = total.double().cpu()
    slack = torch.zeros_like(want)
    for t in range(tokens):
        for s in range(slots):
            e = int(ids[t, s])
            if e < 0:
                continue
            h = (w64[e] @ a[t]).to(BF16).double()
            z = h[:hidden] * torch.sigmoid(h[:hidden]) * h[hidden:]
            step = z.abs().max() / 127
            y = v64[e] @ (torch.round(z / step) * step)
            p = float(share[t, s])
            want[t] += p * y.to(BF16).double()
            # every code and every h may fall the other way; silu moves by at most 1.1 of its argument
            moved = step + 2 ** -8 * (2.2 * h[:hidden].abs() * h[hidden:].abs())
            slack[t] += p * (v64[e].abs() @ moved + 2 ** -8 * y.abs())
    off = (got.double().cpu() - want).abs()
    assert bool((off <= slack + 2 ** -8 * (want.abs() + slack) + 1e-6).all())
    assert float((off ** 2).mean().sqrt()) <= 2 ** -8 * float((want ** 2).mean().sqrt())


def test_a_layer_on_another_stream_and_again(device):
    w, v = _weights(device, 8, 256, 128)
    state = _state(device, 90, 2, 8, 256, 128, 5)
    want = _layer(*state, w, v)
    _same(_layer(*state, w, v), want)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = _layer(*state, w, v, stream=side)
    side.synchronize()
    _same(got, want)


@pytest.mark.parametrize("tokens", [4, 300])
def test_a_layer_in_a_graph(device, tokens):
    """Replayed on other inputs, routes among them, with eager work between the replays."""
    w, v = _weights(device, 8, 256, 128)
    state = _state(device, tokens, 2, 8, 256, 128, 5)
    lin = _row8(15, (500,), 256, device)
    gain = state[1]

    def calls(x, gain, residual, ids, share):
        out, total = _layer(x, gain, residual, ids, share, w, v)
        y = M.row8_linear(M.rms_row8(out, gain), lin)
        dx, dgain = M.rms_bprop(out, total, gain, dsum=x)
        return out, total, y, dx, dgain

    calls(*state)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = calls(*state)
    for seed in range(4):
        for to, of in zip(state, _state(device, tokens, 2, 8, 256, 128, 20 + seed)):
            to.copy_(of)
        for t in held:
            t.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        _same(held, calls(*state))


def test_rows_beyond_32_bit_offsets(device):
    """4.6e9 codes: the last rows are what they are alone."""
    c, rows = 65536, 70000
    x = torch.zeros((rows, c), dtype=BF16, device=device)
    last = _real(1, (40, c), BF16, device)
    x[-40:] = last
    gain = torch.ones((c,), device=device)
    kept = M.rms_row8(x, gain)
    want = M.rms_row8(last, gain)
    assert torch.equal(kept.codes[-40:], want.codes) and torch.equal(kept.scales[-40:], want.scales)
    assert not bool(kept.codes[:5].any())
    made = M.act_row8(x)
    want = M.act_row8(last)
    assert torch.equal(made.codes[-40:], want.codes) and torch.equal(made.scales[-40:], want.scales)
    y = M.row8_expand(made, dtype=BF16)
    assert torch.equal(y[-40:], M.row8_expand(want, dtype=BF16))
    del x, y
    w = _row8(3, (48,), c, device)
    assert torch.equal(M.row8_linear(made, w)[-40:], M.row8_linear(want, w))
    # as weights of experts, the rows of x gathered from the end
    wide = M.Row8(made.codes.view(70, 1000, c), made.scales.view(70, 1000))
    offsets = torch.zeros(71, dtype=torch.int32, device=device)
    offsets[70] = 48
    got = M.row8_experts(w, wide, offsets)
    assert torch.equal(got[:, -40:], M.row8_linear(w, want))
    index = torch.arange(rows - 48, rows, dtype=torch.int32, device=device)
    one = M.Row8(w.codes[None], w.scales[None])
    at = torch.tensor([0, 48], dtype=torch.int32, device=device)
    got = M.row8_experts(made, one, at, rows=index)
    assert torch.equal(got[-40:], M.row8_linear(want, w))
