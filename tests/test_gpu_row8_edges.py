"""Calls on 8-bit rows that the documentation allows and that are easy to get wrong: products in graphs with
their workspaces, two streams at once, no rows to take from, more tiles than one launch has, falling
offsets, the same token twice, and the wrappers' refusals."""
import pytest
import torch

import my_own_cnn_amd as M

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _codes(seed, shape, device):
    g = torch.Generator(device=device).manual_seed(seed)
    return torch.randint(-128, 128, shape, generator=g, device=device, dtype=torch.int32).to(torch.int8)


def _row8(seed, shape, device):
    g = torch.Generator(device=device).manual_seed(seed + 100)
    return M.Row8(_codes(seed, shape, device), torch.rand(shape[:-1], generator=g, device=device))


def _want(x, w, kind):
    y = (x.codes.double() @ w.codes.double().t().contiguous()).float() * x.scales[:, None] * w.scales
    return y.to(kind)


# tiles that take more than 64 KB of LDS, and rows copied to a workspace
@pytest.mark.parametrize("rows,c,k", [(700, 1040, 16397), (1030, 2064, 2050), (2050, 643, 6150), (1003, 2051, 1537)])
def test_products_in_graphs(device, rows, c, k):
    x, w = _row8(1, (rows, c), device), _row8(2, (k, c), device)
    assert (M.row8_workspace_size(rows, rows, c, k) > 0) == M.plan_row8_linear(rows, c, k)[3] == (c % 16 > 0)
    M.row8_linear(x, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = M.row8_linear(x, w, dtype=F32)
    for seed in range(3):
        x.codes.copy_(_codes(seed + 5, (rows, c), device))
        y.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, M.row8_linear(x, w, dtype=F32)) and torch.equal(y, _want(x, w, F32))


def test_a_workspace_of_the_callers_and_two_streams_at_once(device):
    x, w = _row8(1, (1030, 643), device), _row8(2, (2050, 643), device)
    size = M.row8_workspace_size(1030, 1030, 643, 2050)
    assert size == (1030 + 2050) * 640 + (1030 + 2050) * 128
    want = _want(x, w, BF16)
    own = [torch.empty(size, dtype=torch.uint8, device=device) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [M.row8_linear(x, w, workspace=ws, stream=s) for _ in range(10) for ws, s in zip(own, streams)]
    got += [M.row8_linear(x, w, stream=s) for _ in range(10) for s in streams]
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in got)
    with pytest.raises(M.MiqError, match="smaller"):
        M.row8_linear(x, w, workspace=own[0][:-16])
    offsets = torch.tensor([0, 1000, 1030], dtype=torch.int32, device=device)
    w2 = M.Row8(torch.stack([w.codes, w.codes]), torch.stack([w.scales, w.scales]))
    assert (M.row8_workspace_size(1030, 1030, 643, 2050, 2) > 0) == M.plan_row8_linear(1030, 643, 2050, 2)[3]
    assert torch.equal(M.row8_experts(x, w2, offsets), want)


@pytest.mark.parametrize("rows,c,k", [(5, 64, 33), (900, 1000, 520)])
def test_no_rows_to_take_from(device, rows, c, k):
    """An index into nothing: every row stands for zeros."""
    x, w = _row8(1, (0, c), device), _row8(2, (3, k, c), device)
    bias = torch.randn((3, k), device=device)
    offsets = torch.tensor([0, 2, 2, rows], dtype=torch.int32, device=device)
    index = torch.zeros(rows, dtype=torch.int32, device=device)
    got = M.row8_experts(x, w, offsets, rows=index, bias=bias, dtype=F32)
    want = torch.cat([bias[:1].expand(2, k), bias[2:].expand(rows - 2, k)])
    assert torch.equal(got, want)
    assert torch.equal(M.row8_experts(x, w, offsets, rows=index, dtype=BF16), torch.zeros((rows, k), dtype=BF16, device=device))


@pytest.mark.parametrize("n,c,k", [(40, 64, 33), (3000, 256, 520)])
def test_falling_offsets_stay_inside(device, n, c, k):
    """Offsets that fall: a range that would end before it starts is empty, none leaves the rows."""
    x, w = _row8(1, (n, c), device), _row8(2, (4, k, c), device)
    offsets = torch.tensor([n, 0, n // 2, 3, 3], dtype=torch.int32, device=device)
    wide = torch.full((n + 2, k), -7.0, dtype=F32, device=device)
    M.row8_experts(x, w, offsets, out=wide[1:-1])
    want = torch.full((n + 2, k), -7.0, device=device)
    want[1: 1 + n // 2] = _want(x, M.Row8(w.codes[1], w.scales[1]), F32)[: n // 2]
    assert torch.equal(wide, want)


def test_more_tiles_than_a_launch(device):
    """2^28 rows: both kernels take more than one round of their largest grid."""
    for rows, c, k in [((1 << 28) + 70, 16, 16), ((1 << 28) + 70, 144, 16)]:
        x = torch.zeros((rows, c), dtype=torch.int8, device=device)
        last = _codes(3, (200, c), device)
        x[-200:] = last
        x[(1 << 27) - 3: (1 << 27) + 197] = last
        scales = torch.ones(rows, device=device)
        w = _row8(2, (k, c), device)
        y = M.row8_linear(M.Row8(x, scales), w)
        want = M.row8_linear(M.Row8(last, scales[:200]), w)
        assert torch.equal(y[-200:], want) and torch.equal(y[(1 << 27) - 3: (1 << 27) + 197], want)
        assert not bool(y[:1000].any()) and not bool(y[-1200:-200].any())
        del x, y


def test_a_token_that_names_an_expert_twice(device):
    ids = torch.tensor([[1, 1], [0, 1], [1, 0]], dtype=torch.int32, device=device)
    plan = M.experts_plan(ids, 2)
    assert plan.offsets.tolist() == [0, 2, 6] and plan.rows.tolist() == [1, 2, 0, 0, 1, 2]
    assert plan.places.tolist() == [[2, 3], [0, 4], [5, 1]]
    x, w = _row8(1, (3, 64), device), _row8(2, (2, 20, 64), device)
    share = torch.tensor([[0.25, 0.5], [1.0, 2.0], [0.5, 0.5]], device=device)
    y = M.experts_join(M.row8_experts(x, w, plan.offsets, rows=plan.rows, dtype=F32), plan.places, share)
    of = [_want(x, M.Row8(w.codes[e], w.scales[e]), F32) for e in range(2)]
    want = torch.stack([of[1][0] * 0.25 + of[1][0] * 0.5, of[0][1] + of[1][1] * 2, of[1][2] * 0.5 + of[0][2] * 0.5])
    assert torch.equal(y, want)


def test_refusals(device):
    x, gain = torch.zeros((3, 8), device=device), torch.ones(8, device=device)
    kept = M.act_row8(x)
    w, ws = M.Row8(kept.codes, kept.scales), M.Row8(kept.codes[None], kept.scales[None])
    offsets = torch.zeros(2, dtype=torch.int32, device=device)
    ids = torch.zeros((3, 2), dtype=torch.int32, device=device)
    refused = [
        (lambda: M.rms_fprop(x.half(), gain), "float32 or bfloat16"),
        (lambda: M.rms_fprop(x, gain[:7]), "gain must be"),
        (lambda: M.rms_fprop(x, gain, add=x[:2]), "add must be"),
        (lambda: M.rms_fprop(x, gain, add=x.bfloat16()), "add must be"),
        (lambda: M.rms_fprop(x, gain, total=x), "total needs add"),
        (lambda: M.rms_fprop(x.t(), gain), "dense"),
        (lambda: M.rms_fprop(x, gain, out=x[:, :4]), "out must be"),
        (lambda: M.rms_row8(x, gain, kept=M.Row8(kept.codes[:2], kept.scales[:2])), "kept must hold"),
        (lambda: M.rms_bprop(x[:2], x, gain), "dy must be"),
        (lambda: M.rms_bprop(x, x, gain, dsum=x.bfloat16()), "dsum must be"),
        (lambda: M.rms_bprop(x, x, gain, accumulate=True), "accumulate needs"),
        (lambda: M.rms_bprop(x, x, gain, dgain=gain, dtype=BF16), "dgain must be"),
        (lambda: M.act_row8(x, "tanh"), "act must be"),
        (lambda: M.act_row8(x[:, :7], gated=True), "even"),
        (lambda: M.row8_expand(M.Row8(kept.codes, kept.scales[:2])), "scales must be"),
        (lambda: M.row8_expand(M.Row8(kept.codes.int(), kept.scales)), "int8"),
        (lambda: M.row8_expand(kept, dtype=torch.float16), "float32 or bfloat16"),
        (lambda: M.row8_linear(kept, M.Row8(kept.codes[:, :4].contiguous(), kept.scales)), "w must be"),
        (lambda: M.row8_linear(kept, ws), "w must be"),
        (lambda: M.row8_linear(M.Row8(kept.codes.t(), gain), w), "contiguous"),
        (lambda: M.row8_linear(kept, w, bias=gain), "bias must be"),
        (lambda: M.row8_linear(kept, w, bias=kept.scales.bfloat16()), "contiguous torch.float32"),
        (lambda: M.row8_linear(kept, w, add=x), "add must be"),
        (lambda: M.row8_experts(kept, w, offsets), "w must be"),
        (lambda: M.row8_experts(kept, ws, offsets[:1]), "offsets must be"),
        (lambda: M.row8_experts(kept, ws, offsets.long()), "int32"),
        (lambda: M.row8_experts(kept, ws, offsets, rows=ids), "one dimension"),
        (lambda: M.experts_plan(ids.float(), 2), "int32 or int64"),
        (lambda: M.experts_plan(ids, 0), "at least 1"),
        (lambda: M.experts_plan(ids[None], 2), "tokens"),
        (lambda: M.experts_join(x, ids.long()), "int32"),
        (lambda: M.experts_join(x, ids, x), "share must be"),
        (lambda: M.experts_join(x, ids, add=x[:2]), "add must be"),
    ]
    for call, text in refused:
        with pytest.raises(ValueError, match=text):
            call()
    with pytest.raises(M.MiqError, match="eps"):
        M.rms_fprop(x, gain, eps=0.0)
    with pytest.raises(M.MiqError, match="4096"):
        M.experts_plan(ids, 4097)
