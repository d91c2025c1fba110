"""Forms of the token-network operators' calls: row slices of bf16 tensors, other streams, graphs of the
unsorted table gradient, bf16 tables' gradients from fp32 rows, sums added to bf16 weights.  Each is
compared with the plain call on contiguous tensors (tested against 64 bits elsewhere), bit for bit, or
with exact integers."""
import pytest
import torch

import my_own_cnn_amd as M

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _slice(t, before, after):
    """t, held as a slice of wider rows: (the slice, the whole tensor filled with -7 around it)."""
    wide = torch.full(t.shape[:-1] + (before + t.shape[-1] + after,), -7.0, dtype=t.dtype, device=t.device)
    part = wide[..., before: before + t.shape[-1]]
    part.copy_(t)
    return part, wide


def _around(part, wide, before):
    width = part.shape[-1]
    return bool((wide[..., :before] == -7).all() and (wide[..., before + width:] == -7).all())


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("c", [1, 7, 33, 64, 100, 1003])
def test_act8_of_row_slices(device, kind, gated, c):
    g = torch.Generator().manual_seed(c)
    width = 2 * c if gated else c
    x = torch.randn((3, 5, width), generator=g).to(kind).to(device)
    dy = torch.randn((3, 5, c), generator=g).to(kind).to(device)
    y, kept = M.act8_fprop(x, "gelu", gated=gated)
    dx, again = M.act8_bprop(dy, kept), M.act8_expand(kept, apply=True, dtype=kind)
    for before, after in [(1, 0), (3, 2), (8, 9)]:
        xs, ds = _slice(x, before, after)[0], _slice(dy, after + 1, before)[0]
        out, wide = _slice(torch.zeros_like(y), before, after)
        ys, ks = M.act8_fprop(xs, "gelu", gated=gated, out=out)
        assert torch.equal(ys, y) and torch.equal(ks.codes, kept.codes) and torch.equal(ks.scales, kept.scales)
        assert _around(out, wide, before)
        out, wide = _slice(torch.zeros_like(dx), after, before + 1)
        assert torch.equal(M.act8_bprop(ds, kept, out=out), dx) and _around(out, wide, after)
        out, wide = _slice(torch.zeros_like(y), before, after)
        assert torch.equal(M.act8_expand(kept, apply=True, out=out), again) and _around(out, wide, before)
        if not gated:
            ks = M.act8_keep(xs)
            assert torch.equal(ks.codes, kept.codes) and torch.equal(ks.scales, kept.scales)


@pytest.mark.parametrize("kind", [F32, BF16])
def test_act8_and_lookup_on_another_stream(device, kind):
    g = torch.Generator().manual_seed(4)
    x = torch.randn((700, 2 * 300), generator=g).to(kind).to(device)
    dy = torch.randn((700, 300), generator=g).to(kind).to(device)
    ids = torch.randint(-2, 700, (900,), generator=g).to(device)

    def calls(**on):
        y, kept = M.act8_fprop(x, "silu", gated=True, **on)
        only = M.act8_keep(dy, **on)
        return [y, kept.codes, kept.scales, M.act8_bprop(dy, kept, **on), M.act8_expand(kept, apply=True, **on),
                only.codes, only.scales, M.act8_expand(only, dtype=kind, **on), M.embed_fprop(x, ids, scale=3.0, **on),
                M.embed_grad(M.embed_fprop(dy, ids, **on), ids, 700, **on)]

    want = calls()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = calls(stream=side)
    side.synchronize()
    for i, (a, b) in enumerate(zip(got, want)):
        assert torch.equal(a, b), i


@pytest.mark.parametrize("tokens,vocab,c", [(3, 5, 3), (200, 50, 130), (1000, 90, 33), (5000, 300, 520), (20000, 1100, 65)])
def test_bf16_table_gradient_of_fp32_rows(device, tokens, vocab, c):
    """The sums are the fp32 table's, in the same order, rounded once."""
    g = torch.Generator().manual_seed(tokens)
    dy = torch.randn((tokens, c), generator=g).to(device)
    ids = torch.randint(-vocab // 4, vocab, (tokens,), generator=g).to(device)
    want = M.embed_grad(dy, ids, vocab, scale=0.75)
    assert torch.equal(M.embed_grad(dy, ids, vocab, scale=0.75, dtype=BF16), want.to(BF16))


@pytest.mark.parametrize("tokens", [200, 1000])
def test_unsorted_gradient_in_a_graph(device, tokens):
    vocab, c = 300, 130
    assert M.plan_embed_grad(vocab, c, tokens) == (0, 0)
    dy = torch.zeros((tokens, c), device=device)
    ids = torch.zeros(tokens, dtype=torch.int64, device=device)
    out = torch.empty((vocab, c), device=device)
    M.embed_grad(dy, ids, vocab, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        M.embed_grad(dy, ids, vocab, out=out)
    for seed in range(4):
        g = torch.Generator().manual_seed(seed)
        dy.copy_(torch.randn((tokens, c), generator=g))
        ids.copy_(torch.randint(-20, vocab + 20, (tokens,), generator=g) // (seed + 1))
        out.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, M.embed_grad(dy, ids, vocab))


@pytest.mark.parametrize("rows,c,k,split", [(40, 96, 33, False), (224, 2048, 2048, False), (2048, 512, 512, True)])
def test_weight_gradient_added_to_bf16(device, rows, c, k, split):
    """One product of small integers per weight, added to 5: at most 3 * 64 + 5, exact in bf16."""
    assert (M.plan_act8_grad(rows, c, k, BF16)[1] > 1) == split
    g = torch.Generator().manual_seed(rows)
    x = torch.randint(-3, 4, (rows, c), generator=g).float()
    x[:, ::32] = 64  # steps of 1: integers are kept as they are
    at = torch.randint(0, rows, (k,), generator=g)
    d = torch.randint(-3, 4, (k,), generator=g).float()
    dy = torch.zeros((rows, k))
    dy[at, torch.arange(k)] = d
    dw, wide = _slice(torch.full((k, c), 5.0, dtype=BF16, device=device), 3, 2)
    M.act8_grad(dy.to(BF16).to(device), M.act8_keep(x.to(device)), accumulate=True, out=dw)
    assert torch.equal(dw.cpu().float(), 5 + d[:, None] * x[at]) and _around(dw, wide, 3)
