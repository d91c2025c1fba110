"""The embedding gradient on tables of more than 2^27 rows: every way to run it (no tokens, one launch,
ranked, three counting passes), compared on the device.  Values are small integers, whose sums are
exact in bf16, so results must be equal."""
import pytest
import torch

import my_own_cnn_amd as M

pytestmark = pytest.mark.gpu

ROWS = (1 << 27) + 33
BF16 = torch.bfloat16


@pytest.mark.parametrize("vocab", [1 << 27, ROWS, 1 << 28])
def test_no_tokens_zero_every_row(device, vocab):
    assert M.plan_embed_grad(vocab, 1, 0) == (0, 0) and M.embed_grad_workspace_size(vocab, 1, 0) == 0
    ids = torch.zeros(0, dtype=torch.int64, device=device)
    out = torch.full((vocab, 1), -7.0, dtype=BF16, device=device)
    M.embed_grad(torch.zeros((0, 1), dtype=BF16, device=device), ids, vocab, out=out)
    assert int(torch.count_nonzero(out)) == 0
    out.fill_(3)
    M.embed_grad(torch.zeros((0, 1), dtype=BF16, device=device), ids, vocab, out=out, accumulate=True)
    assert bool((out == 3).all())


@pytest.mark.parametrize("tokens,sorts", [(1, 0), (5, 0), (256, 0), (257, 1), (1024, 1), (9000, 6)])
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_gradient_of_a_large_table(device, tokens, sorts, kind):
    assert M.plan_embed_grad(ROWS, 1, tokens)[0] == sorts
    g = torch.Generator().manual_seed(tokens)
    # a fifth on eight rows spread over the table's ends and powers of two, the rest anywhere
    some = torch.tensor([0, 1, 1 << 20, 1 << 26, (1 << 27) - 1, 1 << 27, ROWS - 2, ROWS - 1])
    ids = torch.randint(0, ROWS, (tokens,), generator=g)
    ids = torch.where(torch.rand((tokens,), generator=g) < 0.2, some[torch.randint(0, 8, (tokens,), generator=g)], ids)
    ids = torch.where(torch.rand((tokens,), generator=g) < 0.1, torch.tensor(ROWS), ids)  # outside the table
    ids[0], ids[-1] = ROWS - 1, 0
    dy = torch.randint(-1, 2, (tokens, 1), generator=g)
    there = ids < ROWS
    rows, at = torch.unique(ids[there], return_inverse=True)
    sums = torch.zeros((rows.numel(), 1), dtype=torch.int64).index_add_(0, at, dy[there])
    assert int(sums.abs().max()) <= 256
    out = torch.full((ROWS, 1), -7.0, dtype=BF16, device=device)
    idd = ids.to(kind).to(device)
    M.embed_grad(dy.to(BF16).to(device), idd, ROWS, out=out)
    assert torch.equal(out[rows.to(device)].cpu(), sums.to(BF16))
    assert int(torch.count_nonzero(out)) == int(torch.count_nonzero(sums))
    out.fill_(5)
    M.embed_grad(dy.to(BF16).to(device), idd, ROWS, out=out, accumulate=True)
    assert torch.equal(out[rows.to(device)].cpu(), (sums + 5).to(BF16))
    assert int(torch.count_nonzero(out - 5)) == int(torch.count_nonzero(sums))
