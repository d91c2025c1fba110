"""The weight gradient from kept rows, term by term, on the main loop of every tile with and without a split
of the rows.

Each column of dy holds one value, at a row of its own, so every weight is one product.  An fp32 value of
24 significant bits goes through the matrix instructions as three bf16 pieces, whose products with a kept
value are exact (8 by 8 bits): two additions that round, by a whole unit at most (2^-23 of the result), the
first of them of pieces below 2^-7 of it.  So the error is below 4 * 2^-24 of the product, and a piece that
is lost, doubled or taken from another row or step is beyond it.  A bf16 value's product is exact."""
import pytest
import torch

import my_own_cnn_amd as M

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24


def _columns(seed, rows, k):
    """(row, value) of each column's one entry: every step of 32 rows, values of 24 bits, the last one set."""
    g = torch.Generator().manual_seed(seed)
    at = (torch.arange(k) % (rows // 32)) * 32 + torch.randint(0, 32, (k,), generator=g)
    d = (torch.randint(1 << 22, 1 << 23, (k,), generator=g) * 2 + 1).double()
    d = d * (torch.randint(0, 2, (k,), generator=g) * 2 - 1) * 2.0 ** torch.randint(-60, 20, (k,), generator=g).double()
    return at, d


@pytest.mark.parametrize("rows,c,k,plan,kind", [
    (224, 256, 256, (64, 1), F32), (224, 2048, 2048, (128, 1), F32), (224, 4096, 4096, (256, 1), F32),
    (1024, 512, 512, (64, 4), F32), (4096, 512, 512, (128, 16), F32), (4096, 2048, 2048, (256, 4), F32),
    (224, 256, 256, (64, 1), BF16), (224, 2048, 2048, (128, 1), BF16), (224, 4096, 4096, (256, 1), BF16),
    (2048, 512, 512, (64, 4), BF16), (4096, 2048, 1024, (128, 2), BF16), (4096, 2048, 2048, (256, 4), BF16),
])
def test_every_weight_is_one_product(device, rows, c, k, plan, kind):
    assert M.plan_act8_grad(rows, c, k, kind) == plan
    at, d = _columns(rows + k, rows, k)
    bits = d.float().view(torch.int32)
    assert torch.equal(d.float().double(), d) and bool(((bits & 1) == 1).all())
    # what the bound has to tell apart: the value without its third piece
    cut = (bits & ~0xFF).view(F32).double()
    assert int(((cut - d).abs() > 4 * U * d.abs()).sum()) > 0.9 * k
    dy = torch.zeros((rows, k))
    dy[at, torch.arange(k)] = d.float()
    dy = dy.to(kind).to(device)
    x = torch.randn((rows, c), generator=torch.Generator().manual_seed(c)).to(device)
    kept = M.act8_keep(x)
    got = M.act8_grad(dy, kept).double()
    value = dy[at.to(device), torch.arange(k, device=device)].double()
    want = value[:, None] * M.act8_expand(kept).double()[at.to(device)]
    if kind == BF16:
        assert torch.equal(got, want)
    else:
        assert bool(((got - want).abs() <= 4 * U * want.abs()).all())
