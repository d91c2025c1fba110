"""Every kernel and tile of the products of 8-bit rows, at rows that start on 16 bytes, on 4 and anywhere, with
ragged edges in every direction, bit for bit against exact integer sums (fp64 on the device holds them) and the
fp32 operations after them."""
import pytest
import torch

import my_own_cnn_amd as M

F32, BF16 = torch.float32, torch.bfloat16

# rows, c, k, experts and what the plan gives them: few rows?, a tile, rows copied first?  Few tiles and many.
CASES = [
    (3, 80, 50, 1, (True, 16, 16, False)),
    (3, 84, 50, 1, (True, 16, 16, False)),
    (3, 83, 50, 1, (True, 16, 16, False)),
    (3, 9, 50, 1, (True, 16, 16, False)),
    (5, 4112, 33, 4, (True, 16, 16, False)),
    (5, 64, 1033, 4, (True, 16, 32, False)),
    (1, 68, 4100, 1, (True, 16, 32, False)),
    (1, 67, 4101, 1, (True, 16, 32, False)),
    (100, 64, 520, 4, (True, 32, 16, False)),
    (20, 68, 2050, 1, (True, 32, 16, False)),
    (20, 67, 2051, 1, (True, 32, 16, False)),
    (200, 64, 520, 4, (True, 32, 32, False)),
    (20, 68, 4097, 1, (True, 32, 32, False)),
    (20, 67, 4100, 1, (True, 32, 32, False)),
    (130, 64, 1030, 4, (True, 64, 32, False)),
    (33, 68, 4100, 1, (True, 64, 32, False)),
    (33, 67, 4099, 1, (True, 64, 32, False)),
    (70, 336, 4100, 1, (False, 64, 64, False)),
    (400, 80, 2049, 3, (False, 64, 64, False)),
    (16400, 80, 70, 1, (False, 64, 64, False)),
    (64, 4112, 4099, 1, (False, 64, 64, False)),
    (8200, 80, 130, 1, (False, 64, 64, False)),
    (70, 339, 4100, 1, (False, 64, 64, False)),
    (64, 643, 4100, 3, (False, 64, 64, False)),
    (260, 2051, 1030, 1, (False, 64, 64, True)),
    (1030, 339, 4100, 1, (False, 64, 64, True)),
    (70, 80, 8200, 1, (False, 64, 128, False)),
    (1030, 1040, 2050, 1, (False, 128, 128, False)),
    (400, 80, 8199, 3, (False, 64, 128, False)),
    (70, 339, 8200, 1, (False, 64, 128, False)),
    (64, 339, 8200, 3, (False, 64, 128, False)),
    (1030, 2051, 1030, 1, (False, 64, 128, True)),
    (1003, 2051, 1537, 1, (False, 64, 128, True)),
    (4100, 643, 2050, 4, (False, 64, 128, True)),
    (16400, 336, 70, 1, (False, 128, 128, False)),
    (700, 80, 4100, 3, (False, 128, 128, False)),
    (700, 656, 2050, 1, (False, 64, 128, False)),
    (16400, 339, 70, 1, (False, 128, 128, False)),
    (200, 339, 8200, 3, (False, 128, 128, False)),
    (1030, 643, 2050, 1, (False, 128, 128, True)),
    (8200, 67, 6150, 4, (False, 128, 128, True)),
    (700, 80, 8200, 3, (False, 128, 256, False)),
    (1030, 80, 6151, 1, (False, 128, 256, False)),
    (700, 339, 8200, 3, (False, 128, 256, False)),
    (1030, 2051, 6150, 1, (False, 128, 256, True)),
    (4100, 67, 16400, 4, (False, 128, 256, True)),
    (700, 1040, 16397, 1, (False, 256, 256, False)),
    (2050, 1040, 6150, 4, (False, 256, 256, False)),
    (2050, 643, 6150, 1, (False, 256, 256, True)),
]


@pytest.mark.parametrize("rows,c,k,experts,plan", CASES)
def test_the_plan(rows, c, k, experts, plan):
    assert M.plan_row8_linear(rows, c, k, experts) == plan


def test_every_tile_is_among_them():
    plans = {c[4] for c in CASES}
    few = {(True, r, k, False) for r, k in ((16, 16), (16, 32), (32, 16), (32, 32), (64, 32))}
    tiles = {(False, r, k, p) for r, k in ((64, 64), (64, 128), (128, 128), (128, 256)) for p in (False, True)}
    assert plans == few | tiles | {(False, 256, 256, False), (False, 256, 256, True)}


def test_plans_of_nothing_and_refused():
    assert M.plan_row8_linear(0, 64, 64) == (False, 0, 0, False) == M.plan_row8_linear(64, 64, 0)
    assert M.plan_row8_linear(64, 0, 64)[0]
    with pytest.raises(M.MiqError, match="131071"):
        M.plan_row8_linear(1, 131072, 1)
    with pytest.raises(M.MiqError, match="4096"):
        M.plan_row8_linear(1, 1, 1, 4097)
    assert M.lib().miq_plan_row8_linear(1, 1, 1, 1, None) != 0


def _codes(g, *shape):
    return torch.randint(-128, 128, shape, generator=g, device="cuda", dtype=torch.int32).to(torch.int8)


def _want(x, w, xs, ws, bias, add, kind):
    y = (x.double() @ w.double().t().contiguous()).float() * xs[:, None] * ws
    y = y if bias is None else y + bias
    return (y if add is None else y + add.float()).to(kind)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,c,k,experts,plan", CASES)
@pytest.mark.parametrize("kind", [F32, BF16])
def test_products(device, rows, c, k, experts, plan, kind):
    g = torch.Generator(device=device).manual_seed(rows + c)
    x, w = _codes(g, rows, c), _codes(g, experts, k, c)
    xs, ws = torch.rand(rows, generator=g, device=device), torch.rand((experts, k), generator=g, device=device) + 0.01
    bias = torch.randn((experts, k), generator=g, device=device)
    add = torch.randn((rows, k), generator=g, device=device).to(kind)
    if experts == 1:
        one = M.Row8(w[0], ws[0])
        got = M.row8_linear(M.Row8(x, xs), one, dtype=kind)
        assert torch.equal(got, _want(x, w[0], xs, ws[0], None, None, kind))
        got = M.row8_linear(M.Row8(x, xs), one, bias=bias[0], add=add)
        assert torch.equal(got, _want(x, w[0], xs, ws[0], bias[0], add, kind))
        return
    cuts = torch.sort(torch.randint(0, rows + 1, (experts - 1,), generator=g, device=device)).values.tolist()
    cuts = [0] + cuts + [rows]
    offsets = torch.tensor(cuts, dtype=torch.int32, device=device)
    index = torch.randint(0, rows, (rows,), generator=g, device=device, dtype=torch.int32)
    for of, with_bias in ((None, True), (index, False)):
        got = M.row8_experts(M.Row8(x, xs), M.Row8(w, ws), offsets, rows=of, bias=bias if with_bias else None, dtype=kind)
        for e in range(experts):
            at = torch.arange(cuts[e], cuts[e + 1], device=device)
            src = at if of is None else of[at].long()
            want = _want(x[src], w[e], xs[src], ws[e], bias[e] if with_bias else None, None, kind)
            assert torch.equal(got[cuts[e]: cuts[e + 1]], want), (e, of is None)


@pytest.mark.gpu
@pytest.mark.parametrize("c,tile", [(144, 128), (656, 256)])
@pytest.mark.parametrize("kind", [F32, BF16])
def test_a_large_output(device, c, tile, kind):
    """One that is written past the caches; the last rows and channels of ragged tiles."""
    g = torch.Generator(device=device).manual_seed(5)
    rows, k = 16100, 8192
    assert M.plan_row8_linear(rows, c, k)[:3] == (False, tile, 256)
    x, w = _codes(g, rows, c), _codes(g, k, c)
    xs, ws = torch.rand(rows, generator=g, device=device), torch.rand(k, generator=g, device=device)
    got = M.row8_linear(M.Row8(x, xs), M.Row8(w, ws), dtype=kind)
    assert torch.equal(got, _want(x, w, xs, ws, None, None, kind))
