"""The embedding table's lookup and gradient on the GPU (miq_embed_fprop, miq_embed_grad).

The lookup is one fp32 product per value, rounded once: equal to the plain product bit for bit.
The gradient is compared with sums in 64 bits.  A row of n tokens is n - 1 fp32 additions in some
order and one product, each off by at most 2^-24 of a partial sum that is at most the row's sum of
magnitudes S: n * 2^-24 * S; a bf16 table holds the rounding of a value within that.  Integer inputs make
every partial sum exact, so there the result must be equal whatever the order."""
import numpy as np
import pytest
import torch

import my_own_cnn_amd as M

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
IDS = {"i32": torch.int32, "i64": torch.int64}


def _ids(seed, tokens, vocab, how):
    rng = np.random.default_rng(seed)
    if how == "same":
        ids = np.full(tokens, vocab // 2)
    elif how == "none":
        ids = np.where(rng.random(tokens) < 0.5, -1, vocab)
    elif how == "skewed":  # as words are: a few rows take most tokens
        ids = np.minimum(np.exp(rng.random(tokens) * np.log(vocab + 1)).astype(np.int64) - 1, vocab - 1)
        ids = np.where(rng.random(tokens) < 0.1, rng.choice([-1, vocab, vocab + 7, -2 ** 31], tokens), ids)
    else:
        ids = rng.integers(0, vocab, tokens)
    return ids.astype(np.int64)


# ---- lookup ----------------------------------------------------------------------------------

@pytest.mark.parametrize("tokens,vocab,c", [(1, 1, 1), (3, 5, 7), (65, 11, 8), (17, 40, 63), (130, 64, 64), (33, 100, 257),
                                            (9, 30, 1001), (5, 9, 2048), (4, 6, 2052), (1000, 3, 16)])
@pytest.mark.parametrize("table_type,out_type", [(F32, F32), (F32, BF16), (BF16, BF16), (BF16, F32)])
def test_lookup_is_the_scaled_row(device, tokens, vocab, c, table_type, out_type):
    g = torch.Generator().manual_seed(tokens * 7 + c)
    table = torch.randn((vocab, c), generator=g).to(table_type)
    for kind in ("i32", "i64"):
        ids = torch.from_numpy(_ids(tokens + c, tokens, vocab, "skewed")).to(IDS[kind])
        got = M.embed_fprop(table.to(device), ids.to(device), scale=1.7, dtype=out_type).cpu()
        there = (ids >= 0) & (ids < vocab)
        want = table[torch.where(there, ids, 0).long()].float() * torch.tensor(1.7, dtype=F32)
        want = torch.where(there[:, None], want, torch.zeros(())).to(out_type)
        assert got.dtype == out_type and torch.equal(got, want)


@pytest.mark.parametrize("kind", [F32, BF16])
def test_lookup_of_row_slices_shapes_and_no_tokens(device, kind):
    g = torch.Generator().manual_seed(3)
    wide = torch.randn((50, 41), generator=g).to(kind).to(device)
    table = wide[:, 3:36]  # rows 41 apart, every alignment
    ids = torch.randint(0, 50, (2, 3, 5), generator=g).to(device)
    into = torch.full((2, 3, 5, 49), -7.0, dtype=kind, device=device)
    got = M.embed_fprop(table, ids, out=into[..., 5:38])
    assert torch.equal(got, table[ids])
    assert (into[..., :5] == -7).all() and (into[..., 38:] == -7).all()
    assert M.embed_fprop(table, ids[:0]).shape == (0, 3, 5, 33)
    empty = torch.empty((0, 9), dtype=kind, device=device)
    assert (M.embed_fprop(empty, ids) == 0).all()


def test_lookup_carries_infinities_and_nan(device):
    table = torch.tensor([[float("inf"), -0.0, float("nan")], [1.0, 2.0, 3.0]], device=device)
    got = M.embed_fprop(table, torch.tensor([0, -1, 1], device=device), scale=2.0).cpu().numpy()
    np.testing.assert_array_equal(got, np.array([[np.inf, -0.0, np.nan], [0, 0, 0], [2, 4, 6]], np.float32))


# ---- gradient ----------------------------------------------------------------------------------

def _want(dy, ids, vocab):
    """(sums in 64 bits, sums of magnitudes, tokens per row)"""
    sums, mags = np.zeros((vocab, dy.shape[1])), np.zeros((vocab, dy.shape[1]))
    there = (ids >= 0) & (ids < vocab)
    np.add.at(sums, ids[there], dy[there])
    np.add.at(mags, ids[there], np.abs(dy[there]))
    return sums, mags, np.bincount(ids[there], minlength=vocab)


GRADS = [  # tokens, vocab, c, how the ids fall
    (1, 1, 1, "even"), (1, 9, 5, "even"), (2, 3, 8, "same"), (5, 2, 64, "even"), (63, 50, 7, "skewed"),
    (64, 64, 65, "skewed"), (65, 1000, 32, "even"), (300, 3, 513, "even"), (257, 40, 1001, "skewed"),
    (4096, 5000, 24, "skewed"), (8191, 100, 16, "skewed"), (8192, 70000, 8, "even"), (8193, 300, 16, "skewed"),
    (8193, 5, 512, "same"), (20000, 50021, 40, "skewed"), (20011, 1, 33, "even"), (40000, 1 << 21, 8, "skewed"),
    (256, 300, 16, "same"), (1024, 7, 512, "same"), (1024, 60000, 4, "even"), (1000, 90, 1024, "skewed"),
    (682, 50, 1536, "skewed"), (683, 50, 1536, "skewed"), (1025, 90, 72, "skewed"), (1024, 9, 1, "none"),
    (600, 70, 48, "none"), (9000, 70, 48, "none"), (100000, 1030, 64, "skewed"),
]


@pytest.mark.parametrize("tokens,vocab,c,how", GRADS)
@pytest.mark.parametrize("dy_type,out_type", [(F32, F32), (BF16, F32), (BF16, BF16)])
def test_gradient_against_64_bits(device, tokens, vocab, c, how, dy_type, out_type):
    ids = _ids(tokens + vocab, tokens, vocab, how)
    g = torch.Generator().manual_seed(tokens + c)
    dy = torch.randn((tokens, c), generator=g).to(dy_type)
    scale = 0.75
    sums, mags, n = _want(dy.double().numpy(), ids, vocab)
    kind = torch.int32 if tokens % 2 and how != "skewed" else torch.int64
    args = dy.to(device), torch.from_numpy(ids).to(kind).to(device), vocab
    got = M.embed_grad(*args, scale=scale, dtype=out_type)
    again = M.embed_grad(*args, scale=scale, dtype=out_type)
    assert torch.equal(got, again)  # the same bits every time
    got = got.cpu().double().numpy()
    bound = n[:, None] * 2.0 ** -24 * mags * scale
    low, high = sums * scale - bound, sums * scale + bound
    if out_type == BF16:
        low, high = (torch.from_numpy(v).float().bfloat16().double().numpy() for v in (low, high))
    assert (got >= low).all() and (got <= high).all()
    assert (got[n == 0] == 0).all()


@pytest.mark.parametrize("tokens,vocab,c,how", [(700, 90, 72, "skewed"), (5000, 11, 520, "skewed"), (30000, 4000, 24, "skewed"),
                                                (12000, 30, 8, "same")])
def test_gradient_of_integers_is_exact_and_accumulates(device, tokens, vocab, c, how):
    ids = _ids(tokens, tokens, vocab, how)
    dy = np.random.default_rng(c).integers(-3, 4, (tokens, c)).astype(np.float64)
    sums, _, n = _want(dy, ids, vocab)
    dyd, idd = torch.from_numpy(dy).float().to(device), torch.from_numpy(ids).to(device)
    got = M.embed_grad(dyd, idd, vocab, scale=2.0)
    np.testing.assert_array_equal(got.cpu().numpy(), 2 * sums)
    # rows without a token keep what they hold, NaN too
    start = torch.full((vocab, c), 5.0, device=device)
    start[torch.from_numpy(n == 0).to(device)] = float("nan")
    out = M.embed_grad(dyd, idd, vocab, accumulate=True, out=start)
    want = np.where((n == 0)[:, None], np.nan, 5 + sums)
    np.testing.assert_array_equal(out.cpu().numpy(), want)


@pytest.mark.parametrize("kind", [F32, BF16])
def test_gradient_of_row_slices_and_no_tokens(device, kind):
    rng = np.random.default_rng(9)
    dy = torch.from_numpy(rng.integers(-3, 4, (4, 25, 51)).astype(np.float32)).to(kind).to(device)[..., 7:40]
    ids = torch.from_numpy(rng.integers(0, 20, (4, 25))).to(device)
    into = torch.full((20, 41), -7.0, dtype=kind, device=device)
    M.embed_grad(dy, ids, 20, out=into[:, 5:38])
    want, _, _ = _want(dy.cpu().double().numpy().reshape(100, 33), ids.cpu().numpy().reshape(-1), 20)
    np.testing.assert_array_equal(into[:, 5:38].cpu().double().numpy(), want)
    M.embed_grad(dy, ids, 20, out=into[:, 5:38], accumulate=True)  # sums of integers: exact in bf16 to 256
    np.testing.assert_array_equal(into[:, 5:38].cpu().double().numpy(), 2 * want)
    assert (into[:, :5] == -7).all() and (into[:, 38:] == -7).all()
    none = M.embed_grad(dy[:0], ids[:0], 20)
    assert none.shape == (20, 33) and (none == 0).all()
    kept = torch.full((20, 33), 3.0, device=device)
    assert (M.embed_grad(dy[:0], ids[:0], 20, accumulate=True, out=kept) == 3).all()


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("tokens,c", [(1500, 33), (1500, 1030), (9000, 33)])
def test_sorted_gradient_of_row_slices_with_nan_where_no_token_is(device, kind, tokens, c):
    rng = np.random.default_rng(tokens + c)
    ids = rng.integers(-300, 600, tokens)  # a third without a token
    values = rng.integers(-2, 3, (tokens, c + 9)).astype(np.float32)
    values[ids < 0] = np.nan
    dy = torch.from_numpy(values).to(kind).to(device)[:, 7:7 + c]
    idd = torch.from_numpy(ids).to(device)
    into = torch.full((600, c + 4), -7.0, dtype=kind, device=device)
    out = into[:, 3:3 + c]
    M.embed_grad(dy, idd, 600, out=out)
    want, _, _ = _want(np.nan_to_num(values[:, 7:7 + c]).astype(np.float64), ids, 600)
    np.testing.assert_array_equal(out.cpu().double().numpy(), want)
    M.embed_grad(dy, idd, 600, out=out, accumulate=True)  # sums of integers: exact in bf16 to 256
    np.testing.assert_array_equal(out.cpu().double().numpy(), 2 * want)
    assert (into[:, :3] == -7).all() and (into[:, 3 + c:] == -7).all()


def test_gradient_rows_beyond_32_bit_offsets(device):
    tokens, c = 70000, 32768  # 2.3e9 values of dy
    dy = torch.zeros((tokens, c), dtype=BF16, device=device)
    ids = torch.full((tokens,), -1, device=device)
    for t, row in [(0, 1), (65537, 3), (69998, 1), (69999, 4)]:
        dy[t] = torch.randint(-3, 4, (c,), device=device).to(BF16)
        ids[t] = row
    d = M.embed_grad(dy, ids, 6, dtype=BF16)
    assert torch.equal(d[1], dy[0] + dy[69998]) and torch.equal(d[3], dy[65537]) and torch.equal(d[4], dy[69999])
    assert (d[[0, 2, 5]] == 0).all()


def test_gradient_against_differences(device):
    """The lookup is linear in its table: with values of few bits its differences are exact."""
    rng = np.random.default_rng(4)
    vocab, c, tokens = 13, 9, 200
    table = torch.from_numpy(rng.integers(-8, 9, (vocab, c)).astype(np.float32)).to(device)
    ids = torch.from_numpy(_ids(1, tokens, vocab, "skewed")).to(device)
    dy = torch.from_numpy(rng.integers(-4, 5, (tokens, c)).astype(np.float32)).to(device)
    d = M.embed_grad(dy, ids, vocab, scale=0.5).cpu()

    def loss(t):
        return float((M.embed_fprop(t, ids, scale=0.5).double() * dy.double()).sum())

    for row, col in [(0, 0), (1, 8), (6, 4), (12, 3)]:
        up, down = table.clone(), table.clone()
        up[row, col] += 1
        down[row, col] -= 1
        assert (loss(up) - loss(down)) / 2 == float(d[row, col])


def test_infinite_and_nan_gradients_stay_in_their_rows(device):
    dy = torch.ones((6, 16), device=device)
    dy[1, 3], dy[4, 5] = float("inf"), float("nan")
    ids = torch.tensor([2, 0, 2, -1, 7, 0], device=device)
    got = M.embed_grad(dy, ids, 9).cpu().numpy()
    want = np.zeros((9, 16), np.float32)
    want[0], want[2], want[7] = 2, 2, 1
    want[0, 3], want[7, 5] = np.inf, np.nan
    np.testing.assert_array_equal(got, want)
    # a position without a token contributes nothing, whatever it holds
    dy[3] = float("nan")
    np.testing.assert_array_equal(M.embed_grad(dy, ids, 9).cpu().numpy(), want)


def test_table_beyond_32_bit_offsets(device):
    vocab, c = 70001, 32768  # 2.3e9 values
    ids = torch.tensor([0, 69999, 70000, 65536, 70000], device=device)
    dy = torch.randint(-3, 4, (5, c), device=device).to(BF16)
    d = M.embed_grad(dy, ids, vocab, dtype=BF16)
    assert torch.equal(d[70000], dy[2] + dy[4]) and torch.equal(d[69999], dy[1]) and torch.equal(d[65536], dy[3])
    assert (d[65537:69999] == 0).all() and (d[1:100] == 0).all()
    assert torch.equal(M.embed_fprop(d, ids[1:4]), torch.stack([dy[1], dy[2] + dy[4], dy[3]]))


@pytest.mark.parametrize("out_type", [F32, BF16])
def test_outputs_beyond_the_caches(device, out_type):
    table = torch.randn((500, 2048), device=device)
    ids = torch.randint(-3, 500, (40000,), device=device)
    got = M.embed_fprop(table, ids, scale=3.0, dtype=out_type)  # 328 and 164 MB
    want = torch.where((ids >= 0)[:, None], table[ids.clamp(min=0)] * 3.0, torch.zeros((), device=device))
    assert torch.equal(got, want.to(out_type))


def test_other_stream_and_graph_replays(device):
    rng = np.random.default_rng(6)
    vocab, c, tokens = 500, 40, 9000
    dy = torch.from_numpy(rng.integers(-3, 4, (tokens, c)).astype(np.float32)).to(device)
    ids = torch.from_numpy(_ids(2, tokens, vocab, "skewed")).to(device)
    want = M.embed_grad(dy, ids, vocab)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = M.embed_grad(dy, ids, vocab, stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    ws = torch.empty(M.embed_grad_workspace_size(vocab, c, tokens), dtype=torch.uint8, device=device)
    out = torch.empty((vocab, c), device=device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        M.embed_grad(dy, ids, vocab, out=out, workspace=ws)
    for seed in range(4):
        ids.copy_(torch.from_numpy(_ids(10 + seed, tokens, vocab, "skewed")).to(device))
        out.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, M.embed_grad(dy, ids, vocab))


def test_refusals(device):
    table = torch.zeros((4, 8), device=device)
    ids = torch.zeros(3, dtype=torch.int64, device=device)
    dy = torch.zeros((3, 8), device=device)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        M.embed_fprop(table.half(), ids)
    with pytest.raises(ValueError, match="int32 or int64"):
        M.embed_fprop(table, ids.short())
    with pytest.raises(ValueError, match="channels must be dense"):
        M.embed_fprop(table.t(), ids)
    with pytest.raises(ValueError, match="device memory"):
        M.embed_fprop(table, ids.cpu())
    with pytest.raises(ValueError, match="out must be"):
        M.embed_fprop(table, ids, out=torch.empty((3, 7), device=device))
    with pytest.raises(ValueError, match="must not overlap"):
        M.embed_grad(dy[:1].expand(3, 8), ids, 4)
    with pytest.raises(ValueError, match="accumulate needs out"):
        M.embed_grad(dy, ids, 4, accumulate=True)
    with pytest.raises(ValueError, match="ids.shape"):
        M.embed_grad(dy[:2], ids, 4)
    dy, ids = torch.zeros((2000, 8), device=device), torch.zeros(2000, dtype=torch.int64, device=device)
    with pytest.raises(M.MiqError, match="workspace is smaller"):
        M.embed_grad(dy, ids, 4, workspace=torch.empty(16, dtype=torch.uint8, device=device))
