"""The norm's backward pass on more rows than its workgroups take at once (miq_rms_bprop): the values loaded
ahead, both turns of the sums and dgain's terms over several rows of a workgroup, in every form of the
kernel.  Against the definition in 64 bits, with u = 2^-24:
  - dx: a sum of c products, c / 1024 + 60 additions one after another, three operations on each; the root's
    half of as much; the operations around them: (c / 512 + 150) u of the sum of magnitudes, as for few rows;
  - dgain: at most as many additions one after another as a workgroup has rows, its 16 rows at once, and the
    parts in 32 threads: (rows / parts + 16 + parts / 32 + 32) u of the sum of magnitudes, besides the root's
    (c / 2048 + 40) u and 4 u for the product's operations.
A bf16 dx is the rounding of a value within these bounds, 2^-8 of it."""
import pytest
import torch

import my_own_cnn_amd as M

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24

# a quarter, a half and all of a wave, in one to four runs; four waves; sixteen; rows read again
FORMS = [(30011, 64), (20003, 200), (9001, 257), (6007, 500), (5003, 1001), (6001, 1000), (3001, 1500), (2053, 2048),
         (1601, 2500), (1301, 4096), (1283, 5000), (1031, 8191), (557, 12001), (523, 16384), (521, 17001), (517, 20001)]


@pytest.mark.parametrize("rows,c", FORMS)
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("more", [False, True])
def test_rows_after_a_workgroups_first(device, rows, c, kind, more):
    g = torch.Generator(device=device).manual_seed(rows + c)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=device)

    x, dy, gain = normal(rows, c).to(kind), normal(rows, c).to(kind), 1 + 0.2 * normal(c)
    dsum = normal(rows, c).to(kind) if more else None
    parts = M.rms_bprop_workspace_size(rows, c) // (4 * c)
    assert rows > (16 if c < 256 else 4 if c < 1025 else 2) * parts  # rows that a workgroup takes at once
    dx, dgain = M.rms_bprop(dy, x, gain, dsum=dsum)

    s, d = x.double(), dy.double()
    r = 1 / torch.sqrt(s.square().mean(1, keepdim=True) + 1e-6)
    n, dn = s * r, d * gain.double()
    want = r * (dn - n * (dn * n).mean(1, keepdim=True))
    size = r * (dn.abs() + n.abs() * (dn * n).abs().mean(1, keepdim=True))
    if more:
        want, size = want + dsum.double(), size + dsum.double().abs()
    off = (c / 512 + 150) * U * size
    half = 2.0 ** -8 if kind == BF16 else U
    assert bool(((dx.double() - want).abs() <= off + half * (want.abs() + off)).all())
    terms = (d * n).abs().sum(0)
    off = (rows / parts + 16 + parts / 32 + 32 + c / 2048 + 44) * U * terms
    assert bool(((dgain.double() - (d * n).sum(0)).abs() <= off).all())
    again = M.rms_bprop(dy, x, gain, dsum=dsum)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dgain)
