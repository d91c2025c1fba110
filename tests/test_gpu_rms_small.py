"""8-bit rows of norms at the ends of fp32 (miq_rms_row8): the definition takes the row's largest magnitude, held
to 2^-110 from below, of the norm itself, whatever s, gain and eps it comes from.

With u = 2^-24 the root is within (c / 2048 + 40) u; codes are the quotient of values with the same root, so
half a step and 127 * 6 u, besides the root's where the largest is held to 2^-110.  A magnitude below the
normal numbers may read zero: 2^-126 of a norm's own, or of s times 2^-80 where squares overflow, which is
2^-126 * 2^80 * r * gain of it; that shifts a code by 127 / m times as much."""
import numpy as np
import pytest
import torch

import my_own_cnn_amd as M

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24
LEAST = 2.0 ** -110
SIZES = [0.0, 1e-36, 5e-36, 1e-34, 1e-30, 1e-20, 1e-15, 1e-3, 1.0, 1e15, 1e18, 3e19, 1e30, 1e37]


@pytest.mark.parametrize("c", [5, 100, 700, 1500, 3000, 12001, 20000])
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("gain_size", [1.0, 1e-20, 1e-30, 1e-36, 1e21, 3e38])
@pytest.mark.parametrize("added", [False, True])
def test_codes_are_of_the_norm(device, c, kind, gain_size, added):
    g = torch.Generator().manual_seed(c)
    x = torch.zeros((len(SIZES), c))
    x[:, :5] = torch.randn((5,), generator=g) * torch.tensor(SIZES)[:, None]
    x = x.to(kind)
    gain = torch.full((c,), gain_size)
    s, g64 = x.double().numpy(), gain.double().numpy()
    for eps in (1e-6, 1e-30):
        eps = float(np.float32(eps))
        r = 1 / np.sqrt((s ** 2).mean(1, keepdims=True) + eps)
        want = s * r * g64
        top = np.abs(want).max(1)
        m = np.maximum(top, LEAST)
        kept = M.rms_row8(x.to(device), gain.to(device), eps=eps, add=torch.zeros_like(x).to(device) if added else None)
        kept = kept[0] if added else kept
        codes, scales = kept.codes.cpu().double().numpy(), kept.scales.cpu().double().numpy()
        over = top > 3.5e38  # the norm leaves fp32: the row stands for NaN
        assert np.isnan(scales[over]).all() and (codes[over] == 0).all()
        fine = top < 3.3e38
        assert (fine | over).all()
        root = (c / 2048 + 40) * U
        lost = 2.0 ** -126 * (1 + g64[0] * (1 + r[:, 0] * 2.0 ** 80 * (np.abs(s).max(1) > 1e17))) * (top > 0)
        near = 0.5 + 127 * (6 * U + root * (top < 1.01 * LEAST) + lost / m)[:, None]
        assert (np.abs(codes - want * (127 / m)[:, None]) <= near)[fine].all()
        assert (np.abs(scales - m / 127) <= (root + 4 * U) * m / 127 + lost / 127)[fine].all()
        assert (scales[top < 0.99 * LEAST] == np.float32(LEAST) / np.float32(127)).all()


def test_small_rows_among_others(device):
    """The rule takes each row by itself: rows that share a wave or follow one another in a workgroup."""
    for rows, c in [(1500, 60), (1500, 130), (9, 2049), (70001, 40)]:
        g = torch.Generator(device=device).manual_seed(c)
        x = torch.randn((rows, c), generator=g, device=device)
        x *= torch.tensor([1.0, 1e-36, 0.0, 1e20, 1e-34], device=device)[torch.randint(5, (rows, 1), generator=g, device=device)]
        gain = 1 + 0.1 * torch.randn((c,), generator=g, device=device)
        kept = M.rms_row8(x, gain)
        want = x.double() / torch.sqrt(x.double().square().mean(1, keepdim=True) + float(np.float32(1e-6))) * gain.double()
        m = want.abs().amax(1).clamp(min=LEAST)
        root = (c / 2048 + 40) * U
        near = 0.5 + 127 * (6 * U + root + 2.0 ** -126 / m[:, None])
        assert bool(((kept.codes.double() - want * (127 / m)[:, None]).abs() <= near).all())
        assert bool(((kept.scales.double() - m / 127).abs() <= (root + 4 * U) * m / 127).all())
