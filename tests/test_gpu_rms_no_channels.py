"""8-bit rows without channels: codes are empty, and each row has the least scale, as act_row8 gives it."""
import numpy as np
import pytest
import torch

import my_own_cnn_amd as M

pytestmark = pytest.mark.gpu

LEAST = float(np.float32(2.0 ** -110) / np.float32(127))


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lead", [(4,), (2, 3), ()])
def test_rows_of_nothing_have_a_scale(device, kind, lead):
    x, gain = torch.zeros(lead + (0,), dtype=kind, device=device), torch.ones(0, device=device)
    kept = M.Row8(torch.zeros(lead + (0,), dtype=torch.int8, device=device), torch.full(lead, float("nan"), device=device))
    got = M.rms_row8(x, gain, kept=kept)
    assert got.scales is kept.scales and got.scales.shape == lead and bool((got.scales == LEAST).all())
    kept.scales.fill_(float("nan"))
    got, total = M.rms_row8(x, gain, add=x, kept=kept)
    assert total.shape == x.shape and bool((got.scales == LEAST).all())
    side = torch.cuda.Stream()
    kept.scales.fill_(float("nan"))
    torch.cuda.synchronize()
    M.rms_row8(x, gain, kept=kept, stream=side)
    side.synchronize()
    assert bool((kept.scales == LEAST).all())
    assert torch.equal(M.act_row8(x).scales, kept.scales)
    w = M.Row8(torch.zeros((5, 0), dtype=torch.int8, device=device), torch.ones(5, device=device))
    bias = torch.randn(5, device=device)
    assert torch.equal(M.row8_linear(got, w, bias=bias, dtype=torch.float32), bias.expand(lead + (5,)))
