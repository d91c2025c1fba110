"""The norm's backward pass where the products dy * gain * x of a row, or their sum, leave fp32 and the gradients do
not (miq_rms_bprop).  Against the definition in 64 bits, within the bounds of ordinary rows: (c / 512 + 150) u of
the sum of magnitudes, u = 2^-24, dgain's three additions and the root's (c / 2048 + 150) u of its terms' magnitudes; a
value below the normal numbers may read zero before it is multiplied by the root: 2^-126 (1 + r)."""
import numpy as np
import pytest
import torch

import my_own_cnn_amd as M

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24


@pytest.mark.parametrize("c", [5, 100, 700, 1500, 3000, 6000, 12001, 20000])
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("x_size,dy_size", [(1e-15, 1e-30), (1e-15, 1e20), (1e-3, 1e-30), (1.0, 1e-28), (1.0, 1e36), (1e5, 1e35),
                                            (1e10, 1e30), (1e15, 1e25), (1e18, 1e21), (1e18, 1e36), (1e25, 1e36),
                                            (1e37, 1e36), (1e37, 1.0), (1.0, 0.0), (0.0, 1e30)])
def test_products_that_leave_fp32(device, c, kind, x_size, dy_size):
    g = torch.Generator().manual_seed(c)
    x = (torch.randn((3, c), generator=g) * x_size).to(kind)
    dy = (torch.randn((3, c), generator=g) * dy_size).to(kind)
    gain = 1 + 0.2 * torch.randn((c,), generator=g)
    eps = float(np.float32(1e-30))
    s, d = x.double().numpy(), dy.double().numpy()
    r = 1 / np.sqrt((s ** 2).mean(1, keepdims=True) + eps)
    n, dn = s * r, d * gain.double().numpy()
    want = r * (dn - n * (dn * n).mean(1, keepdims=True))
    size = r * (np.abs(dn) + np.abs(n) * np.abs(dn * n).mean(1, keepdims=True))
    if np.abs(want).max() > 3e38:
        want, size = want * 0, size * 0 + np.inf  # out of fp32: only dgain is compared
    dx, dgain = M.rms_bprop(dy.to(device), x.to(device), gain.to(device), eps=eps)
    off = (c / 512 + 150) * U * size + 2.0 ** -126 * (1 + r)
    half = 2.0 ** -8 if kind == BF16 else U
    dx = dx.cpu().double().numpy()
    assert ((np.abs(dx - want) <= off + half * (np.abs(want) + off)) | np.isinf(size)).all()
    terms = np.abs(d * n).sum(0)
    assert (np.abs(dgain.cpu().double().numpy() - (d * n).sum(0)) <= (c / 2048 + 150) * U * terms + 3 * 2.0 ** -126).all()
