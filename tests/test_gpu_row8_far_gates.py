"""8-bit rows of activations far below zero (miq_act_row8): what the activation itself leaves below the normal numbers
may read zero, whatever multiplies it.  With u = 2^-24 an activation is within (16 + 4 v^2) u of its value, the
header's 2^-126 (1 + |v|) besides; a code within half a step, and 127 times that over the row's largest, and
127 * 5 u."""
import math

import numpy as np
import pytest
import torch

import my_own_cnn_amd as M

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
LEAST = 2.0 ** -110


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("size", [1.0, 1e5, 1e20, 1e37])
def test_gates_far_below_zero(device, act, size):
    at = np.concatenate([np.arange(-95, -60, 0.5), np.arange(-14.5, -8, 0.1), [-1e4, -1e38, -200.0]]).astype(np.float32)
    g = np.random.default_rng(1)
    gate = np.repeat(at[:, None], 40, 1) * g.uniform(1, 1.0001, (at.size, 40)).astype(np.float32)
    gate = gate.astype(np.float32)
    up = (g.standard_normal((at.size, 40)) * size).astype(np.float32)
    v = gate.astype(np.float64)
    if act == "silu":
        with np.errstate(over="ignore"):
            value = v / (1 + np.exp(-v))
    else:
        value = 0.5 * v * np.vectorize(math.erfc)(-v / math.sqrt(2))
    want = value * up
    off = ((16 + 4 * np.minimum(v ** 2, 1e4)) * U * np.abs(value) + 2.0 ** -126 * (1 + np.abs(v))) * np.abs(up)
    ordinary = np.abs(v[:, 0]) < 300  # beyond, both are zero
    m = np.maximum(np.abs(want).max(1), LEAST)
    m_off = off.max(1) / m
    kept = M.act_row8(torch.from_numpy(np.concatenate([gate, up], 1)).to(device), act, gated=True)
    codes, scales = kept.codes.cpu().double().numpy(), kept.scales.cpu().double().numpy()
    assert (codes[~ordinary] == 0).all() and (scales[~ordinary] == float(np.float32(LEAST) / np.float32(127))).all()
    got = codes * scales[:, None]  # half a step of the row's own scale, the activation's error, the operations'
    near = scales[:, None] * (0.5 + 127 * 5 * U) + off
    assert (np.abs(got - want) <= near)[ordinary].all()
    assert (np.abs(scales - m / 127) <= (m_off + 4 * U) * m / 127)[ordinary].all()
