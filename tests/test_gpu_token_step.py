"""The example's training step on the GPU: its gradients against automatic differentiation in 64
bits at the same kept values, and its loss over a few steps."""
import importlib.util
import math
from pathlib import Path

import pytest
import torch

import my_own_cnn_amd as M

pytestmark = pytest.mark.gpu

_spec = importlib.util.spec_from_file_location("token_step", Path(__file__).resolve().parents[1] / "examples" /
                                               "token_step.py")
T = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(T)


def _through(value, kept):
    """`kept` in place of `value`, whose gradient it passes on."""
    return value + (kept - value).detach()


@pytest.mark.parametrize("batch,length,vocab,channels", [(2, 9, 11, 32), (3, 40, 50, 48)])
def test_gradients_of_a_step(device, batch, length, vocab, channels):
    p = T.init(vocab, channels, device, seed=3)
    ids, _ = T.sequences(batch, length, vocab, device, 1)
    z, kept = T.forward(p, ids)
    dz = torch.randn(z.shape, generator=torch.Generator().manual_seed(2)).to(device) / z.numel()
    g = T.backward(p, kept, dz)

    q = {k: v.double().cpu().requires_grad_() for k, v in p.items()}
    padded = kept["ids"].cpu()
    there = (padded >= 0)[..., None]
    x = torch.where(there, q["E"][padded.clamp(min=0)] * math.sqrt(channels), torch.zeros(()).double())
    kx, kh, ka = (M.act8_expand(kept[n]).double().cpu()[:, 0] for n in ("x", "h", "a"))
    # a layer's own gradient is taken at its kept input, its input's gradient at its weights
    w1 = q["W1"][:, 0].permute(0, 2, 1)
    h = torch.nn.functional.conv1d(_through(x, kx).transpose(1, 2), w1).transpose(1, 2)
    gate, up = _through(h, kh).chunk(2, 2)
    a = gate * torch.sigmoid(gate) * up
    logits = _through(a, ka) @ q["W2"][:, 0, 0].t()
    (logits * dz.double().cpu()[:, 0]).sum().backward()
    # fp32 sums of up to batch * length products, through three layers
    for name in ("W2", "W1", "E"):
        want, got = q[name].grad, g[name].double().cpu()
        off = float((got - want).norm() / want.norm())
        assert off <= 3 * 2.0 ** -24 * math.sqrt(batch * length * vocab) + 3e-6, (name, off)


def test_the_loss_falls_and_a_quarter_is_kept(device):
    p = T.init(32, 32, device)
    losses = [float(T.step(p, *T.sequences(8, 64, 32, device, i), 0.5)) for i in range(40)]
    assert losses[0] > 3 and losses[-1] < 0.7 * losses[0], losses
    _, kept = T.forward(p, T.sequences(8, 64, 32, device, 0)[0])
    small, whole = T.kept_bytes(kept)
    assert small == whole // 4 + whole // 128
