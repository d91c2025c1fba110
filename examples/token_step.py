"""Trains a small token network on one GPU: what it reads is fed by the embedding lookup, what it
keeps between its forward and backward passes is kept in 8 bits.

    python examples/token_step.py [--steps 60] [--tokens 256] [--channels 64]

The network predicts the next token of a sequence from the last three:

    x = sqrt(C) E[ids]                    embed_fprop        rows of a (B, 1, L, C) NHWC tensor
    h = conv(x, W1), 1 x 3, to 2C         conv2d_nhwc_f32
    a = silu(gate(h)) * up(h)             act8_fprop         keeps h in 8 bits
    z = a W2^T, to one logit per token    conv2d_nhwc_f32, 1 x 1

and the backward pass uses what was kept: dW2 from the kept a (act8_grad), dh from the kept h
(act8_bprop), dW1 from the kept x expanded (act8_expand, launch_grad_nhwc), and the table's
gradient by sorted tokens (embed_grad).  Two positions without a token (id -1, rows of zeros) stand
in front of each sequence, so that position t reads t - 2, t - 1 and t.
"""
import argparse
import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import my_own_cnn_amd as M  # noqa: E402
from my_own_cnn_amd.conv import Conv2DParams  # noqa: E402

TAPS = 3


def init(vocab, channels, device, seed=0):
    """E (vocab, C), W1 (2C, 1, 3, C) and W2 (vocab, 1, 1, C)."""
    g = torch.Generator().manual_seed(seed)

    def normal(shape, spread):
        return (torch.randn(shape, generator=g) * spread).to(device)

    return {"E": normal((vocab, channels), channels ** -0.5),
            "W1": normal((2 * channels, 1, TAPS, channels), (TAPS * channels) ** -0.5),
            "W2": normal((vocab, 1, 1, channels), channels ** -0.5)}


def forward(p, ids):
    """Logits (B, 1, L, vocab) of ids (B, L), and what the backward pass needs."""
    before = torch.full((ids.shape[0], TAPS - 1), -1, dtype=ids.dtype, device=ids.device)
    padded = torch.cat([before, ids], 1)
    scale = math.sqrt(p["E"].shape[1])
    x = M.embed_fprop(p["E"], padded[:, None], scale=scale)
    h = M.conv2d_nhwc_f32(x, p["W1"])
    a, kept_h = M.act8_fprop(h, "silu", gated=True)
    z = M.conv2d_nhwc_f32(a, p["W2"])
    return z, {"ids": padded, "scale": scale, "x": M.act8_keep(x), "h": kept_h, "a": M.act8_keep(a)}


def backward(p, kept, dz):
    """The gradients of E, W1 and W2 from the logits' gradient (B, 1, L, vocab)."""
    batch, _, length, vocab = dz.shape
    channels = p["E"].shape[1]
    wide = length + TAPS - 1
    flat = Conv2DParams(0, 0)
    g = {"W2": M.act8_grad(dz, kept["a"]).reshape(p["W2"].shape)}
    da = torch.empty((batch, 1, length, channels), device=dz.device)
    M.launch_bprop_nhwc(dz, p["W2"], da, batch, 1, length, channels, 1, 1, vocab, flat)
    dh = M.act8_bprop(da, kept["h"])
    x = M.act8_expand(kept["x"])
    g["W1"] = torch.empty_like(p["W1"])
    M.launch_grad_nhwc(x, dh, g["W1"], batch, 1, wide, channels, 1, TAPS, 2 * channels, flat)
    dx = torch.empty_like(x)
    M.launch_bprop_nhwc(dh, p["W1"], dx, batch, 1, wide, channels, 1, TAPS, 2 * channels, flat)
    g["E"] = M.embed_grad(dx, kept["ids"][:, None], p["E"].shape[0], scale=kept["scale"])
    return g


def step(p, ids, target, rate):
    """One step of gradient descent; the mean cross-entropy before it."""
    z, kept = forward(p, ids)
    logits = z[:, 0]
    share = torch.softmax(logits, 2)
    loss = -torch.log(share.gather(2, target[..., None])).mean()
    dz = share
    dz.scatter_add_(2, target[..., None], torch.full_like(share[..., :1], -1.0))
    g = backward(p, kept, (dz / target.numel())[:, None].contiguous())
    for name, value in g.items():
        p[name].sub_(value, alpha=rate)
    return loss


def sequences(batch, length, vocab, device, seed):
    """Sequences in which a token follows from the two before it."""
    g = torch.Generator().manual_seed(seed)
    s = torch.randint(0, vocab, (batch, 2), generator=g)
    for _ in range(length - 1):
        s = torch.cat([s, ((3 * s[:, -1:] + 5 * s[:, -2:-1] + 1) % vocab)], 1)
    return s[:, :length].contiguous().to(device), s[:, 1: length + 1].contiguous().to(device)


def kept_bytes(kept):
    """(bytes kept, bytes of the same tensors in fp32)."""
    held = [t for t in kept.values() if isinstance(t, M.Act8)]
    return sum(t.codes.numel() + t.scales.numel() for t in held), sum(4 * t.codes.numel() for t in held)


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--batch", type=int, default=16)
    ap.add_argument("--tokens", type=int, default=256, help="tokens of a sequence")
    ap.add_argument("--vocab", type=int, default=96)
    ap.add_argument("--channels", type=int, default=64)
    ap.add_argument("--rate", type=float, default=0.5)
    args = ap.parse_args()
    device = torch.device("cuda:0")
    p = init(args.vocab, args.channels, device)
    for i in range(args.steps):
        loss = step(p, *sequences(args.batch, args.tokens, args.vocab, device, i), args.rate)
        if i % 10 == 0 or i == args.steps - 1:
            print(f"step {i}: loss {float(loss):.4f}", flush=True)
    _, kept = forward(p, sequences(args.batch, args.tokens, args.vocab, device, 0)[0])
    small, whole = kept_bytes(kept)
    print(f"kept between the passes: {small} bytes, {whole} in fp32")


if __name__ == "__main__":
    main()
