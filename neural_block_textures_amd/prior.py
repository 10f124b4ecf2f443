"""A learned prior over a trained latent's symbols: the bits an arithmetic coder would need for them.

    python -m neural_block_textures_amd.prior model.bin|model.ntcb [--steps 300] [--hidden 256] [--batch 16384] [--lr 2e-3]
        [--state-bits 8|32] [--seed 1] [--fp32-latent]

The print statistics price a latent by the entropy of its histograms, each symbol on its own or against its left neighbour. Here
a small network predicts each symbol from those before it in raster order (the texels to the left and above, and the
texel's own earlier channels), trained on the very latent, and the sum of its log probabilities is the price. One JSON line a level: bits a
symbol under the histogram and under the prior, the prior's own expectation (its entropy), and how often its first
alternative, or one of its first four, is the symbol.

A training step is the operators of ops.py end to end: layers in 8-bit floating point (fp8_linear), the symbols' log
probabilities and their gradient (token_logprobs), and one AdamW step over all weights with an 8-bit state. The price is then
taken with the weights laid out in 8 bits once (their own bits are not part of it). A level on a grid or palette is taken as it is, continuous ones on the post-hoc
8-bit grid (decode.py); a DCT-coded level's symbols are tokens and not texels, and are left out.
"""
from __future__ import annotations

import argparse
import json
import math
import sys

import numpy as np
import torch

from . import decode, ops


def level_symbols(m) -> list:
    """[(level, symbols [H, W, C] as int64, alphabet)] of a model file's levels: each channel's values as indices into its distinct
    ones, ascending. Levels of more than 4096 distinct values in a channel (left continuous) are refused."""
    out, lay = [], m.layout
    for l, ((W, H, C, _), off) in enumerate(zip(lay.levels, lay.offsets)):
        if l == 0 and m.dct is not None:
            continue
        z = m.z[off:off + W * H * C].reshape(H, W, C)
        sym = np.stack([np.unique(z[..., c], return_inverse=True)[1].reshape(H, W) for c in range(C)], -1).astype(np.int64)
        if sym.max() >= 4096:
            raise ValueError(f"level {l} is continuous (over 4096 values in a channel): give it a grid first")
        out.append((l, sym, int(sym.max()) + 1))
    return out


def histogram_bits(sym: np.ndarray) -> float:
    """Bits a symbol by each channel's own histogram (order 0)."""
    total = 0.0
    for c in range(sym.shape[-1]):
        n = np.bincount(sym[..., c].reshape(-1)).astype(np.float64)
        n = n[n > 0]
        total += -(n * np.log2(n / n.sum())).sum()
    return total / sym.size


class Contexts:
    """What a symbol is predicted from: the texels to the left, above, above left and above right (all channels), its texel's earlier
    channels, which channel it is, and a 1; symbols scaled to [-1, 1], 0 outside the plane."""

    def __init__(self, sym: torch.Tensor, alphabet: int):
        self.H, self.W, self.C = sym.shape
        self.width = 6 * self.C + 1
        self.values = sym.float() * (2.0 / max(1, alphabet - 1)) - 1.0
        self.padded = torch.zeros((self.H + 1, self.W + 2, self.C), device=sym.device)
        self.padded[1:, 1:-1] = self.values

    def rows(self, at: torch.Tensor) -> torch.Tensor:
        """[len(at), width] for symbols `at` (flat indices), in bfloat16"""
        texel, c = at // self.C, at % self.C
        y, x = texel // self.W, texel % self.W
        p = self.padded
        one_hot = torch.nn.functional.one_hot(c, self.C).float()
        earlier = torch.arange(self.C, device=at.device)[None] < c[:, None]
        parts = [p[y + 1, x], p[y, x + 1], p[y, x], p[y, x + 2], self.values[y, x] * earlier, one_hot, torch.ones_like(at)[:, None].float()]
        return torch.cat(parts, 1).to(torch.bfloat16)


class Prior:
    """Three layers on a context: width -> hidden -> hidden (added to the first's output) -> alphabet."""

    def __init__(self, width: int, hidden: int, alphabet: int, seed: int, device="cuda"):
        gen = torch.Generator(device=device).manual_seed(seed)
        shapes = [(hidden, width), (hidden, hidden), (alphabet, hidden)]
        self.weights = [(torch.randn(s, generator=gen, device=device) * math.sqrt(1.0 / s[1])).to(torch.bfloat16).requires_grad_(True) for s in shapes]
        self.biases = [torch.zeros(s[0], dtype=torch.bfloat16, device=device, requires_grad=True) for s in shapes]

    def parameters(self) -> list:
        return self.weights + self.biases

    def laid_out(self) -> list:
        """The weights in 8 bits, for passes without gradients."""
        return [ops.fp8_quantize(w.detach(), 128) for w in self.weights]

    def logits(self, x: torch.Tensor, weights=None) -> torch.Tensor:
        w, b = self.weights if weights is None else weights, self.biases
        h = torch.relu(ops.fp8_linear(x, w[0]) + b[0])
        h = h + torch.relu(ops.fp8_linear(h, w[1]) + b[1])
        return ops.fp8_linear(h, w[2]) + b[2]


def fit(sym: torch.Tensor, alphabet: int, steps: int = 300, hidden: int = 256, batch: int = 16384, lr: float = 2e-3, state_bits: int = 8, seed: int = 1):
    """(Prior, Contexts) trained on symbols [H, W, C] that are on the GPU."""
    if steps < 0 or hidden < 1 or batch < 1 or not sym.numel():
        raise ValueError(f"steps from 0 on, hidden units and a batch from 1 on, and symbols are needed, not {steps}, {hidden}, {batch} and {list(sym.shape)}")
    ctx = Contexts(sym, alphabet)
    prior = Prior(ctx.width, hidden, alphabet, seed, sym.device)
    opt = ops.AdamW(prior.parameters(), lr=lr, weight_decay=0.01, state_bits=state_bits, master=True, seed=seed)
    gen = torch.Generator(device=sym.device).manual_seed(seed)
    flat = sym.reshape(-1)
    for step in range(steps):
        at = torch.randint(0, flat.numel(), (min(batch, flat.numel()),), generator=gen, device=sym.device)
        bits = ops.token_logprobs(prior.logits(ctx.rows(at)), flat[at]).logprob
        opt.zero_grad()
        (-bits.mean()).backward()
        opt.lr = lr * 0.5 * (1 + math.cos(math.pi * step / steps))
        opt.step()
    return prior, ctx


@torch.no_grad()
def price(prior: Prior, ctx: Contexts, sym: torch.Tensor, batch: int = 1 << 17) -> dict:
    """The symbols' bits under the prior, its expectation of them, and how often its first one and four alternatives hold the symbol."""
    flat, weights = sym.reshape(-1), prior.laid_out()
    top = min(4, prior.weights[2].shape[0])
    total = torch.zeros(4, dtype=torch.float64, device=sym.device)
    for start in range(0, flat.numel(), batch):
        at = torch.arange(start, min(start + batch, flat.numel()), device=sym.device)
        r = ops.token_logprobs(prior.logits(ctx.rows(at), weights), flat[at], top=top)
        hit = r.top_ids == flat[at, None]
        total += torch.stack([-r.logprob.double().sum(), r.entropy.double().sum(), hit[:, 0].double().sum(), hit.double().sum()])
    bits, expected, first, four = (total / flat.numel()).tolist()
    return {"prior_bits": bits / math.log(2), "expected_bits": expected / math.log(2), "first": first, "first_four": four}


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("model")
    ap.add_argument("--steps", type=int, default=300)
    ap.add_argument("--hidden", type=int, default=256)
    ap.add_argument("--batch", type=int, default=16384)
    ap.add_argument("--lr", type=float, default=2e-3)
    ap.add_argument("--state-bits", type=int, default=8, choices=(8, 32))
    ap.add_argument("--seed", type=int, default=1)
    ap.add_argument("--fp32-latent", action="store_true", help="the stored values, not the post-hoc 8-bit grid (levels must be on a grid already)")
    a = ap.parse_args(argv)
    for l, sym, alphabet in level_symbols(decode.load(a.model, q8=not a.fp32_latent)):
        dev = torch.from_numpy(sym).cuda()
        prior, ctx = fit(dev, alphabet, a.steps, a.hidden, a.batch, a.lr, a.state_bits, a.seed)
        out = {"level": l, "symbols": sym.size, "alphabet": alphabet, "histogram_bits": histogram_bits(sym), **price(prior, ctx, dev)}
        out["saved"] = 1.0 - out["prior_bits"] / out["histogram_bits"] if out["histogram_bits"] else 0.0
        print(json.dumps(out), flush=True)


if __name__ == "__main__":
    sys.exit(main())
