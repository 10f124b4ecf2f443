"""A learned prior over a trained latent's symbols: the bits an arithmetic coder would need for them.

    python -m neural_block_textures_amd.prior model.bin|model.ntcb [--steps 300] [--hidden 256] [--batch 16384] [--lr 2e-3]
        [--state-bits 8|32] [--seed 1] [--fp32-latent] [--tile 0] [--layers 2] [--heads 8] [--stepped 0]

The print statistics price a latent by the entropy of its histograms, each symbol on its own or against its left neighbour. Here
a small network predicts each symbol from those before it in raster order (the texels to the left and above, and the
texel's own earlier channels), trained on the very latent, and the sum of its log probabilities is the price. One JSON line a level: bits a
symbol under the histogram and under the prior, the prior's own expectation (its entropy), and how often its first
alternative, or one of its first four, is the symbol.

With --tile T the model looks further than the neighbours: the plane is cut into tiles of T x T texels, a tile's symbols are a sequence in raster order, and blocks of
layer norm, rotary positions (row, column, channel) and causal attention over the tile come between the contexts and the alphabet. Everything a symbol is
predicted from still lies before it in the plane's raster order. Tiles of all sizes (those of the edges are smaller) are packed into one batch; TilePrior.step predicts
single symbols from the keys and values of those before them in their tiles. A decoder knows a symbol's neighbours in other tiles only in the plane's raster order, and raster_logprobs goes
that way, from a plane that holds nothing else yet; with --stepped N the first N symbols' bits are given as it predicts them, beside those of the pass over whole tiles.

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
        self.alphabet = alphabet
        self.values = self._scaled(sym)
        self.padded = torch.zeros((self.H + 1, self.W + 2, self.C), device=sym.device)
        self.padded[1:, 1:-1] = self.values

    def _scaled(self, sym):
        return sym.float() * (2.0 / max(1, self.alphabet - 1)) - 1.0

    def put(self, at: torch.Tensor, sym: torch.Tensor) -> None:
        """Symbols that have become known, at flat indices `at`"""
        texel, c = at // self.C, at % self.C
        y, x = texel // self.W, texel % self.W
        self.values[y, x, c] = self.padded[y + 1, x + 1, c] = self._scaled(sym)

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


class TilePrior:
    """A context's first layer, `layers` blocks of attention over a tile's earlier symbols and of two layers on each, and the alphabet's logits. Heads have
    hidden / heads elements, a multiple of 8; their pairs turn with a symbol's row, column and channel."""

    def __init__(self, width: int, hidden: int, alphabet: int, layers: int, heads: int, seed: int, device="cuda"):
        if layers < 1 or heads < 1 or hidden % heads or hidden // heads % 8 or hidden // heads > 128:
            raise ValueError(f"blocks and heads from 1 on are needed, heads of a multiple of 8 elements up to 128, not {layers} of {heads} in {hidden}")
        gen = torch.Generator(device=device).manual_seed(seed)
        self.heads, self.dim = heads, hidden // heads
        pairs = self.dim // 2
        self.sections = (pairs - pairs // 4 - (pairs - pairs // 4) // 2, (pairs - pairs // 4) // 2, pairs // 4)
        part = lambda x: x.to(torch.bfloat16).requires_grad_(True)  # noqa: E731
        matrix = lambda n, k, f=1.0: part(torch.randn((n, k), generator=gen, device=device) * (f * k ** -0.5))  # noqa: E731
        ones, zeros = (lambda n: part(torch.ones(n, device=device))), (lambda n: part(torch.zeros(n, device=device)))
        self.first, self.first_bias = matrix(hidden, width), zeros(hidden)
        small = (2 * layers) ** -0.5                      # what a block adds, so that their sum keeps its size
        self.blocks = [{"norm": ones(hidden), "norm_bias": zeros(hidden), "qkv": matrix(3 * hidden, hidden), "out": matrix(hidden, hidden, small),
                        "norm2": ones(hidden), "norm2_bias": zeros(hidden), "up": matrix(2 * hidden, hidden), "up_bias": zeros(2 * hidden),
                        "down": matrix(hidden, 2 * hidden, small)} for _ in range(layers)]
        self.last_norm, self.last_norm_bias, self.last, self.last_bias = ones(hidden), zeros(hidden), matrix(alphabet, hidden), zeros(alphabet)

    def parameters(self) -> list:
        return [self.first, self.first_bias, *(p for b in self.blocks for p in b.values()), self.last_norm, self.last_norm_bias, self.last, self.last_bias]

    def laid_out(self) -> dict:
        """The matrices in 8 bits, for passes without gradients."""
        return {id(p): ops.fp8_quantize(p.detach(), 128) for p in self.parameters() if p.dim() == 2}

    def _pass(self, x, positions, attend, weights):
        matrix = (lambda p: p) if weights is None else (lambda p: weights[id(p)])
        h = torch.relu(ops.fp8_linear(x, matrix(self.first)) + self.first_bias)
        for n, b in enumerate(self.blocks):
            qkv = ops.fp8_linear(ops.layer_norm(h, b["norm"], b["norm_bias"]), matrix(b["qkv"])).view(len(h), 3 * self.heads, self.dim)
            q, k = ops.rotary(positions, qkv[:, :self.heads], qkv[:, self.heads:2 * self.heads], sections=self.sections)
            h = h + ops.fp8_linear(attend(n, q, k, qkv[:, 2 * self.heads:]).reshape(len(h), -1), matrix(b["out"]))
            up = torch.relu(ops.fp8_linear(ops.layer_norm(h, b["norm2"], b["norm2_bias"]), matrix(b["up"])) + b["up_bias"])
            h = h + ops.fp8_linear(up, matrix(b["down"]))
        return ops.fp8_linear(ops.layer_norm(h, self.last_norm, self.last_norm_bias), matrix(self.last)) + self.last_bias

    def logits(self, x: torch.Tensor, positions: torch.Tensor, ends: torch.Tensor, weights=None) -> torch.Tensor:
        """[symbols, alphabet] for packed tiles: contexts [symbols, width], positions [symbols, 3], ends int32 [tiles + 1]."""
        return self._pass(x, positions, lambda n, q, k, v: ops.attention(q, k, v, cu_q=ends, cu_k=ends), weights)

    def cache(self, tiles: int, symbols: int) -> list:
        """Room for the keys and values of `symbols` symbols of each of `tiles` tiles, for each block."""
        room = lambda: torch.empty((tiles, symbols, self.heads, self.dim), dtype=torch.bfloat16, device=self.first.device)  # noqa: E731
        return [(room(), room()) for _ in self.blocks]

    @torch.no_grad()                                      # (a cache that is written in place keeps no graph)
    def step(self, x: torch.Tensor, positions: torch.Tensor, cache: list, lens: torch.Tensor, weights=None) -> torch.Tensor:
        """[tiles, alphabet] for one more symbol of each tile, the lens[i]-th (int32 [tiles]) of tile i; its keys and values go into the cache. Lengths are read on the GPU: where a tile's
        has no room its last place is written over, and the prediction is wrong."""
        if len(cache) != len(self.blocks) or not len(x) == len(positions) == len(lens):
            raise ValueError(f"one context, position and length a tile and a cache for each block are needed, not {len(x)}, {len(positions)} and {len(lens)}, and {len(cache)} for {len(self.blocks)}")
        for room in (r for pair in cache for r in pair):
            if room.dim() != 4 or len(room) != len(x) or room.shape[1] < 1 or room.shape[1] != cache[0][0].shape[1] or room.shape[2:] != (self.heads, self.dim):
                raise ValueError(f"the cache must be [{len(x)} tiles, symbols, {self.heads} heads, {self.dim}], not {list(room.shape)}")
        each, at = torch.arange(len(x), device=x.device), lens.long().clamp(0, cache[0][0].shape[1] - 1)

        def attend(n, q, k, v):
            keys, values = cache[n]
            keys[each, at], values[each, at] = k, v
            return ops.attention(q[:, None], keys, values, k_lens=lens + 1)

        return self._pass(x, positions, attend, weights)


class Tiles:
    """A plane's symbols tile by tile: their flat indices in raster order within each, and where each tile ends."""

    def __init__(self, shape, tile: int, device):
        H, W, C = shape
        if tile < 1:
            raise ValueError(f"tiles have 1 texel a side or more, not {tile}")
        flat = torch.arange(H * W * C, device=device).view(H, W, C)
        cut = [flat[y:y + tile, x:x + tile].reshape(-1) for y in range(0, H, tile) for x in range(0, W, tile)]
        self.shape, self.tile, self.order, self.lengths = shape, tile, cut, [len(c) for c in cut]

    def batch(self, which) -> tuple:
        """(flat indices, positions [symbols, 3], ends) of some tiles, packed"""
        at = torch.cat([self.order[i] for i in which])
        _, W, C = self.shape
        texel = at // C
        ends = np.cumsum([0] + [self.lengths[i] for i in which], dtype=np.int32)
        return at, torch.stack([texel // W, texel % W, at % C], 1), torch.from_numpy(ends).to(at.device)

    def groups(self, symbols: int) -> list:
        """All tiles, in runs of at most `symbols` symbols (one tile at least)."""
        out, size = [[]], 0
        for i, n in enumerate(self.lengths):
            if out[-1] and size + n > symbols:
                out.append([])
                size = 0
            out[-1].append(i)
            size += n
        return out


def fit_tiles(sym: torch.Tensor, alphabet: int, tile: int, steps: int = 300, hidden: int = 256, layers: int = 2, heads: int = 8, batch: int = 16384, lr: float = 2e-3,
              state_bits: int = 8, seed: int = 1):
    """(TilePrior, Contexts, Tiles) trained on symbols [H, W, C] that are on the GPU, some `batch` symbols of whole tiles a step."""
    if steps < 0 or hidden < 1 or batch < 1 or not sym.numel():
        raise ValueError(f"steps from 0 on, hidden units and a batch from 1 on, and symbols are needed, not {steps}, {hidden}, {batch} and {list(sym.shape)}")
    ctx, tiles = Contexts(sym, alphabet), Tiles(sym.shape, tile, sym.device)
    prior = TilePrior(ctx.width, hidden, alphabet, layers, heads, seed, sym.device)
    opt = ops.AdamW(prior.parameters(), lr=lr, weight_decay=0.01, state_bits=state_bits, master=True, seed=seed)
    rng, flat = np.random.default_rng(seed), sym.reshape(-1)
    count = min(len(tiles.lengths), max(1, batch // max(tiles.lengths)))
    for step in range(steps):
        at, positions, ends = tiles.batch(rng.choice(len(tiles.lengths), count, replace=False))
        bits = ops.token_logprobs(prior.logits(ctx.rows(at), positions, ends), flat[at]).logprob
        opt.zero_grad()
        (-bits.mean()).backward()
        opt.lr = lr * 0.5 * (1 + math.cos(math.pi * step / steps))
        opt.step()
    return prior, ctx, tiles


@torch.no_grad()
def step_logprobs(prior: TilePrior, ctx: Contexts, tiles: Tiles, sym: torch.Tensor, which) -> torch.Tensor:
    """Log probabilities of the symbols of tiles of one size, [tiles, symbols], predicted one at a time in all tiles together, with contexts of the finished plane: TilePrior.step against the pass
    over whole tiles. (A decoder has no such contexts across the tiles' borders, and goes as raster_logprobs does.)"""
    n = tiles.lengths[which[0]]
    if any(tiles.lengths[i] != n for i in which):
        raise ValueError("tiles of one size are needed")
    at, positions, _ = tiles.batch(which)
    at, positions = at.view(-1, n), positions.view(-1, n, 3)
    flat, weights, cache = sym.reshape(-1), prior.laid_out(), prior.cache(len(at), n)
    lens, out = torch.zeros(len(at), dtype=torch.int32, device=sym.device), []
    for i in range(n):
        out.append(ops.token_logprobs(prior.step(ctx.rows(at[:, i]), positions[:, i], cache, lens, weights), flat[at[:, i]]).logprob)
        lens += 1
    return torch.stack(out, 1)


@torch.no_grad()
def raster_logprobs(prior: TilePrior, tiles: Tiles, sym: torch.Tensor, alphabet: int, count: int = None) -> torch.Tensor:
    """Log probabilities of the plane's first `count` symbols (all of them where it is None), predicted one at a time in its raster order: contexts of a plane that holds the symbols before and
    nothing else, keys and values of the symbol's own tile. A decoder that reads the symbol where this one looks it up goes the same way."""
    H, W, C = tiles.shape
    flat, n = sym.reshape(-1), sym.numel() if count is None else count
    if not 0 <= n <= flat.numel():
        raise ValueError(f"0 to {flat.numel()} symbols can be predicted, not {n}")
    ctx, weights, across = Contexts(torch.zeros_like(sym), alphabet), prior.laid_out(), -(-W // tiles.tile)
    cache, lens = prior.cache(across, max(tiles.lengths)), torch.zeros(across, dtype=torch.int32, device=sym.device)      # of one row of tiles, the next row's after it
    at = torch.arange(n, device=sym.device)
    positions, out = torch.stack([at // C // W, at // C % W, at % C], 1), torch.empty(n, device=sym.device)
    for i in range(n):
        if i % (tiles.tile * W * C) == 0:
            lens.zero_()
        one, t = slice(i, i + 1), i // C % W // tiles.tile
        own = slice(t, t + 1)
        logits = prior.step(ctx.rows(at[one]), positions[one], [(k[own], v[own]) for k, v in cache], lens[own], weights)
        out[one] = ops.token_logprobs(logits, flat[one]).logprob
        ctx.put(at[one], flat[one])
        lens[own] += 1
    return out


@torch.no_grad()
def packed_logprobs(prior: TilePrior, ctx: Contexts, tiles: Tiles, sym: torch.Tensor, batch: int = 1 << 17) -> torch.Tensor:
    """Log probabilities of all symbols, in the plane's raster order, by passes over whole tiles"""
    flat, weights = sym.reshape(-1), prior.laid_out()
    out = torch.empty(flat.numel(), device=sym.device)
    for which in tiles.groups(batch):
        at, positions, ends = tiles.batch(which)
        out[at] = ops.token_logprobs(prior.logits(ctx.rows(at), positions, ends, weights), flat[at]).logprob
    return out


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
def price(prior, ctx: Contexts, sym: torch.Tensor, batch: int = 1 << 17, tiles: Tiles = None) -> dict:
    """The symbols' bits under the prior (a TilePrior with its tiles), its expectation of them, and how often its first one and four alternatives hold the symbol."""
    flat, weights = sym.reshape(-1), prior.laid_out()
    top = min(4, prior.parameters()[-1].numel())
    total = torch.zeros(4, dtype=torch.float64, device=sym.device)

    def parts():
        if tiles is None:
            for start in range(0, flat.numel(), batch):
                at = torch.arange(start, min(start + batch, flat.numel()), device=sym.device)
                yield at, prior.logits(ctx.rows(at), weights)
        else:
            for which in tiles.groups(batch):
                at, positions, ends = tiles.batch(which)
                yield at, prior.logits(ctx.rows(at), positions, ends, weights)

    for at, logits in parts():
        r = ops.token_logprobs(logits, flat[at], top=top)
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
    ap.add_argument("--tile", type=int, default=0, help="attention over tiles of this many texels a side (0: the neighbours alone)")
    ap.add_argument("--layers", type=int, default=2, help="blocks of attention")
    ap.add_argument("--heads", type=int, default=8)
    ap.add_argument("--stepped", type=int, default=0, help="predict a level's first so many symbols one at a time too, as a decoder has to (with --tile)")
    a = ap.parse_args(argv)
    if a.stepped < 0 or (a.stepped and not a.tile):
        ap.error("--stepped takes a number from 0 on, and --tile beside it")
    for l, sym, alphabet in level_symbols(decode.load(a.model, q8=not a.fp32_latent)):
        dev = torch.from_numpy(sym).cuda()
        tiles = None
        if a.tile:
            prior, ctx, tiles = fit_tiles(dev, alphabet, a.tile, a.steps, a.hidden, a.layers, a.heads, a.batch, a.lr, a.state_bits, a.seed)
        else:
            prior, ctx = fit(dev, alphabet, a.steps, a.hidden, a.batch, a.lr, a.state_bits, a.seed)
        out = {"level": l, "symbols": sym.size, "alphabet": alphabet, "histogram_bits": histogram_bits(sym), **price(prior, ctx, dev, tiles=tiles)}
        out["saved"] = 1.0 - out["prior_bits"] / out["histogram_bits"] if out["histogram_bits"] else 0.0
        if a.stepped:
            n = min(a.stepped, sym.size)
            bits = lambda x: -x.double().mean().item() / math.log(2)  # noqa: E731
            out.update(stepped=n, stepped_bits=bits(raster_logprobs(prior, tiles, dev, alphabet, n)), packed_bits=bits(packed_logprobs(prior, ctx, tiles, dev)[:n]))
        print(json.dumps(out), flush=True)


if __name__ == "__main__":
    sys.exit(main())
