"""Symbols predicted one at a time in the plane's raster order, as a decoder has to: as the pass over whole tiles predicts them, from nothing that comes later."""
import json
import math
import os

import numpy as np
import pytest
import torch

from neural_block_textures_amd import ops, prior
from tests.helpers import GOLDEN

pytestmark = pytest.mark.gpu


def plane(H, W, C, alphabet, seed):
    return torch.from_numpy(np.random.default_rng(seed).integers(0, alphabet, (H, W, C))).cuda()


def test_as_whole_tiles(monkeypatch):
    """Tiles of four shapes, two of them of 16 symbols. A logit of a step and of the whole pass differ by what sums in another order round to: 8 tensors of 16 bits a block and 3 beside them, each off by a step of its largest
    value at most (products in 32 bits here: 8-bit codes would turn such a difference into a 16th); a log probability by that of its logit and of the log sum."""
    def linear(x, w):
        return (x.float() @ (w.values() if isinstance(w, ops.Fp8Tensor) else w.float()).T.contiguous()).to(x.dtype)

    sym = plane(10, 14, 2, 32, 4)
    p, ctx, tiles = prior.fit_tiles(sym, 32, 4, steps=4, hidden=64, layers=2, heads=4, batch=512)
    assert set(tiles.lengths) == {32, 16, 8}
    monkeypatch.setattr(prior.ops, "fp8_linear", linear)
    with torch.no_grad():
        at, positions, ends = tiles.batch(range(len(tiles.lengths)))
        largest = p.logits(ctx.rows(at), positions, ends, p.laid_out()).float().abs().max()
    one, whole = prior.raster_logprobs(p, tiles, sym, 32), prior.packed_logprobs(p, ctx, tiles, sym)
    assert one.shape == whole.shape == (280,) and (one - whole).abs().max() <= 2 * (8 * 2 + 3) * 2.0 ** -8 * largest
    assert torch.equal(prior.raster_logprobs(p, tiles, sym, 32, 50), one[:50])


def test_nothing_later_is_known():
    sym = plane(7, 9, 2, 16, 5)
    p, ctx, tiles = prior.fit_tiles(sym, 16, 4, steps=2, hidden=64, layers=1, heads=4, batch=512)
    before = prior.raster_logprobs(p, tiles, sym, 16)
    later = sym.reshape(-1).clone()
    later[70:] = 15 - later[70:]
    after = prior.raster_logprobs(p, tiles, later.view(sym.shape), 16)
    assert torch.equal(before[:70], after[:70]) and not torch.equal(before[70:], after[70:])


def test_the_price_of_whole_tiles():
    sym = plane(9, 11, 3, 20, 6)
    p, ctx, tiles = prior.fit_tiles(sym, 20, 4, steps=2, hidden=64, layers=1, heads=2, batch=512)
    want = prior.price(p, ctx, sym, batch=100, tiles=tiles)["prior_bits"]
    got = -prior.packed_logprobs(p, ctx, tiles, sym, batch=100).double().mean().item() / math.log(2)
    assert abs(got - want) <= 1e-6 * want


def test_the_command(capsys):
    prior.main([os.path.join(GOLDEN, "ref_m1234_model.bin"), "--steps", "10", "--hidden", "64", "--tile", "8", "--layers", "1", "--heads", "4", "--stepped", "40"])
    for line in capsys.readouterr().out.splitlines():
        x = json.loads(line)
        assert x["stepped"] == 40 and 0 < x["stepped_bits"] < math.inf and 0 < x["packed_bits"] < math.inf
