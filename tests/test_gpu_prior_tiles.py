"""The prior with attention over tiles: it runs, sees nothing that comes later, prices as its logits say, predicts one symbol at a time as it does all at once; and the blocks' operators one after
another pass gradients as they do one by one."""
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


def test_tiles_cover_the_plane():
    sym = plane(20, 35, 3, 9, 1)
    tiles = prior.Tiles(sym.shape, 16, sym.device)
    at, positions, ends = tiles.batch(range(len(tiles.lengths)))
    assert sorted(tiles.lengths) == sorted([16 * 16 * 3] * 2 + [16 * 3 * 3] + [4 * 16 * 3] * 2 + [4 * 3 * 3]) and ends[-1] == sym.numel() and ends.dtype == torch.int32
    assert torch.equal(at.sort().values, torch.arange(sym.numel(), device="cuda"))
    y, x, c = positions.unbind(1)
    assert torch.equal(sym[y, x, c], sym.reshape(-1)[at])
    for i in range(len(tiles.lengths)):
        assert (at[ends[i]:ends[i + 1]].diff() > 0).all()              # a tile's symbols in the plane's order
    assert [i for g in tiles.groups(800) for i in g] == list(range(6)) and all(len(g) == 1 or sum(tiles.lengths[i] for i in g) <= 800 for g in tiles.groups(800))


def test_nothing_later_is_seen():
    sym = plane(16, 16, 2, 16, 2)
    p, ctx, tiles = prior.fit_tiles(sym, 16, 8, steps=2, hidden=64, layers=2, heads=4, batch=512)
    at, positions, ends = tiles.batch([0, 3])
    with torch.no_grad():
        before = p.logits(ctx.rows(at), positions, ends)
        later = sym.reshape(-1).clone()
        cut = at[70]                                                    # of the first tile; the second tile lies behind it in the plane
        later[cut:] = 15 - later[cut:]
        after = p.logits(prior.Contexts(later.view(sym.shape), 16).rows(at), positions, ends)
    assert torch.equal(before[:71], after[:71]) and not torch.equal(before[71:], after[71:])


def test_the_price_is_that_of_the_logits():
    sym = plane(21, 30, 3, 50, 3)
    p, ctx, tiles = prior.fit_tiles(sym, 50, 8, steps=3, hidden=64, layers=1, heads=2, batch=700)
    r = prior.price(p, ctx, sym, batch=600, tiles=tiles)
    total = entropy = 0.0
    with torch.no_grad():
        for which in tiles.groups(600):
            at, positions, ends = tiles.batch(which)
            logp = torch.log_softmax(p.logits(ctx.rows(at), positions, ends, p.laid_out()).double(), 1)
            total -= logp.gather(1, sym.reshape(-1)[at, None]).sum().item()
            entropy -= (logp * logp.exp()).sum().item()
    want, expected = total / sym.numel() / math.log(2), entropy / sym.numel() / math.log(2)
    assert abs(r["prior_bits"] - want) < 1e-5 * want and abs(r["expected_bits"] - expected) < 1e-5 * expected


def test_one_symbol_at_a_time(monkeypatch):
    """Logits of a step and of the whole pass differ by what sums in another order round to: 8 tensors of 16 bits a block and 3 beside them, each off by a step of its largest value at most (products in
    32 bits here: 8-bit codes would turn such a difference into a 16th)."""
    def linear(x, w):
        return (x.float() @ (w.values() if isinstance(w, ops.Fp8Tensor) else w.float()).T.contiguous()).to(x.dtype)

    sym = plane(16, 24, 2, 32, 4)
    p, ctx, tiles = prior.fit_tiles(sym, 32, 8, steps=4, hidden=64, layers=2, heads=4, batch=512)
    weights = p.laid_out()
    with torch.no_grad():
        monkeypatch.setattr(prior.ops, "fp8_linear", linear)
        at, positions, ends = tiles.batch(range(6))
        whole = p.logits(ctx.rows(at), positions, ends, weights).view(6, 128, -1).float()
        cache, lens = p.cache(6, 150), torch.zeros(6, dtype=torch.int32, device="cuda")
        for block in cache:
            for room in block:
                room.fill_(float("nan"))                               # what is not yet there is not read
        for i in range(128):
            one = p.step(ctx.rows(at.view(6, 128)[:, i]), positions.view(6, 128, 3)[:, i], cache, lens, weights).float()
            lens += 1
            assert (one - whole[:, i]).abs().max() <= (8 * 2 + 3) * 2.0 ** -8 * whole.abs().max(), i
    monkeypatch.undo()
    logp = prior.step_logprobs(p, ctx, tiles, sym, range(6))
    assert logp.shape == (6, 128) and logp.isfinite().all() and (logp < 0).all()


def test_a_blocks_operators_pass_gradients_on():
    """layer norm, rotary positions and attention in one graph, against the same operators' gradients handed on one by one: the same bits."""
    g = torch.Generator(device="cuda").manual_seed(5)
    r = lambda *s: torch.randn(s, generator=g, device="cuda").bfloat16()  # noqa: E731
    N, H, D = 300, 4, 32
    x, w, b, do = r(N, 3 * H * D), r(3 * H * D), r(3 * H * D), r(N, H, D)
    pos = torch.randint(0, 99, (N, 3), generator=g, device="cuda")
    ends = torch.tensor([0, 100, 101, 300], dtype=torch.int32, device="cuda")
    for t in (x, w, b):
        t.requires_grad_(True)

    def norm(x):
        return ops.layer_norm(x, w, b).view(N, 3 * H, D)

    y = norm(x)
    q, k = ops.rotary(pos, y[:, :H], y[:, H:2 * H], sections=(6, 6, 4))
    o = ops.attention(q, k, y[:, 2 * H:], cu_q=ends, cu_k=ends)
    got = torch.autograd.grad(o, (x, w, b), do)
    y1 = norm(x)
    y2 = y1.detach().requires_grad_(True)
    q1, k1 = ops.rotary(pos, y2[:, :H], y2[:, H:2 * H], sections=(6, 6, 4))
    q2, k2, v2 = (t.detach().requires_grad_(True) for t in (q1, k1, y2[:, 2 * H:]))
    o2 = ops.attention(q2, k2, v2, cu_q=ends, cu_k=ends)
    dq, dk, dv = torch.autograd.grad(o2, (q2, k2, v2), do)
    dy, = torch.autograd.grad((q1, k1), y2, (dq, dk))
    dy[:, 2 * H:] = dv
    want = torch.autograd.grad(y1, (x, w, b), dy)
    assert torch.equal(o, o2) and all(torch.equal(p, s) for p, s in zip(got, want))


def test_the_command(capsys):
    prior.main([os.path.join(GOLDEN, "ref_m1234_model.bin"), "--steps", "20", "--hidden", "64", "--tile", "8", "--layers", "1", "--heads", "4"])
    lines = [json.loads(x) for x in capsys.readouterr().out.splitlines()]
    assert [x["level"] for x in lines] == [0, 1]
    for x in lines:
        assert 0 < x["prior_bits"] < math.inf and 0 <= x["first"] <= x["first_four"] <= 1
