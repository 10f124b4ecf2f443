"""The learned prior end to end: it prices a plane with structure far below its histogram, near what the plane was drawn from; its
figures are those of its own logits in 64 bits; and the command runs on a model file."""
import json
import math
import os

import numpy as np
import pytest
import torch

from neural_block_textures_amd import prior
from tests.helpers import GOLDEN

pytestmark = pytest.mark.gpu


def plane(H, W, C, alphabet, seed):
    """A smooth plane plus uniform noise of 8 neighbouring symbols: 3 bits a symbol are noise, whatever the histogram says."""
    g = np.random.default_rng(seed)
    y, x = np.mgrid[0:H, 0:W]
    base = np.stack([(np.sin(x / 37 + c) + np.cos(y / 23 - c)) * 0.2 + 0.5 for c in range(C)], -1) * (alphabet - 9)
    return np.clip(base.round().astype(np.int64) + g.integers(0, 8, (H, W, C)), 0, alphabet - 1)


@pytest.mark.parametrize("state_bits", [8, 32])
def test_a_plane_of_known_noise(state_bits):
    print("prior", state_bits, flush=True)
    sym = plane(192, 256, 2, 64, 1)
    dev = torch.from_numpy(sym).cuda()
    p, ctx = prior.fit(dev, 64, steps=400, hidden=128, batch=16384, lr=4e-3, state_bits=state_bits)
    r = prior.price(p, ctx, dev, batch=30011)
    h = prior.histogram_bits(sym)
    print(h, r, flush=True)
    assert h > 4.5 and 2.9 < r["prior_bits"] < h - 0.7       # at least half of what the histogram wastes
    assert abs(r["expected_bits"] - r["prior_bits"]) < 0.3
    assert 0.05 < r["first"] < r["first_four"] < 1


def test_the_price_is_that_of_the_logits():
    sym = plane(40, 50, 3, 200, 2)
    dev = torch.from_numpy(sym).cuda()
    p, ctx = prior.fit(dev, 200, steps=5, hidden=64, batch=1000)
    r = prior.price(p, ctx, dev, batch=777)
    with torch.no_grad():
        logits = torch.cat([p.logits(ctx.rows(a), p.laid_out()) for a in torch.arange(sym.size, device="cuda").split(777)]).double()
    logp = torch.log_softmax(logits, 1)
    want = -logp.gather(1, dev.reshape(-1, 1)).mean().item() / math.log(2)
    entropy = -(logp * logp.exp()).sum(1).mean().item() / math.log(2)
    assert abs(r["prior_bits"] - want) < 1e-5 * want and abs(r["expected_bits"] - entropy) < 1e-5 * entropy


def test_the_command(capsys):
    prior.main([os.path.join(GOLDEN, "ref_m1234_model.bin"), "--steps", "150", "--hidden", "128"])
    lines = [json.loads(x) for x in capsys.readouterr().out.splitlines()]
    print(lines, flush=True)
    assert [x["level"] for x in lines] == [0, 1]
    for x in lines:
        assert 0 < x["prior_bits"] < x["histogram_bits"] + 0.05 and 0 <= x["first"] <= x["first_four"] <= 1
