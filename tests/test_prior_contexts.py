"""The prior's contexts and symbols without a GPU: a context holds nothing of the symbol itself or of later ones, and a level's symbols are
its values' ranks."""
import os

import numpy as np
import pytest
import torch

from neural_block_textures_amd import decode, prior
from tests.helpers import GOLDEN


def test_contexts_are_causal():
    g = torch.Generator().manual_seed(1)
    sym = torch.randint(0, 50, (5, 7, 3), generator=g)
    at = torch.arange(sym.numel())
    base = prior.Contexts(sym, 50).rows(at).float()
    assert base.shape == (105, 19)
    for i in (0, 1, 20, 52, 104):
        changed = sym.clone().reshape(-1)
        changed[i] = (changed[i] + 25) % 50
        other = prior.Contexts(changed.view_as(sym), 50).rows(at).float()
        same = (other == base).all(1)
        assert same[:i + 1].all()                             # nothing at or before it
        if i < 104:
            y, x, c = i // 21, i // 3 % 7, i % 3
            later = [(y, x, d) for d in range(c + 1, 3)] + [(y, x + 1, d) for d in range(3) if x < 6]
            later += [(y + 1, x + dx, d) for dx in (-1, 0, 1) for d in range(3) if y < 4 and 0 <= x + dx < 7]
            want = torch.zeros(105, dtype=torch.bool)
            for p, q, d in later:
                want[(p * 7 + q) * 3 + d] = True
            assert torch.equal(~same, want)


def test_symbols_of_a_model_file():
    m = decode.load(os.path.join(GOLDEN, "ref_m1234_model.bin"))
    levels = prior.level_symbols(m)
    assert [l for l, _, _ in levels] == list(range(len(m.layout.levels)))
    for (l, sym, alphabet), (W, H, C, _) in zip(levels, m.layout.levels):
        assert sym.shape == (H, W, C) and alphabet <= 256 and sym.min() == 0 and sym.max() == alphabet - 1
        z = m.z[m.layout.offsets[l]:][:W * H * C].reshape(-1, C)
        for c in range(C):
            order = np.argsort(z[:, c], kind="stable")
            assert (np.diff(sym.reshape(-1, C)[order, c]) >= 0).all()
            assert len(np.unique(z[:, c])) == sym[..., c].max() + 1


def test_a_continuous_level_is_refused():
    m = decode.load(os.path.join(GOLDEN, "ref_m1234_model.bin"), q8=False)
    m.z = np.linspace(0, 1, m.z.size, dtype=np.float32)
    with pytest.raises(ValueError, match="continuous"):
        prior.level_symbols(m)


def test_histogram_bits():
    sym = np.array([0, 0, 1, 1, 0, 1, 2, 3]).reshape(2, 2, 2)      # channel 0: 0 1 0 2, channel 1: 0 1 1 3
    assert abs(prior.histogram_bits(sym) - 1.5) < 1e-12
