"""What the prior over tiles refuses before anything is on the GPU, and how it cuts a plane."""
import pytest
import torch

from neural_block_textures_amd import prior


@pytest.mark.parametrize("kw", [{"steps": -1}, {"hidden": 0}, {"batch": 0}, {"sym": torch.zeros((0, 4, 2), dtype=torch.int64)}])
def test_fit(kw):
    sym = kw.pop("sym", torch.zeros((4, 4, 2), dtype=torch.int64))
    with pytest.raises(ValueError, match="are needed"):
        prior.fit_tiles(sym, 4, 4, **kw)


@pytest.mark.parametrize("hidden,heads,layers", [(64, 3, 1), (64, 16, 1), (512, 2, 1), (64, 4, 0), (64, 0, 1)])
def test_heads(hidden, heads, layers):
    with pytest.raises(ValueError, match="blocks and heads"):
        prior.TilePrior(13, hidden, 4, layers, heads, 1, "cpu")


def test_tiles():
    with pytest.raises(ValueError, match="1 texel"):
        prior.Tiles((4, 4, 1), 0, "cpu")
    t = prior.Tiles((5, 7, 2), 4, "cpu")
    assert t.lengths == [32, 24, 8, 6] and t.order[1].tolist() == [2 * (7 * y + x) + c for y in range(4) for x in range(4, 7) for c in range(2)]


@pytest.mark.parametrize("dim", [8, 16, 32, 40, 128])
def test_sections(dim):
    p = prior.TilePrior(13, 2 * dim, 4, 1, 2, 1, "cpu")
    assert sum(p.sections) == dim // 2 and min(p.sections) >= 1
