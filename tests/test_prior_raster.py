"""Contexts as a decoder has them: a plane that is filled in its raster order gives each symbol the context that the finished plane does; what the command and the walk refuse."""
import numpy as np
import pytest
import torch

from neural_block_textures_amd import prior


@pytest.mark.parametrize("shape,alphabet", [((5, 7, 3), 9), ((1, 4, 2), 1), ((6, 1, 1), 4)])
def test_contexts_of_what_is_known(shape, alphabet):
    r = np.random.default_rng(1)
    sym = torch.from_numpy(r.integers(0, alphabet, shape))
    whole, known = prior.Contexts(sym, alphabet), prior.Contexts(torch.from_numpy(r.integers(0, alphabet, shape)), alphabet)     # (what is not known yet may be anything)
    for i in range(sym.numel()):
        at = torch.tensor([i])
        assert torch.equal(known.rows(at), whole.rows(at)), i
        known.put(at, sym.reshape(-1)[at])
    assert torch.equal(known.values, whole.values) and torch.equal(known.padded, whole.padded)


def test_tiles_in_step_would_need_symbols_to_come():
    """Tiles that go on together, each symbol in turn, have contexts of symbols that other tiles have not reached: why a decoder goes through the plane."""
    tiles = prior.Tiles((8, 8, 1), 4, "cpu")
    turn = torch.empty(64, dtype=torch.int64)
    for order in tiles.order:
        turn[order] = torch.arange(len(order))
    left = turn.view(8, 8)[:, 3]                            # of the texels to the left of the second column of tiles
    assert (left[0] > turn.view(8, 8)[0, 4]).all()


@pytest.mark.parametrize("n", [-1, 33])
def test_counts(n):
    sym = torch.zeros((4, 4, 2), dtype=torch.int64)
    with pytest.raises(ValueError, match="0 to 32 symbols"):
        prior.raster_logprobs(prior.TilePrior(13, 64, 4, 1, 4, 1, "cpu"), prior.Tiles(sym.shape, 4, "cpu"), sym, 4, n)


@pytest.mark.parametrize("args", [["--stepped", "5"], ["--tile", "8", "--stepped", "-1"]])
def test_the_command_refuses(args, capsys):
    with pytest.raises(SystemExit):
        prior.main(["model.bin", *args])
    assert "--stepped takes" in capsys.readouterr().err
