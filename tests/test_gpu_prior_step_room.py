"""A step for single symbols whose lengths leave the cache: the last (first) place is written, and nothing outside of the tile's room."""
import pytest
import torch

from neural_block_textures_amd import prior

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("length", [10, 11, 2 ** 31 - 1, -1, -7])
def test_lengths_that_leave_the_cache(length):
    p = prior.TilePrior(13, 64, 4, 2, 4, 1)
    whole = [[torch.full((5, 10, 4, 16), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)] for _ in p.blocks]
    cache = [(k[1:4], v[1:4]) for k, v in whole]
    lens = torch.tensor([3, length, 9], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    with torch.no_grad():
        x, positions = torch.randn(3, 13, generator=g, device="cuda").bfloat16(), torch.zeros(3, 3, dtype=torch.int64, device="cuda")
        logits = p.step(x, positions, cache, lens)
        alone = p.step(x[::2].contiguous(), positions[::2], [(k[::2].clone(), v[::2].clone()) for k, v in cache], lens[::2])
    assert logits.shape == (3, 4) and torch.equal(logits[::2], alone)
    for k, v in whole:
        for room in (k, v):
            changed = (room != 7).flatten(2).any(-1)
            want = torch.zeros_like(changed)
            want[1, 3] = want[2, 9 if length > 0 else 0] = want[3, 9] = True
            assert torch.equal(changed, want)


def test_no_graph_is_kept():
    """... from step to step, where a caller has gradients on."""
    p = prior.TilePrior(13, 64, 4, 2, 4, 1)
    cache, lens = p.cache(2, 10), torch.zeros(2, dtype=torch.int32, device="cuda")
    for _ in range(3):
        logits = p.step(torch.ones(2, 13, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, 3, dtype=torch.int64, device="cuda"), cache, lens)
        lens += 1
    assert not logits.requires_grad and not any(room.requires_grad for pair in cache for room in pair)
