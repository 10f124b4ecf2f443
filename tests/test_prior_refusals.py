"""What the prior and its optimizer refuse before anything is on the GPU."""
import math

import pytest
import torch

from neural_block_textures_amd import ops, prior


@pytest.mark.parametrize("kw", [{"steps": -1}, {"hidden": 0}, {"batch": 0}, {"sym": torch.zeros((0, 4, 2), dtype=torch.int64)}])
def test_fit(kw):
    sym = kw.pop("sym", torch.zeros((4, 4, 2), dtype=torch.int64))
    with pytest.raises(ValueError, match="are needed"):
        prior.fit(sym, 4, **kw)


@pytest.mark.parametrize("kw", [{"lr": math.nan}, {"eps": math.nan}, {"weight_decay": math.nan}, {"betas": (0.9,)}, {"betas": (0.9, 0.9, 0.9)}, {"betas": (0.9, math.nan)}])
def test_adamw(kw):
    with pytest.raises(ValueError, match="must not be negative, the two betas"):
        ops.AdamW([torch.zeros(3)], **kw)
