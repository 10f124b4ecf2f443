"""attention in float16 where its range ends: probabilities far below a row's largest."""
import pytest
import torch

from tests.attention_reference import U
from neural_block_textures_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("below", [5.0, 10.0, 14.0, 16.5, 17.25, 17.5, 19.0, 20.5])
@pytest.mark.parametrize("rows,keys,heads", [(1, 60000, 1), (200, 9000, 1), (3000, 6000, 32)])     # (the last has blocks enough: its sums are not made in parts)
def test_one_key_above_many(below, rows, keys, heads):
    """One key's score is `below` above all others', whose small probabilities make up the result: its value is 0, theirs 0.5 to 1. A probability is rounded to float16 at 2^7 times its share of the largest: half a step
    of what is normal, else 2^-25 2^-7. The scores are exact."""
    D = 64
    q, k, v = torch.zeros(rows, heads, D, device="cuda").half(), torch.zeros(keys, 1, D, device="cuda").half(), (0.5 + 0.5 * torch.rand(keys, 1, D, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")).half()
    q[..., 0], k[..., 0] = 1, -below
    k[0, 0, 0], v[0] = 0, 0
    got = ops.attention(q, k, v, causal=False, scale=1.0).double()
    p = torch.softmax(k[:, 0, 0].double(), 0)
    want, size = p @ v[:, 0].double(), v[:, 0].double().abs().sum(0)
    h = 2.0 ** -11
    tol = (3 * h + (keys + 8) * U + 2.0 ** -22) * want + 2.0 ** -32 * size * (1 + want)    # (2^-22: the exponential's ulp and its argument's rounding; the sum of probabilities is off by as much as 2^-32 each)
    assert ((got - want).abs() <= 1.01 * tol).all(), float(((got - want).abs() / tol).max())
