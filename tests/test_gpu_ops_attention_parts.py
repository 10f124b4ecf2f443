"""Sums that few blocks would make alone, in parts: of keys (outputs, queries' gradients) and of rows (keys' and values' gradients)."""
import pytest
import torch

from tests.attention_reference import check, reference
from neural_block_textures_amd import ops

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda()


def ends(lengths):
    return torch.tensor([0, *lengths]).cumsum(0).int().cuda()


# few queries of many keys; many of few; one long sequence; parts that have no keys (short sequences beside a long one, none at all)
CASES = [([9, 27], [2900, 4100], 4, 1, 128), ([5], [9000], 2, 2, 16), ([1500], [1500], 2, 1, 40), ([1, 0, 40, 1700], [1, 0, 3500, 1700], 3, 1, 64), ([700, 3], [5, 2700], 1, 1, 96), ([0, 50], [4000, 0], 1, 1, 32),
         ([130, 6, 130], [130, 5000, 20], 2, 2, 128)]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("nq,nk,Hq,Hk,D", CASES)
def test_few_blocks(nq, nk, Hq, Hk, D, dtype, causal):
    """... with rows behind the last sequence, keys alike but for a little, against the definition; alone, each gradient is the same."""
    t = TYPES[dtype]
    eq, ek = ends(nq), ends(nk)
    q, do = randn(1, sum(nq) + 3, Hq, D).to(t), (0.1 * randn(2, sum(nq) + 3, Hq, D)).to(t)
    k, v = (1 + 0.25 * randn(3, sum(nk) + 5, Hk, D)).to(t), randn(4, sum(nk) + 5, Hk, D).to(t)

    def grads(wanted):
        x = [a.clone().requires_grad_(i in wanted) for i, a in enumerate((q, k, v))]
        o = ops.attention(*x, causal=causal, cu_q=eq, cu_k=ek)
        return o.detach(), dict(zip(wanted, torch.autograd.grad(o, [x[i] for i in wanted], do)))

    o, g = grads([0, 1, 2])
    a, b = [0, *torch.tensor(nq).cumsum(0).tolist()], [0, *torch.tensor(nk).cumsum(0).tolist()]
    want = reference(q, k, v, do, [(a[i], a[i + 1], b[i], b[i + 1]) for i in range(len(nq))], causal)
    for name, got in (("o", o), ("dq", g[0]), ("dk", g[1]), ("dv", g[2])):
        check(got, *want[name], name)
    for i in range(3):
        assert torch.equal(grads([i])[1][i], g[i])
    with torch.no_grad():
        check(ops.attention(q, k, v, causal=causal, cu_q=eq, cu_k=ek), *want["o"], "o")
