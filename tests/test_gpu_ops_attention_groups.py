"""attention with 32 to 1024 query heads to a key head (a tile of rows is then few queries, or lies inside one), and one sequence alone among no others."""
import pytest
import torch

from tests.attention_reference import check, reference
from neural_block_textures_amd import ops

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def randn(seed, *shape):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def both(q, k, v, do, spans, causal, **kw):
    x = [t.clone().requires_grad_(True) for t in (q, k, v)]
    o = ops.attention(*x, causal=causal, **kw)
    got = dict(zip(("o", "dq", "dk", "dv"), (o, *torch.autograd.grad(o, x, do))))
    for name, (values, tol) in reference(q, k, v, do, spans, causal).items():
        check(got[name], values, tol, name)


# query heads, key heads, width, lengths of queries and keys
CASES = [(32, 1, 64, [3, 40, 0, 17], [70, 40, 5, 200]), (64, 1, 32, [7, 30], [200, 9]), (64, 2, 128, [40, 1], [40, 130]), (65, 1, 64, [5, 33], [5, 150]), (96, 1, 128, [21], [65]), (128, 1, 72, [9, 2], [9, 190]),
         (256, 2, 32, [6], [300]), (999, 1, 64, [3, 4], [50, 4]), (1024, 1, 32, [3, 5], [5, 129]), (1024, 1, 128, [2], [2500])]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("Hq,Hk,D,nq,nk", CASES)
def test_wide_groups(Hq, Hk, D, nq, nk, dtype, causal):
    print("attention", Hq, Hk, D, nq, nk, dtype, causal, flush=True)
    t = TYPES[dtype]
    eq, ek = ([0, *torch.tensor(n).cumsum(0).tolist()] for n in (nq, nk))
    q, do = randn(1, eq[-1], Hq, D).to(t), (0.1 * randn(2, eq[-1], Hq, D)).to(t)
    k, v = randn(3, ek[-1], Hk, D).to(t), (0.5 + randn(4, ek[-1], Hk, D)).to(t)
    ends = [torch.tensor(e, dtype=torch.int32, device="cuda") for e in (eq, ek)]
    both(q, k, v, do, list(zip(eq[:-1], eq[1:], ek[:-1], ek[1:])), causal, cu_q=ends[0], cu_k=ends[1])


@pytest.mark.parametrize("n", [1, 5, 130])
def test_one_sequence(n):
    q, k, v, do = (randn(s, n, 1, 16).half() for s in (1, 2, 3, 4))
    e = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    both(q, k, v, do, [(0, n, 0, n)], True, cu_q=e, cu_k=e)
