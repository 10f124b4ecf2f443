"""attention in float16 where its range ends: probabilities far below a row's largest, and gradients of sequences and rows of very different size."""
import pytest
import torch

from tests.attention_reference import U, check, reference
from neural_block_textures_amd import ops

pytestmark = pytest.mark.gpu


def randn(seed, *shape):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def on_gpu(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


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


def run(q, k, v, do, **kw):
    x = [t.clone().requires_grad_(True) for t in (q, k, v)]
    o = ops.attention(*x, **kw)
    return dict(zip(("o", "dq", "dk", "dv"), (o.detach(), *torch.autograd.grad(o, x, do))))


# lengths of queries and of keys, heads, width (the last: sums in parts)
SIZES = [([300, 260, 5], [300, 260, 5], 2, 2, 64), ([70, 33], [500, 200], 6, 2, 72), ([1, 1, 1], [90, 900, 300], 4, 1, 32), ([260, 300], [260, 300], 2, 1, 128), ([9, 12], [6000, 5000], 2, 1, 128),
         ([3000, 2000], [40, 200], 2, 1, 64)]


@pytest.mark.parametrize("nq,nk,Hq,Hk,D", SIZES)
def test_sequences_of_different_size(nq, nk, Hq, Hk, D):
    """Gradients and values of a sequence that are 10^4 and 30 times another's leave the other's gradients as they are alone, and so does one that is not finite."""
    eq, ek = [0], [0]
    for a, b in zip(nq, nk):
        eq.append(eq[-1] + a)
        ek.append(ek[-1] + b)
    q, do = randn(1, eq[-1], Hq, D).half(), (2e-3 * randn(2, eq[-1], Hq, D)).half()
    k, v = randn(3, ek[-1], Hk, D).half(), (0.3 * randn(4, ek[-1], Hk, D)).half()
    kw = dict(cu_q=on_gpu(eq), cu_k=on_gpu(ek))
    plain = run(q, k, v, do, **kw)
    v[:ek[1]] *= 30
    do[:eq[1]] *= 10000
    got = run(q, k, v, do, **kw)
    for a, b, c, d in zip(eq[:-1], eq[1:], ek[:-1], ek[1:]):
        want = reference(q[a:b], k[c:d], v[c:d], do[a:b], [(0, b - a, 0, d - c)])
        for name, (values, tol) in want.items():
            check(got[name][slice(a, b) if name in ("o", "dq") else slice(c, d)], values, tol, f"{name} of {a}")
    do[0, 0, 0] = float("inf")
    broken = run(q, k, v, do, **kw)
    for x in (got, broken):
        for name in x:
            rest = slice(eq[1] if name in ("o", "dq") else ek[1], None)
            assert torch.equal(x[name][rest], plain[name][rest]), name


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("rows,keys", [(300, 300), (20, 7000)])
def test_rows_of_different_size(D, rows, keys):
    """Gradients of a row that are 10^6 times the others' leave the others' dq as precise as without it."""
    q, k, v, do = randn(1, rows, 2, D).half(), randn(2, keys, 2, D).half(), randn(3, keys, 2, D).half(), (1e-5 * randn(4, rows, 2, D)).half()
    few = do.clone()
    do[7] *= 3000000
    few[7] = 0
    values, tol = reference(q, k, v, few, [(0, rows, 0, keys)])["dq"]
    got = run(q, k, v, do)["dq"]
    keep = [i for i in range(rows) if i != 7]
    check(got[keep], values[keep], tol[keep], "dq")
    assert got[7].isfinite().all()
