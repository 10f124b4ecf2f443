"""Long rows' sums lose nothing of many small terms beside large ones: log p and entropy against 64 bits to a bound that hardly grows with the row.

With u = 2^-24 and d = (x - largest) / (T ln 2): an exponential is good to 2 u, its argument to 2.3 u |d| (two roundings of 1 / T ln 2, one of d), which makes
2 u E|d| of the sum, E|d| <= (H + 1) / ln 2. A sum has 16 terms of a chunk, 16 chunks, V / 16384 of these (one wave a row, 64 lanes), then 25 of
lanes, waves and parts; a running largest value that rises costs 3 u each time, 12 times in a random row: below (112 + V / 16384) u in all."""
import pytest
import torch

from tests.test_gpu_ops_logprobs import U, close, ops, reference

pytestmark = pytest.mark.gpu


def rows(kind, N, V, dtype):
    gen = torch.Generator(device="cuda").manual_seed(V)
    if kind == "random":
        return (torch.randn((N, V), generator=gen, device="cuda") * 2.5).to(dtype)
    x = torch.full((N, V), -1e10 if kind == "alike" else -16.75, dtype=torch.float32, device="cuda").to(dtype)
    if kind == "peak":                                     # one value, the others a little below 2^-24 of it each
        x[:, 77] = 0
    if kind == "peaks":                                    # one in each lane's first values
        x[:, 0:1024:8] = 0
    return x


@pytest.mark.parametrize("kind", ["peak", "peaks", "random", "alike"])
@pytest.mark.parametrize("N,V,top,dtype", [(4100, 131072, 4, torch.bfloat16), (4100, 50001, 4, torch.float16), (600, 131072, 0, torch.bfloat16), (600, 131072, 0, torch.float32),
                                           (2100, 131072, 4, torch.float32), (3, 131072, 0, torch.bfloat16), (40, 9001, 8, torch.float32), (4100, 2000, 4, torch.bfloat16)])
def test_sums(N, V, top, dtype, kind):
    if kind == "alike" and dtype == torch.float16:
        pytest.skip("a 16-bit float ends before the row's path does")
    print("logprobs sums", N, V, top, dtype, kind, flush=True)
    x = rows(kind, N, V, dtype)
    T = 0.7 if kind == "random" else 1.0
    t = torch.full((N,), 77, device="cuda")
    t[1::2] = V - 1
    r = ops().token_logprobs(x, t, top=top, temperature=T)
    few = torch.tensor([0, 1, N // 2, N - 1], device="cuda")
    w = reference(x[few], t[few], top, T, -100)
    base = U * (112 + V / 16384)
    error = base + 2 * U * (w["entropy"] + 1) / 0.69
    close(r.logprob[few], w["logprob"], 4 * U * w["logprob"].abs() + error, "logprob")
    close(r.entropy[few], w["entropy"], error * (2 + w["entropy"]), "entropy")
