"""A training layer over more rows than one product's sum takes (2^23): the weights' gradient is the sum of those of its parts."""
import pytest
import torch

from neural_block_textures_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,K,N,need_x,dtype", [(2 ** 23 + 300, 9, 5, True, torch.float32), (2 ** 24 + 2 ** 10 + 7, 33, 40, False, torch.bfloat16)])
def test_more_rows_than_2_23(M, K, N, need_x, dtype):
    print("fp8 far", M, K, N, need_x, dtype, flush=True)
    gen = torch.Generator(device="cuda").manual_seed(3)
    ints = lambda *s: torch.randint(-1, 2, s, generator=gen, device="cuda").to(dtype)  # noqa: E731
    x, w, dy = ints(M, K), ints(N, K), ints(M, N)
    x.requires_grad_(need_x)
    w.requires_grad_(True)
    y = ops.fp8_linear(x, w)
    got = torch.autograd.grad(y, [x, w] if need_x else [w], dy)
    # sums of -1, 0 and 1: exact, then rounded once to the weights' type
    want = sum(a.double().t() @ b.double() for a, b in zip(dy.split(2 ** 22), x.detach().split(2 ** 22)))
    assert torch.equal(got[-1], want.to(dtype))
    if need_x:
        assert torch.equal(got[0], dy @ w.detach())
    for a in (0, 2 ** 23 - 100, M - 200):
        assert torch.equal(y[a:a + 200].detach(), (x[a:a + 200] @ w.t()).detach())
