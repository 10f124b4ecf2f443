"""Sizes of zero are no error, wherever among the axes they stand, for tensors as they are made and cut out of larger ones."""
import pytest
import torch

from neural_block_textures_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(0,), (0, 3), (3, 0), (2, 0, 3), (0, 2, 3), (2, 3, 0), (2, 3, 0, 4), (1, 0, 1), (4, 2, 0, 1, 3)])
@pytest.mark.parametrize("V", [1, 40, 3000])
def test_token_logprobs(shape, V):
    for x in (torch.zeros((*shape, V), device="cuda"), torch.zeros((*(s + 2 for s in shape), V + 3), device="cuda")[tuple(slice(0, s) for s in shape)][..., 1:V + 1]):
        x.requires_grad_(True)
        t = torch.zeros(shape, dtype=torch.int64, device="cuda")
        r = ops.token_logprobs(x, t, top=1)
        assert r.logprob.shape == shape and r.entropy.shape == shape and r.top_ids.shape == (*shape, 1) and r.top_logprobs.shape == (*shape, 1)
        dx, = torch.autograd.grad(r.logprob.sum() + r.top_logprobs.sum(), x)
        assert dx.shape == x.shape


@pytest.mark.parametrize("shape,K,N", [((0,), 8, 5), ((2, 0, 3), 8, 5), ((4,), 0, 5), ((4,), 8, 0), ((0, 2), 0, 0), ((20,), 0, 300)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_fp8_linear(shape, K, N, dtype):
    x, w = torch.ones((*shape, K), device="cuda", dtype=dtype, requires_grad=True), torch.ones((N, K), device="cuda", dtype=dtype, requires_grad=True)
    y = ops.fp8_linear(x, w)
    assert y.shape == (*shape, N) and not y.any()
    dx, dw = torch.autograd.grad(y.sum(), (x, w))
    assert dx.shape == x.shape and dw.shape == w.shape and not dx.any() and not dw.any()
    z = ops.fp8_linear(x.detach(), ops.fp8_quantize(w.detach(), 128))
    assert z.shape == y.shape and not z.any()


def test_optimizer_of_nothing():
    for bits in (8, 32):
        p = torch.zeros((0, 4), device="cuda")
        opt = ops.AdamW([p], state_bits=bits, master=True)
        opt.step([torch.zeros((0, 4), device="cuda")])
        assert opt.calls == 1 and opt.moments()[0].numel() == 0
