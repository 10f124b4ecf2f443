"""The operators have no forward-mode derivative, and say so where a tangent would be dropped: also for tensors that need no gradient."""
import pytest
import torch
from torch.autograd import forward_ad

from neural_block_textures_amd import ops

pytestmark = pytest.mark.gpu


def dual(x):
    return forward_ad.make_dual(x, torch.ones_like(x))


@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(grad):
    x, w = torch.randn(4, 200, device="cuda"), torch.randn(6, 200, device="cuda")
    w8 = ops.fp8_quantize(w, 128)
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    with forward_ad.dual_level():
        dx, dw = dual(x.clone().requires_grad_(grad)), dual(w.clone().requires_grad_(grad))
        for call in (lambda: ops.token_logprobs(dx, t, top=2), lambda: ops.fp8_linear(dx, w), lambda: ops.fp8_linear(x, dw), lambda: ops.fp8_linear(dx, w8)):
            with pytest.raises(ValueError, match="no forward-mode derivative"):
                call()
        with torch.no_grad(), pytest.raises(ValueError, match="no forward-mode derivative"):
            ops.fp8_linear(dx, w)
        plain = ops.fp8_linear(x, w)                          # others are not affected
    assert torch.equal(plain, ops.fp8_linear(forward_ad.unpack_dual(x).primal, w))
