"""A step and autograd's record of its parameters: what it has changed may no longer be differentiated through, what it left alone may."""
import pytest
import torch

from neural_block_textures_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [8, 32])
def test_a_graph_over_a_parameter_that_the_step_left_alone(bits):
    a, b = (torch.randn(30, device="cuda").requires_grad_(True) for _ in range(2))
    opt = ops.AdamW([a, b], state_bits=bits)
    y = (a * b).sum()                                        # keeps both for its backward
    before = a._version, b._version
    opt.step([None, None])
    assert (a._version, b._version) == before
    opt.step([None, torch.ones(30, device="cuda")])
    assert a._version == before[0] and b._version > before[1]
    z = (2.0 * a).square().sum() + y.detach()
    opt.step([None, torch.ones(30, device="cuda")])
    z.backward()
    assert torch.equal(a.grad, 8 * a.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_a_saved_parameter_that_was_skipped():
    a, b = (torch.randn(30, device="cuda").requires_grad_(True) for _ in range(2))
    opt = ops.AdamW([a, b])
    y = (a.square()).sum()
    opt.step([None, torch.ones(30, device="cuda")])
    y.backward()
    assert torch.equal(a.grad, 2 * a.detach())
