"""What a step reads and writes is what its optimizer was made for, whatever has happened to the tensors since; a refused step changes nothing."""
import pytest
import torch

from neural_block_textures_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("change", ["shorter", "type", "layout", "gone"])
def test_a_parameter_that_has_changed_in_place(change):
    whole = torch.zeros(40, 50, device="cuda")
    q, other = torch.nn.Parameter(whole), torch.nn.Parameter(torch.ones(7, device="cuda"))
    opt = ops.AdamW([other, q])
    reason = "another size, type or layout"
    if change == "shorter":
        q.data = whole[:3]
    elif change == "type":
        q.data = whole.view(torch.bfloat16)
    elif change == "layout":
        q.data = whole.t()
    else:
        q.data, reason = torch.empty(0, device="cuda"), "moved"
    with pytest.raises(ValueError, match=reason):
        opt.step([torch.ones(7, device="cuda"), torch.ones_like(q)])
    assert opt.calls == 0 and not opt.steps.any() and (other == 1).all()
    q.data = whole                                            # as it was
    opt.step([torch.ones(7, device="cuda"), torch.ones(40, 50, device="cuda")])
    assert opt.calls == 1 and (whole != 0).all()
