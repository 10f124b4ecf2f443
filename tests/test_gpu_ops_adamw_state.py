"""An optimizer's state as it is saved and taken back: all of it or nothing."""
import pytest
import torch

from neural_block_textures_amd import ops

pytestmark = pytest.mark.gpu


def made(bits, seed=5, calls=2):
    params = [torch.full((n,), 0.5, device="cuda") for n in (300, 7)]
    opt = ops.AdamW(params, state_bits=bits, master=True, seed=seed)
    for k in range(calls):
        opt.step([torch.full((300,), 0.1 + k, device="cuda"), None])
    return opt


def held(opt):
    return [t.clone() for t in (opt.exp_avg, opt.exp_avg_sq, opt.exp_avg_exp, opt.exp_avg_sq_exp, opt.master) if t is not None], opt.steps.tolist(), opt.calls


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("change", [{"exp_avg_sq": None}, {"exp_avg_sq": torch.zeros(5)}, {"master": torch.zeros(5)}, {"step": [1, 2, 3]}, {"step": -1}, {"step": [1, -1]}, {"step": 1.5}, {"calls": -1}])
def test_a_state_that_does_not_fit_changes_nothing(bits, change):
    state, opt = made(bits, calls=4).state_dict(), made(bits)
    before = held(opt)
    with pytest.raises(ValueError, match=next(iter(change)) + " must be"):
        opt.load_state_dict({**state, **change})
    after = held(opt)
    assert all(torch.equal(a, b) for a, b in zip(before[0], after[0])) and before[1:] == after[1:]
    opt.load_state_dict(state)
    assert opt.steps.tolist() == [4, 0] and opt.calls == 4
    for step, want in ((3, [3, 3]), (3.0, [3, 3]), ([2], [2, 2]), (torch.tensor([5, 6]), [5, 6])):
        opt.load_state_dict({**state, "step": step})
        assert opt.steps.tolist() == want
