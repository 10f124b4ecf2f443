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


def test_a_run_goes_on_bit_for_bit_in_an_optimizer_of_another_seed():
    grads = [torch.randn(300, generator=torch.Generator(device="cuda").manual_seed(k), device="cuda") for k in range(6)]
    ends = []
    for cut in (6, 3):
        p = torch.full((300,), 0.5, device="cuda")
        opt = ops.AdamW([p], state_bits=8, seed=2 ** 64 - 1)
        for g in grads[:cut]:
            opt.step([g])
        if cut < 6:
            saved, opt = opt.state_dict(), ops.AdamW([p], state_bits=8, seed=77)
            opt.load_state_dict(saved)
            for g in grads[cut:]:
                opt.step([g])
        ends.append([p, *opt.moments()])
    assert all(torch.equal(a, b) for a, b in zip(*ends))
    old = {k: v for k, v in opt.state_dict().items() if k != "seed"}
    other = ops.AdamW([torch.zeros(300, device="cuda")], state_bits=8, seed=9)
    other.load_state_dict(old)
    assert other.seed == 9


def test_seeds_out_of_range():
    for seed in (-1, 2 ** 64):
        with pytest.raises(ValueError, match="seed must be"):
            ops.AdamW([torch.zeros(3, device="cuda")], seed=seed)
