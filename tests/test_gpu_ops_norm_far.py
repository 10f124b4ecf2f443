"""layer_norm's gradients in rows so long that the sums over rows need more threads than one dimension of a launch holds."""
import pytest
import torch

from neural_block_textures_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("C", [2 ** 26 - 1, 2 ** 26 + 40])
def test_columns_of_the_longest_rows(C):
    """One row: the bias's gradient is dy itself, the weight's dy h. A sum of a thread's C / 1024 values and of 1024 threads is off by no more than n = C / 1024 + 1024 roundings of the sum of magnitudes, so the mean by
    n u mean|x|, the variance by n u of itself and h by these and half a step."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((1, C), generator=g, device="cuda").bfloat16()
    dy = torch.randn((1, C), generator=g, device="cuda").bfloat16()
    w, b = (torch.ones(C, dtype=torch.bfloat16, device="cuda").requires_grad_(True) for _ in range(2))
    dw, db = torch.autograd.grad(ops.layer_norm(x, w, b), (w, b), dy)
    assert torch.equal(db, dy[0])
    mean, size, var = float(x.double().mean()), float(x.double().abs().mean()), float(x.double().var(correction=0))
    n = (C / 1024 + 1024) * 2.0 ** -24
    worst = 0.0
    for a in range(0, C, 2 ** 24):
        c = slice(a, a + 2 ** 24)
        h = (x[0, c].double() - mean) * (var + 1e-5) ** -0.5
        want = dy[0, c].double() * h
        tol = dy[0, c].double().abs() * n * (size * (var + 1e-5) ** -0.5 + h.abs()) + (2.0 ** -8 + 2.0 ** -21) * want.abs()
        worst = max(worst, float(((dw[c].double() - want).abs() - 1.01 * tol - 1e-30).max()))
    assert worst <= 0
