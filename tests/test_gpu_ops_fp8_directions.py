"""fp8_linear's gradient against differences along directions of their own."""
import pytest
import torch

from tests.test_gpu_ops_fp8 import gen, ops, whole_numbers

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", range(6))
def test_gradient_along_a_direction(seed):
    """On values that 8 bits hold exactly the layer is the product itself, linear in each operand: whole differences are exact."""
    x, w = whole_numbers(1, 64, 128, 1).requires_grad_(True), whole_numbers(2, 32, 128, 128).requires_grad_(True)
    dy = torch.randint(-2, 3, (64, 32), generator=gen(3), device="cuda").float()
    dx, dw = torch.autograd.grad(ops().fp8_linear(x, w), (x, w), dy)
    f = lambda a, b: ((a @ b.t()) * dy.double()).sum()  # noqa: E731
    X, W = x.detach().double(), w.detach().double()
    g = gen(100 + seed)
    u, v = (torch.randint(-3, 4, t.shape, generator=g, device="cuda").double() for t in (X, W))
    assert f(X + u, W) - f(X - u, W) == 2 * (dx.double() * u).sum()
    assert f(X, W + v) - f(X, W - v) == 2 * (dw.double() * v).sum()
