"""AdamW where the root's argument is a subnormal 32-bit number and eps does not hide it, and where eps is one itself.

The step is held against the formula in 64 bits on the averages that the step itself has stored (32-bit state), so that only the update's own
arithmetic is asked about: 12 u of the update and 3 u of the weight, u = 2^-24, as in test_gpu_ops_adamw.py. With an 8-bit state the averages are not
stored as they were used: from the formula's, whose subnormal v is off by at most 2 units of 2^-149, and whose m, two terms that may cancel, by 3 u of these."""
import pytest
import torch

from tests.test_gpu_ops_adamw import U, gen, near, ops

pytestmark = pytest.mark.gpu
LR, B1, B2, DECAY = 1e-2, 0.9, 0.999, 0.1


def gradients(n, size, seed, zeros):
    g = torch.randn(n, generator=gen(seed), device="cuda")
    g = torch.sign(g) * (g.abs() + 0.2) * size
    if zeros:
        g[::7] = 0
    return g


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("eps,size,zeros", [(0.0, 1e-19, False), (0.0, 2e-20, False), (0.0, 1e-3, False), (0.0, 1e12, False), (1e-30, 1e-19, True), (1e-40, 1e-19, True), (1e-40, 1e-3, True), (1e-21, 3e-20, True), (1e-12, 1e-6, True),
                                            (1e-8, 1e-19, True), (1e-8, 1e-9, True)])
def test_small_gradients_and_eps(eps, size, zeros, master, bits):
    print("adamw small", eps, size, master, bits, flush=True)
    n = 5003
    p = torch.randn(n, generator=gen(1), device="cuda")
    opt = ops().AdamW([p], lr=LR, betas=(B1, B2), eps=eps, weight_decay=DECAY, state_bits=bits, master=master)
    eps32 = float(torch.tensor(eps, dtype=torch.float32))
    for t in range(1, 4):
        g = gradients(n, size, 10 + t, zeros)
        q, before = p.clone().double(), [x[:n].double() for x in opt.moments()]
        opt.step([g])
        m, v = (x[:n].double() for x in opt.moments())
        wide = torch.zeros(n, dtype=torch.float64, device="cuda")
        if bits == 8:
            m, v = B1 * before[0] + (1 - B1) * g.double(), B2 * before[1] + (1 - B2) * g.double() ** 2
            m, v = torch.where(m.abs() < 2.0 ** -149, 0.0, m), torch.where(v < 2.0 ** -149, 0.0, v)
            wide = torch.where(v > 0, (2 * 2.0 ** -149 / v.clamp_min(1e-60)).clamp_max(4.0), 0.0)
            wide += 3 * U * (B1 * before[0].abs() + (1 - B1) * g.double().abs()) / m.abs().clamp_min(1e-60)
        up = LR / (1 - B1 ** t) * m / (torch.sqrt(v / (1 - B2 ** t)) + eps32)
        up = torch.where(m == 0, 0.0, up) if eps > 0 else up
        assert torch.isfinite(up).all()
        near(p, q * (1 - LR * DECAY) - up, up.abs() * (12 * U + wide) + 3 * U * q.abs() + 2.0 ** -149, (t, "p"))
