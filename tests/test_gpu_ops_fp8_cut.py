"""How far a product of two 8-bit matrices may be from the exact one, for any codes: rows of large and of subnormal ones, mixed and with zeros.

The matrix instruction aligns eight neighbouring products to the largest exponent among them (the sum of its factors', where a subnormal code's is that of
2^-6, and a factor of 0 does not count) and cuts each off 13 bits below: seven of them lose less than 2^-13 of that power each, the largest itself
nothing. The eights' sums are added in 32 bits: 2^-24 of the magnitudes' sum for each addition, and the result's own rounding."""
import pytest
import torch

from tests.test_gpu_ops_fp8 import HALF, gen, ops

pytestmark = pytest.mark.gpu


def codes(seed, R, K):
    """rows whose codes lie in different ranges, some of them subnormal, with zeros among them; exponent bytes 120 to 130"""
    g = gen(seed)
    c = torch.randint(0, 127, (R, K), generator=g, device="cuda")          # (127 and 255 are NaN)
    top = torch.tensor([127, 8, 127, 20, 3, 60], device="cuda")[torch.arange(R, device="cuda") % 6]
    c = c % top[:, None]
    c[torch.arange(R, device="cuda") % 5 == 4] *= (torch.rand((1, K), generator=g, device="cuda") < 0.3)
    c = c + 128 * torch.randint(0, 2, (R, K), generator=g, device="cuda")
    whole = torch.zeros((R, -(-K // 128) * 128), dtype=torch.uint8, device="cuda")
    whole[:, :K] = c.to(torch.uint8)
    return whole


def tensor(seed, R, K, rows):
    e = torch.zeros((-(-R // rows), -(-K // 512) * 4), dtype=torch.uint8, device="cuda")
    n = -(-K // 128)
    e[:, :n] = torch.randint(120, 131, (e.shape[0], n), generator=gen(seed + 1), device="cuda").to(torch.uint8)
    return ops().Fp8Tensor(codes(seed, R, K), e, (R, K), rows)


def exponents(t):
    """of each value as the instruction takes it; far below all others for zeros"""
    R, K = t.shape
    c = t.codes.int() & 127
    scale = t.exps.int().repeat_interleave(t.block_rows, 0)[:R].repeat_interleave(128, 1)[:, :t.codes.shape[1]] - 127
    return torch.where(c == 0, -10000, (c >> 3).clamp_min(1) - 7 + scale)


@pytest.mark.parametrize("M,N,K", [(1, 60, 300), (16, 70, 1030), (30, 90, 513), (70, 130, 700), (300, 200, 260), (64, 64, 7000), (2100, 1100, 128)])
@pytest.mark.parametrize("rows", [(1, 128), (1, 1)])
def test_any_codes(M, N, K, rows):
    print("fp8 cut", M, N, K, rows, flush=True)
    a, b = tensor(M, M, K, rows[0]), tensor(N + 7, N, K, rows[1])
    A, B = a.values().double(), b.values().double()
    want, size = A @ B.t(), A.abs() @ B.abs().t()
    lost = torch.zeros_like(want)
    ea, eb = exponents(a), exponents(b)
    for k in range(0, ea.shape[1], 8):
        most = (ea[:, None, k] + eb[None, :, k])
        for j in range(1, 8):
            most = torch.maximum(most, ea[:, None, k + j] + eb[None, :, k + j])
        lost += 7 * torch.pow(2.0, (most - 13).double())
    adds = ea.shape[1] / 8 + 64
    for dtype in (torch.float32, torch.bfloat16):
        got = ops().fp8_matmul(a, b, dtype).double()
        bound = lost + adds * 2.0 ** -24 * size + (want.abs() + lost) * HALF[dtype] * 1.01
        bad = ~((got - want).abs() <= bound)
        assert not bad.any(), (int(bad.sum()), got[bad][:3].tolist(), want[bad][:3].tolist(), bound[bad][:3].tolist())
