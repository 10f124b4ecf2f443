"""rotary and its gradient against the definition in 64 bits (in 60 digits where a position is far).

A sine or cosine is off by at most 4 u (u = 2^-24): 2^-23 from its series and the rounding of its argument, the rest from the angle, so that a result is off by 6 u (|a| + |b|) and its rounding."""
from decimal import Decimal, getcontext

import pytest
import torch

from neural_block_textures_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def angles(positions, sections, base, one_ladder):
    P, out, p = sum(sections), [], 0
    for a, n in enumerate(sections):
        for j in range(n):
            out.append(positions[..., a].double() * base ** (-p / P if one_ladder else -j / n))
            p += 1
    return torch.stack(out, -1)


def turned(x, angle, interleaved):
    x, P = x.detach().double(), angle.shape[-1]
    c, s = torch.cos(angle)[..., None, :], torch.sin(angle)[..., None, :]
    y, size = x.clone(), torch.zeros_like(x)
    lo, hi = (slice(0, 2 * P, 2), slice(1, 2 * P, 2)) if interleaved else (slice(0, P), slice(P, 2 * P))
    a, b = x[..., lo], x[..., hi]
    y[..., lo], y[..., hi] = a * c - b * s, a * s + b * c
    size[..., lo] = size[..., hi] = a.abs() + b.abs()
    return y, size


def check(got, x, angle, interleaved):
    want, size = turned(x, angle, interleaved)
    tol = 0.5 * torch.finfo(x.dtype).eps * want.abs() + 6 * U * size + torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    assert got.dtype == x.dtype and got.shape == x.shape and ((got.double() - want).abs() <= 1.01 * tol).all()
    rest = 2 * angle.shape[-1]
    assert torch.equal(got[..., rest:], x[..., rest:])


def randn(seed, *shape):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("N,Hq,Hk,D,sections,one_ladder,interleaved", [
    (1, 32, 8, 128, (16, 24, 24), True, False), (1, 1, 1, 2, (1,), False, True), (257, 3, 1, 64, (32,), False, False), (100, 4, 2, 80, (8, 16, 16), False, True),
    (63, 5, 5, 6, (1, 1), True, False), (40, 2, 1, 34, (3, 0, 5), False, False), (40, 2, 1, 34, (3, 0, 5), False, True), (9, 2, 2, 256, (128,), True, True), (2000, 8, 8, 32, (6, 6, 4), False, False),
    (30, 2, 2, 24, (1, 1, 1, 1, 1, 1, 1, 1), False, False), (11, 1, 3, 70, (11, 13), True, False), (5000, 2, 0, 64, (8, 8), False, True),
    (300, 4, 2, 80, (4, 2, 3), True, False), (300, 4, 2, 80, (4, 2, 3), True, True), (50, 3, 1, 128, (20, 20, 23), False, False), (50, 3, 1, 128, (20, 20, 23), False, True), (20, 2, 2, 26, (3,), False, False),
    (20, 2, 2, 18, (8,), False, False), (20, 2, 2, 18, (8,), False, True)])
def test_sizes(N, Hq, Hk, D, sections, one_ladder, interleaved, dtype):
    print("rotary", N, Hq, Hk, D, sections, dtype, flush=True)
    t = TYPES[dtype]
    pos = torch.randint(-300, 3000, (N, len(sections)), generator=torch.Generator(device="cuda").manual_seed(N), device="cuda")
    x = [randn(k, N, h, D).to(t).requires_grad_(True) for k, h in enumerate((Hq, Hk)) if h]
    kw = dict(sections=sections, one_ladder=one_ladder, interleaved=interleaved)
    out = ops.rotary(pos, *x, **kw)
    out = (out,) if len(x) == 1 else out
    angle = angles(pos, sections, 10000.0, one_ladder)
    for y, z in zip(out, x):
        check(y, z, angle, interleaved)
    dy = [randn(9 + k, *y.shape).to(t) for k, y in enumerate(out)]
    for dx, d in zip(torch.autograd.grad(out, x, dy), dy):
        check(dx, d, -angle, interleaved)
    with torch.no_grad():
        small = ops.rotary(pos.int(), *x, **kw)
    assert all(torch.equal(a, b) for a, b in zip(small if len(x) == 2 else (small,), out))


@pytest.mark.parametrize("far", [10 ** 6 + 3, 2 ** 31 - 1, -2 ** 31, 2 ** 40 + 12345])
def test_far_positions(far):
    getcontext().prec = 60
    two_pi = 2 * Decimal("3.14159265358979323846264338327950288419716939937510582097494459")
    P = 8
    x = randn(1, 1, 1, 2 * P)
    y = ops.rotary(torch.tensor([[far]], device="cuda"), x, sections=(P,), base=500.0)
    angle = []
    for j in range(P):
        turn = Decimal(far) * (Decimal(500) ** (Decimal(-j) / P)) / two_pi
        angle.append(float((turn - turn.to_integral_value()) * two_pi))
    want, size = turned(x, torch.tensor([angle], dtype=torch.float64, device="cuda"), False)
    # frequencies of at most 1 are off by 2^-57 of themselves, and by half a unit of 2^-64 of a turn
    assert ((y.double() - want).abs() <= (6 * U + abs(far) * (2.0 ** -57 + 2.0 ** -65 * 6.3)) * size + U * want.abs()).all()


@pytest.mark.parametrize("layout", ["fused", "four axes", "transposed", "every other", "odd start", "expanded", "positions apart"])
def test_layouts(layout):
    N, H, D, s = 48, 4, 64, (8, 16)
    pos = torch.randint(0, 500, (N, 2), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    whole = randn(2, N, 3 * H, D).to(torch.bfloat16)
    q, k = whole[:, :H], whole[:, H:2 * H]
    if layout == "four axes":
        pos, q, k = pos.view(4, 12, 2), q.view(4, 12, H, D), k.view(4, 12, H, D)
    elif layout == "transposed":
        q, k = whole[:, :H].contiguous().transpose(0, 1).contiguous().transpose(0, 1), k
    elif layout == "every other":
        q, k = randn(5, N, H, 2 * D).to(torch.bfloat16)[..., ::2], k
    elif layout == "odd start":
        q = torch.empty(N * H * D + 1, dtype=torch.bfloat16, device="cuda")[1:].view(N, H, D).copy_(q)
    elif layout == "expanded":
        k = k[:, :1].expand(N, H, D)
    elif layout == "positions apart":
        pos = torch.stack([pos, -pos], 0).permute(1, 2, 0)[..., 0]
    q, k = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
    a, b = ops.rotary(pos, q, k, sections=s)
    angle = angles(pos, s, 10000.0, False)
    check(a, q, angle, False)
    check(b, k, angle, False)
    dq, dk = torch.autograd.grad((a, b), (q, k), (a.detach(), b.detach()))
    check(dq, a.detach(), -angle, False)
    check(dk, b.detach(), -angle, False)
    only, = torch.autograd.grad(ops.rotary(pos, q, k, sections=s)[1], k, b.detach())       # q's gradient is not asked for
    assert torch.equal(only, dk)


def test_rows_far_apart():
    buf = torch.empty(3 * 900_000_000 + 256, dtype=torch.bfloat16, device="cuda")
    q = buf.as_strided((4, 2, 64), (900_000_000, 64, 1))
    q.copy_(randn(1, 4, 2, 64))
    pos = torch.arange(4, device="cuda")[:, None]
    assert torch.equal(ops.rotary(pos, q, sections=(32,)), ops.rotary(pos, q.clone(), sections=(32,)))


def test_values_that_are_not_finite():
    x = randn(1, 3, 2, 20)
    plain = ops.rotary(torch.arange(3, device="cuda")[:, None], x, sections=(4,))
    x[1, 0, 2], x[2, 1, 15] = float("nan"), float("inf")
    y = ops.rotary(torch.arange(3, device="cuda")[:, None], x, sections=(4,))
    assert y[1, 0, [2, 6]].isnan().all() and y[2, 1, 15] == float("inf")
    y[1, 0, [2, 6]], y[2, 1, 15] = plain[1, 0, [2, 6]], plain[2, 1, 15]
    assert torch.equal(y, plain)


def test_empty():
    for shape in ((0, 3, 8), (5, 0, 8)):
        q = torch.zeros(shape, device="cuda", requires_grad=True)
        y = ops.rotary(torch.zeros(shape[0], 1, dtype=torch.int64, device="cuda"), q, sections=(4,))
        assert y.shape == q.shape and torch.autograd.grad(y, q, torch.zeros_like(y))[0].shape == q.shape


def test_refusals():
    pos, q = torch.zeros(4, 2, dtype=torch.int64, device="cuda"), torch.zeros(4, 3, 16, device="cuda")
    for call, reason in ((lambda: ops.rotary(pos.float(), q, sections=(4, 4)), "positions is Float"), (lambda: ops.rotary(pos, q, sections=(4,)), "a number for each"),
                         (lambda: ops.rotary(pos, q, sections=(4, 5)), "9 pairs"), (lambda: ops.rotary(pos, q, sections=(0, 0)), "0 pairs"), (lambda: ops.rotary(pos, q, sections=(-1, 4)), "not -1"),
                         (lambda: ops.rotary(pos, q[:3], sections=(4, 4)), "leading axes"), (lambda: ops.rotary(pos, q, q.half(), sections=(4, 4)), "one type"),
                         (lambda: ops.rotary(pos, q.double(), sections=(4, 4)), "q is Double"), (lambda: ops.rotary(pos, q, sections=(4, 4), base=0.5), "base"),
                         (lambda: ops.rotary(pos, q[..., :15], sections=(2, 2)), "even number"), (lambda: ops.rotary(pos.cpu(), q, sections=(4, 4)), "on the GPU"),
                         (lambda: ops.rotary(pos, q, sections=(4, 4), base=float("nan")), "base")):
        with pytest.raises(ValueError, match=reason):
            call()
    y = ops.rotary(pos, q.requires_grad_(True), sections=(4, 4))
    g, = torch.autograd.grad((y * y).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()
