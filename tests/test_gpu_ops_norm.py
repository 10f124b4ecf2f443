"""layer_norm and its gradients against the definition in 64 bits.

Tolerances, with u = 2^-24: a 32-bit sum over a row adds at most 32 values of a lane, 6 steps of a wave and 16 waves, so that it is off by at most 54 u of the sum of
magnitudes; with X = (max|x| + |mean|) s a row's h is off by 55 u X from the mean and 32 u |h| from s, 100 u X together. y is then off by 100 u X |w| + 3 u (|y| + |b|) and its rounding. dx = s (t - a - h c):
a is off by 56 u mean|t|, c by 56 u mean|t h| + 100 u X mean|t|, h by 100 u X. The sums over rows add at most 150 terms in a row at these sizes (up to 2^17 rows)."""
import pytest
import torch

from neural_block_textures_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def half_step(t):
    return 0.5 * torch.finfo(t).eps


def made(N, C, dtype, wtype, seed=0, shift=0.3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    x = (r(N, C) + shift * r(N, 1)).to(dtype)
    return x, (1 + 0.3 * r(C)).to(wtype), (0.2 * r(C)).to(wtype), (0.1 * r(N, C)).to(dtype)


def check(x, w, b, dy, y, dx, dw, db, eps=1e-5):
    C = x.shape[-1]
    X, W, B, G = (t.detach().double() if t is not None else None for t in (x, w, b, dy))
    W = torch.ones(C, dtype=torch.float64, device="cuda") if W is None else W
    B = torch.zeros(C, dtype=torch.float64, device="cuda") if B is None else B
    var, mean = torch.var_mean(X, 1, correction=0, keepdim=True)
    s = (var + eps) ** -0.5
    h = (X - mean) * s
    big = (X.abs().amax(1, keepdim=True) + mean.abs()) * s
    tiny = torch.finfo(x.dtype).smallest_normal * half_step(x.dtype) * 2
    want = h * W + B
    tol = half_step(x.dtype) * want.abs() + 100 * U * big * W.abs() + 3 * U * (want.abs() + B.abs()) + tiny
    assert y.dtype == x.dtype and ((y.double() - want).abs() <= tol * 1.01).all()
    if dy is None:
        return
    t = G * W
    a, c = t.mean(1, keepdim=True), (t * h).mean(1, keepdim=True)
    want = s * (t - a - h * c)
    at, ah = t.abs().mean(1, keepdim=True), (t * h).abs().mean(1, keepdim=True)
    tol = half_step(x.dtype) * want.abs() + s * U * (4 * t.abs() + 60 * at + h.abs() * (60 * ah + 100 * big * at) + c.abs() * 104 * big + 36 * want.abs() / s) + tiny
    assert dx.dtype == x.dtype and ((dx.double() - want).abs() <= tol * 1.01).all()
    for got, v, e in ((dw, G * h, (G.abs() * big).sum(0) * 100 * U), (db, G, 0)):
        if got is None:
            continue
        want = v.sum(0)
        tol = half_step(got.dtype) * want.abs() + 150 * U * v.abs().sum(0) + e + torch.finfo(got.dtype).smallest_normal
        assert ((got.double() - want).abs() <= tol * 1.01).all()


@pytest.mark.parametrize("dtype,wtype", [("bf16", "bf16"), ("fp16", "fp32"), ("fp32", "fp32")])
@pytest.mark.parametrize("N,C", [(1, 1), (1, 256), (3, 7), (65, 64), (33, 65), (1000, 128), (77, 129), (300, 256), (129, 513), (70, 1024), (50, 1601), (9, 2048), (31, 2049), (17, 4099), (40, 8192),
                                 (5, 8193), (3, 20000), (7, 32768), (5, 33000)])
def test_sizes(N, C, dtype, wtype):
    print("norm", N, C, dtype, flush=True)
    x, w, b, dy = made(N, C, TYPES[dtype], TYPES[wtype], N + C)
    for t in (x, w, b):
        t.requires_grad_(True)
    y = ops.layer_norm(x, w, b)
    check(x, w, b, dy, y, *torch.autograd.grad(y, (x, w, b), dy))
    with torch.no_grad():
        assert torch.equal(ops.layer_norm(x, w, b), y)


def test_many_rows():
    x, w, b, dy = made(100003, 48, torch.bfloat16, torch.bfloat16)
    for t in (x, w, b):
        t.requires_grad_(True)
    y = ops.layer_norm(x, w, b)
    grads = torch.autograd.grad(y, (x, w, b), dy)
    check(x, w, b, dy, y, *grads)
    again = torch.autograd.grad(ops.layer_norm(x, w, b), (x, w, b), dy)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))      # the same order of sums


@pytest.mark.parametrize("which", ["none", "weight", "bias"])
def test_without_weight_or_bias(which):
    x, w, b, dy = made(37, 300, torch.float16, torch.float16)
    x.requires_grad_(True)
    w, b = (w if which == "weight" else None), (b if which == "bias" else None)
    for t in (w, b):
        if t is not None:
            t.requires_grad_(True)
    y = ops.layer_norm(x, w, b)
    asked = [t for t in (x, w, b) if t is not None]
    grads = dict(zip(map(id, asked), torch.autograd.grad(y, asked, dy)))
    check(x, w, b, dy, y, *(grads.get(id(t)) if t is not None else None for t in (x, w, b)))


def test_frozen_parts():
    x, w, b, dy = made(37, 300, torch.bfloat16, torch.bfloat16)
    w.requires_grad_(True)
    y = ops.layer_norm(x, w, b)                                       # a frozen input: the weight's gradient alone
    dw, = torch.autograd.grad(y, w, dy)
    x2 = x.clone().requires_grad_(True)
    dx, dw2 = torch.autograd.grad(ops.layer_norm(x2, w, b), (x2, w), dy)
    assert torch.equal(dw, dw2)
    dx2, = torch.autograd.grad(ops.layer_norm(x2, w.detach(), b), x2, dy)
    assert torch.equal(dx, dx2)


@pytest.mark.parametrize("layout", ["odd start", "wide rows", "transposed", "three axes", "shifted", "expanded", "every other"])
def test_layouts(layout):
    g = torch.Generator(device="cuda").manual_seed(5)
    whole = torch.randn(20, 12, 41, generator=g, device="cuda").to(torch.bfloat16)
    flat = whole.flatten()
    x = {"odd start": flat[1:1 + 12 * 40].view(12, 40), "wide rows": flat.view(120, 82)[:, 3:60], "transposed": whole[0].t(), "three axes": whole, "shifted": whole[:, :-1],
         "expanded": whole[0, :1].expand(9, 41), "every other": whole[..., ::2]}[layout]
    w = torch.rand(x.shape[-1], generator=g, device="cuda").to(torch.bfloat16)
    dy = torch.randn(x.shape, generator=g, device="cuda").to(torch.bfloat16)
    x = x.detach().requires_grad_(True)
    y = ops.layer_norm(x, w)
    dx, = torch.autograd.grad(y, x, dy)
    assert y.shape == x.shape == dx.shape
    C = x.shape[-1]
    check(x.reshape(-1, C), w, None, dy.reshape(-1, C), y.reshape(-1, C), dx.reshape(-1, C), None, None)
    strided = torch.empty(*dy.shape[:-1], 2 * C, dtype=dy.dtype, device="cuda")[..., ::2]
    strided.copy_(dy)                                                 # a gradient that does not lie whole
    dx2, = torch.autograd.grad(ops.layer_norm(x, w), x, strided)
    assert torch.equal(dx, dx2)


def test_rows_far_apart():
    """Rows past 2^31 elements from the first."""
    rows, stride = 5, 600_000_000
    buf = torch.empty((rows - 1) * stride + 256, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((rows, 256), (stride, 1))
    x.copy_(torch.randn(rows, 256, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda"))
    x.requires_grad_(True)
    y = ops.layer_norm(x)
    dy = torch.ones_like(y) * torch.arange(256, device="cuda").to(torch.bfloat16)
    dx, = torch.autograd.grad(y, x, dy)
    near = x.detach().clone().requires_grad_(True)
    y2 = ops.layer_norm(near)
    assert torch.equal(y, y2) and torch.equal(dx, torch.autograd.grad(y2, near, dy)[0])


@pytest.mark.parametrize("C", [40, 300, 3000])
def test_values_that_are_not_finite(C):
    x, w, b, dy = made(6, C, torch.float32, torch.float32)
    plain = ops.layer_norm(x, w, b)
    x[1, 3], x[2, 0], x[4, C - 1] = float("nan"), float("inf"), -float("inf")
    y = ops.layer_norm(x, w, b)
    assert y[[1, 2, 4]].isnan().all()
    assert torch.equal(y[[0, 3, 5]], plain[[0, 3, 5]])
    x.requires_grad_(True)
    dx, = torch.autograd.grad(ops.layer_norm(x, w, b), x, dy)
    assert dx[[1, 2, 4]].isnan().all() and dx[[0, 3, 5]].isfinite().all()


def test_constant_rows():
    x = torch.full((3, 100), 7.0, device="cuda", requires_grad=True)
    y = ops.layer_norm(x, None, torch.ones(100, device="cuda"))
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.equal(y, torch.ones_like(y)) and torch.equal(dx, torch.zeros_like(dx))


def test_means_far_above_the_spread():
    """A variance as mean of squares less square of the mean would lose all of it."""
    g = torch.Generator(device="cuda").manual_seed(2)
    x = 1000 + torch.randn(50, 700, generator=g, device="cuda")
    check(x, None, None, None, ops.layer_norm(x), None, None, None)


@pytest.mark.parametrize("shape", [(0, 5), (3, 0, 5)])
def test_empty(shape):
    x = torch.zeros(shape, device="cuda", requires_grad=True)
    w = torch.ones(5, device="cuda", requires_grad=True)
    y = ops.layer_norm(x, w, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert y.shape == dx.shape == x.shape and torch.equal(dw, torch.zeros(5, device="cuda"))


def test_gradient_along_directions():
    g = torch.Generator(device="cuda").manual_seed(4)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    x, w, b, dy = r(20, 90), r(90), r(90), r(20, 90)
    for t in (x, w, b):
        t.requires_grad_(True)
    grads = torch.autograd.grad(ops.layer_norm(x, w, b), (x, w, b), dy)
    f = lambda *a: float((torch.nn.functional.layer_norm(a[0].double(), (90,), a[1].double(), a[2].double()) * dy.double()).sum())  # noqa: E731
    for _ in range(4):
        step = [r(*t.shape).double() for t in (x, w, b)]
        e = 1e-4
        diff = (f(*(t.detach().double() + e * d for t, d in zip((x, w, b), step))) - f(*(t.detach().double() - e * d for t, d in zip((x, w, b), step)))) / (2 * e)
        mine = sum(float((p.double() * d).sum()) for p, d in zip(grads, step))
        size = sum(float((p.double().abs() * d.abs()).sum()) for p, d in zip(grads, step))
        assert abs(diff - mine) <= 1e-5 * size      # differences: third derivatives times e^2, below 1e-7 here; the kernel's 32 bits: 200 u


def test_refusals():
    x = torch.zeros(4, 8, device="cuda")
    for call, reason in ((lambda: ops.layer_norm(x.double()), "x is Double"), (lambda: ops.layer_norm(x, torch.ones(7, device="cuda")), "must hold x's 8"),
                         (lambda: ops.layer_norm(x, torch.ones(8, device="cuda").half()), "weight is Half"), (lambda: ops.layer_norm(x.half(), torch.ones(8, device="cuda").half(), torch.ones(8, device="cuda")), "one type"),
                         (lambda: ops.layer_norm(x, torch.ones(8)), "weight must be a tensor on the GPU"), (lambda: ops.layer_norm(x, eps=-1.0), "eps"), (lambda: ops.layer_norm(x, eps=float("nan")), "eps"),
                         (lambda: ops.layer_norm(torch.zeros(4, 0, device="cuda")), "at least one value"), (lambda: ops.layer_norm(torch.zeros((), device="cuda")), "last axis")):
        with pytest.raises(ValueError, match=reason):
            call()
    y = ops.layer_norm(x.requires_grad_(True))
    g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()
