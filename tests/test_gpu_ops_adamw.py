"""AdamW over many tensors against the step in 64 bits, for both states; what 8-bit states stand for, how they are rounded, and
what is left alone.

Tolerances, u = 2^-24: m and v are two products and a sum, 3 u of the terms' sizes; p adds the update, which goes through a square
root, a division and three products (10 u of it), two roundings of p, and p's own type's rounding."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SIZES = [1, 0, 255, 256, 257, 1000, 4095, 4096, 4097, 20000, 3, 8192]
HYPER = dict(lr=3e-3, betas=(0.8, 0.97), eps=1e-6, weight_decay=0.1)


def ops():
    from neural_block_textures_amd import ops as o
    return o


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def tensors(sizes, dtype, seed, shift=0, scale=0.5):
    g, out = gen(seed), []
    for n in sizes:
        whole = torch.empty(n + shift, dtype=dtype, device="cuda")
        whole.copy_(torch.randn(n + shift, generator=g, device="cuda") * scale)
        out.append(whole[shift:])
    return out


def step64(p, g, m, v, t, lr, betas, eps, weight_decay):
    b1, b2 = betas
    g, m, v = g.double(), m.double(), v.double()
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    up = lr / (1 - b1 ** t) * m / (torch.sqrt(v / (1 - b2 ** t)) + eps)
    return p.double() * (1 - lr * weight_decay) - up, m, v, up


def near(a, b, err, what):
    bad = ~((a.double() - b).abs() <= err)
    assert not bad.any(), (what, a[bad][:4].tolist(), b[bad][:4].tolist())


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,gtype,master,shift", [(torch.float32, torch.float32, False, 0), (torch.bfloat16, torch.bfloat16, False, 0), (torch.bfloat16, torch.float32, True, 1),
                                                      (torch.float16, torch.bfloat16, True, 0), (torch.float16, torch.float16, False, 3), (torch.float32, torch.float16, False, 1)])
def test_steps_against_64_bits(dtype, gtype, master, shift, bits):
    print("adamw", dtype, gtype, master, shift, bits, flush=True)
    params = tensors(SIZES, dtype, 1, shift)
    guard = [p._base[:shift].clone() if shift else None for p in params]
    opt = ops().AdamW(params, state_bits=bits, master=master, seed=3, **HYPER)
    for t in range(1, 4):
        grads = tensors(SIZES, gtype, 10 + t, shift, 0.1)
        before = [x.clone() for x in (opt.moments()[0], opt.moments()[1])]
        p0 = [opt.master[o:o + p.numel()].clone() if master else p.clone() for p, o in zip(params, opt.offsets)]
        opt.step(grads)
        m1, v1 = opt.moments()
        for p, q, g, o in zip(params, p0, grads, opt.offsets):
            n = p.numel()
            m0, v0 = before[0][o:o + n], before[1][o:o + n]
            w, m, v, up = step64(q, g, m0, v0, t, **HYPER)
            err = up.abs() * 12 * U + 3 * U * q.abs().double()
            if master:
                near(opt.master[o:o + n], w, err, "master")
                assert torch.equal(p, opt.master[o:o + n].to(dtype))
            else:
                near(p, w, err + w.abs() * HALF[dtype] * 1.01 + 2.0 ** -25, "p")
            if bits == 32:
                near(m1[o:o + n], m, 3 * U * (m0.abs() + g.abs()).double() + 1e-45, "m")
                near(v1[o:o + n], v, 3 * U * v + 1e-45, "v")
            else:                                      # to one of the two neighbours: an eighth of a binade, or the smallest step of the block
                pad = lambda x: torch.nn.functional.pad(x.abs(), (0, -n % 256)).view(-1, 256)  # noqa: E731
                for got, want, lo in ((m1, m, -17), (v1, v, -33)):
                    top = 2.0 ** torch.ceil(torch.log2(pad(want).amax(1).clamp_min(1e-38) / 1.875) + 1e-9)
                    unit = torch.maximum(2.0 ** (torch.floor(torch.log2(want.abs().clamp_min(1e-38)) + 1e-9) - 3), top.repeat_interleave(256)[:n] * 2.0 ** lo)
                    near(got[o:o + n], want, unit * 1.0001, "8-bit state")
            end = -(-n // 256) * 256
            assert not m1[o + n:o + end].any() and not v1[o + n:o + end].any()      # between tensors it stays 0
    for p, g in zip(params, guard):
        assert g is None or torch.equal(p._base[:shift], g)


def test_more_tensors_than_a_launch_takes():
    sizes = [(k * 37) % 600 + 1 for k in range(500)]
    params, grads = tensors(sizes, torch.bfloat16, 1), tensors(sizes, torch.bfloat16, 2)
    p0 = [p.clone() for p in params]
    grads[3] = grads[200] = grads[499] = None
    opt = ops().AdamW(params, **HYPER)
    opt.step(grads)
    zero = torch.zeros(1, device="cuda")
    for k, (p, q, g) in enumerate(zip(params, p0, grads)):
        if g is None:
            assert torch.equal(p, q)
        else:
            w, _, _, up = step64(q, g, zero, zero, 1, **HYPER)
            near(p, w, up.abs() * 12 * U + w.abs() * HALF[torch.bfloat16] * 1.01, k)
    assert opt.steps[3] == 0 and opt.steps[4] == 1


def test_tensors_at_many_different_steps():
    sizes = [(k * 53) % 700 + 1 for k in range(120)]
    params = tensors(sizes, torch.float32, 1)
    opt = ops().AdamW(params, **HYPER)
    zero = torch.zeros(1, device="cuda")
    state = opt.state_dict()
    state["step"] = [3 * (k % 23) for k in range(len(sizes))]      # (more of them than a launch takes)
    opt.load_state_dict(state)
    p0, grads = [p.clone() for p in params], tensors(sizes, torch.float32, 2)
    grads[0] = grads[50] = None
    opt.step(grads)
    for k, (p, q, g) in enumerate(zip(params, p0, grads)):
        if g is None:
            assert torch.equal(p, q)
            continue
        w, _, _, up = step64(q, g, zero, zero, 3 * (k % 23) + 1, **HYPER)
        near(p, w, up.abs() * 12 * U + 3 * U * q.abs().double(), k)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_tensor_without_gradient_keeps_its_state_and_step(bits):
    params = tensors([300, 700], torch.float32, 1)
    opt = ops().AdamW(params, state_bits=bits, **HYPER)
    g = tensors([300, 700], torch.float32, 2)
    opt.step([g[0], None])
    opt.step([g[0], None])
    p1 = params[1].clone()
    m, v = (x.clone() for x in opt.moments())
    assert not m[512:].any() and not v[512:].any()
    opt.step(g)                                         # its first step: bias corrections of step 1, not 3
    w, _, _, up = step64(p1, g[1], m[512:1212], v[512:1212], 1, **HYPER)
    near(params[1], w, up.abs() * 12 * U + 3 * U * p1.abs().double(), "first step")
    assert opt.steps.tolist() == [3, 1]


def test_from_autograd_and_mixed_types():
    a = torch.randn((40, 30), device="cuda", generator=gen(1)).requires_grad_(True)
    b = torch.randn((30,), device="cuda", generator=gen(2)).to(torch.bfloat16).requires_grad_(True)
    opt = ops().AdamW([a, b], **HYPER)
    (a * b.float()).sum().backward()
    p0, g0 = [a.detach().clone(), b.detach().clone()], [a.grad.clone(), b.grad.clone()]
    opt.step()
    zero = torch.zeros(1, device="cuda")
    for p, q, g in zip((a, b), p0, g0):
        w, _, _, up = step64(q, g, zero, zero, 1, **HYPER)
        near(p.detach(), w, up.abs() * 12 * U + 3 * U * q.abs().double() + w.abs() * HALF[p.dtype] * 1.01, "p")
    opt.zero_grad()
    assert a.grad is None and b.grad is None


def test_gradients_that_are_not_contiguous():
    for make in (lambda: torch.randn((20, 30), device="cuda", generator=gen(4)).t(), lambda: torch.randn((1, 20), device="cuda", generator=gen(5)).expand(30, 20)):
        p, q = (torch.ones((30, 20), device="cuda") for _ in range(2))
        ops().AdamW([p], **HYPER).step([make()])
        ops().AdamW([q], **HYPER).step([make().contiguous()])
        assert torch.equal(p, q) and (p != 1).any()


def test_8_bit_codes_stand_for_their_values():
    """Every code at a few block exponents, against the format's definition."""
    codes = torch.arange(256, device="cuda", dtype=torch.uint8)
    opt = ops().AdamW([torch.zeros(256 * 4, device="cuda")], state_bits=8)
    for E in (0, 1, 100, 127, 200, 254, 255):
        opt.exp_avg.copy_(codes.repeat(4))
        opt.exp_avg_sq.copy_(codes.repeat(4))
        opt.exp_avg_exp.fill_(E)
        opt.exp_avg_sq_exp.fill_(E)
        m, v = (x[:256].cpu().double().numpy() for x in opt.moments())
        if E == 255:
            assert np.isnan(m).all() and np.isnan(v).all()
            continue
        for got, bits, bias in ((m, 4, 15), (v, 5, 31)):
            for c in range(256):
                n = c & 127 if bits == 4 else c
                e, f = n >> 3, n & 7
                want = ((1 + f / 8) * 2.0 ** (e - bias) if e else f / 8 * 2.0 ** (1 - bias)) * (-1 if bits == 4 and c > 127 else 1)
                want = float(np.float32(math.ldexp(want, E - 127)))       # a 32-bit subnormal where it is that small
                assert got[c] == want, (E, bits, c, got[c], want)


def test_8_bit_rounding_is_unbiased_and_never_zero():
    """Averages that one step moves by far less than a code's distance arrive where 32-bit ones do, in the mean; a value whose gradient
    is tiny beside its block's largest keeps a v above 0."""
    n = 1 << 16
    p = torch.zeros(n, device="cuda")
    opt = ops().AdamW([p], lr=0.0, betas=(0.9, 0.999), weight_decay=0.0, state_bits=8, seed=7)
    g = torch.full((n,), 0.3, device="cuda")
    g[::256] = 1.0                                       # each block's largest
    g[1::256] = 1e-9
    steps = 1500
    for _ in range(steps):
        opt.step([g])
    m, v = opt.moments()
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[::256] = keep[1::256] = False
    want = 0.09 * (1 - 0.999 ** steps)
    got = v[keep].double().mean().item()
    # one step's rounding has a standard deviation below 0.5 sqrt(0.001 / 0.0625) of a code's distance (an eighth at most), 500 steps are remembered, and
    # 65024 values are averaged: 1.5% / 16 * sqrt(500) * 8 / 255 < 0.1%; 1% is ten of those
    assert abs(got / want - 1) < 0.01, (got, want)
    assert abs(m[keep].double().mean().item() / 0.3 - 1) < 0.01
    assert (v[1::256] > 0).all()
    assert abs(v[::256].double().mean().item() / (1 - 0.999 ** steps) - 1) < 0.05


def test_8_bit_rounding_takes_the_documented_bits():
    """The codes of one step from the format and the counter noise, in integers on the host."""
    mask = (1 << 64) - 1

    def mix(x):
        x = (x + 0x9E3779B97F4A7C15) & mask
        x = ((x ^ (x >> 30)) * 0xBF58476D1CE4E5B9) & mask
        x = ((x ^ (x >> 27)) * 0x94D049BB133111EB) & mask
        return x ^ (x >> 31)

    n, seed = 600, 12345
    p = torch.zeros(n, device="cuda")
    opt = ops().AdamW([torch.zeros(100, device="cuda"), p], betas=(0.5, 0.5), state_bits=8, seed=seed)
    g = torch.randn(n, generator=gen(8), device="cuda")
    opt.step([None, g])
    g32 = g.cpu().numpy()
    m32, v32 = g32 * np.float32(0.5), (g32 * g32) * np.float32(0.5)
    head = mix(seed ^ (5 << 56) ^ (1 << 32))
    for b in range(0, n, 256):
        for x32, top, sh, codes, exps in ((m32, 15, 0, opt.exp_avg, opt.exp_avg_exp), (v32, 31, 16, opt.exp_avg_sq, opt.exp_avg_sq_exp)):
            x = x32[b:b + 256].astype(np.float64)
            most = np.abs(x).max()
            E = math.floor(math.log2(most))
            E += most > 1.875 * 2.0 ** E
            at = 256 + b
            assert int(exps[at // 256]) == E + 127
            for i in range(len(x)):
                r = (mix((head + ((at + i) >> 1) * 0x9E3779B97F4A7C15) & mask) >> (32 * ((at + i) & 1) + sh)) & 0xffff
                a = abs(x[i]) / 2.0 ** E
                e = max(math.floor(math.log2(a)) if a > 0 else -99, 1 - top)
                k = math.floor(a / 2.0 ** (e - 3) + r / 65536)
                code = (e + top) * 8 + k - 8 if a >= 2.0 ** (1 - top) else k
                if top == 31:
                    code = max(code, 1) if a > 0 else 0
                else:
                    code |= 128 if x[i] < 0 else 0
                assert int(codes[at + i]) == code, (b, i, top)


@pytest.mark.parametrize("bits", [32, 8])
def test_zeros_and_values_that_are_not_finite(bits):
    p = torch.ones(1024, device="cuda")
    opt = ops().AdamW([p], state_bits=bits, lr=0.1, weight_decay=0.0)
    g = torch.zeros(1024, device="cuda")
    opt.step([g])
    assert torch.equal(p, torch.ones_like(p)) and not opt.moments()[0].any() and not opt.moments()[1].any()
    g[300], g[600] = math.inf, math.nan
    g[10] = 1.0
    opt.step([g])
    assert torch.isnan(p[[300, 600]]).all()
    g[300] = g[600] = 0.0
    opt.step([g])
    bad = torch.isnan(p)
    assert bad[300] and bad[600] and not bad[:256].any() and not bad[768:].any()
    if bits == 8:
        assert bad[256:768].all()                        # their blocks, from the next step on
    else:
        assert int(bad.sum()) == 2


def test_state_dict_and_repeats():
    runs = []
    for k in range(2):
        params = tensors([1000, 77], torch.bfloat16, 1)
        opt = ops().AdamW(params, state_bits=8, master=True, seed=5, **HYPER)
        for t in range(4):
            if k and t == 2:                             # the second run goes on in a new optimizer
                saved = {n: x.clone() if torch.is_tensor(x) else x for n, x in opt.state_dict().items()}
                opt = ops().AdamW(params, state_bits=8, master=True, seed=5, **HYPER)
                opt.load_state_dict(saved)
            opt.step(tensors([1000, 77], torch.bfloat16, 20 + t, scale=0.1))
        runs.append([*params, opt.master, *opt.moments()])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_set_moments_rounds_to_nearest():
    opt = ops().AdamW([torch.zeros(2000, device="cuda")], state_bits=8)
    m, v = torch.zeros(opt.size, device="cuda"), torch.zeros(opt.size, device="cuda")
    m[:2000], v[:2000] = torch.randn(2000, generator=gen(1), device="cuda"), torch.rand(2000, generator=gen(2), device="cuda")
    opt.set_moments(m, v)
    a, b = opt.moments()
    near(a, m.double(), m.abs().double() / 16 * 1.0001 + m.abs().max() * 2.0 ** -18, "m")
    near(b, v.double(), v.double() / 16 * 1.0001 + 2.0 ** -33, "v")


@pytest.mark.parametrize("at", [0, 1, 2, 3])
def test_set_moments_takes_a_v_without_sign(at):
    """-0 and values below 0 count as 0, and the codes beside them (four to a word) are what they are without."""
    opt = ops().AdamW([torch.zeros(512, device="cuda")], state_bits=8)
    m, v = torch.randn(512, generator=gen(4), device="cuda"), 0.25 + torch.rand(512, generator=gen(5), device="cuda")
    clean, signed = v.clone(), v.clone()
    clean[at::4] = 0.0
    signed[at::8], signed[at + 4::8] = -0.0, -0.125
    opt.set_moments(m, clean)
    wanted = [t.clone() for t in opt.moments()]
    opt.set_moments(m, signed)
    assert all(torch.equal(a, b) for a, b in zip(opt.moments(), wanted))



def test_more_than_2_31_values():
    print("adamw large", flush=True)
    n = 2 ** 31 + 1000
    p = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g[-3:] = 1.0
    g[5] = 1.0
    opt = ops().AdamW([p], lr=0.25, weight_decay=0.0, state_bits=8)
    opt.step([g])
    assert p[-4:].tolist() == [0.0, -0.25, -0.25, -0.25] and p[5] == -0.25
    assert int((p != 0).sum()) == 4
