"""token_logprobs where short rows' arithmetic has its ends: large finite logits, masks of the type's lowest value beside ordinary ones, and
temperatures far from 1. A call holds rows of one kind only, so that no other row of a wave sends them down a more careful path. Definitions
and tolerances are those of test_gpu_ops_logprobs.py, of which what no longer fits a result's type is infinite."""
import pytest
import torch

from tests.test_gpu_ops_logprobs import F16_TINY, HALF, U, close, make, ops, reference

pytestmark = pytest.mark.gpu


def held(want, dtype):
    """what a result past the type's largest value is stored as"""
    return torch.where(torch.isinf(want.to(dtype)), want.to(dtype).double(), want)


def check(x, t, top, T, grad=True):
    n, V = x.shape
    gen = torch.Generator(device="cuda").manual_seed(5)
    g = [torch.randn(s, generator=gen, device="cuda") for s in ((n,), (n,), (n, top))]
    x.requires_grad_(grad)
    r = ops().token_logprobs(x, t, top=top, temperature=T)
    dx = torch.autograd.grad([r.logprob, r.entropy, r.top_logprobs], x, g)[0] if grad else None
    x.requires_grad_(False)
    w = reference(x, t, top, T, -100, g)
    base = U * (V / 64 + 64)
    close(r.logprob, held(w["logprob"], torch.float32), 4 * U * w["logprob"].abs() + base, ("logprob", T))
    close(r.entropy, w["entropy"], base * (2 + w["entropy"].abs()), ("entropy", T))
    assert torch.equal(r.top_ids, w["ids"])
    close(r.top_logprobs, held(w["top"], torch.float32), 4 * U * w["top"].abs() + base, ("top", T))
    if grad:
        tiny = F16_TINY if x.dtype == torch.float16 else 2.0 ** -133
        close(dx, held(w["dx"], x.dtype), w["dx_err"] + w["dx"].abs() * HALF[x.dtype] * 1.01 + tiny, ("dx", T))


DTYPES = [torch.float32, torch.bfloat16, torch.float16]
SHORT = [5, 33, 64, 100, 256, 300, 512, 1000]          # groups of 4 to 64 lanes, whole and ragged


def fits(value, dtype):
    return abs(value) <= torch.finfo(dtype).max


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", SHORT + [2000])
def test_large_values(V, dtype):
    """Rows of one value, all but one, and neighbours of it: log V where all are equal, whatever their size."""
    print("logprobs large", V, dtype, flush=True)
    n = 70
    t = torch.arange(n, device="cuda") % V
    for size in (5e4, 1e7, 1e8, 1e9, 1e10, 1e15, 1e25, 1e35):
        for value in (size, -size):
            if not fits(value, dtype):
                continue
            same = torch.full((n, V), value, device="cuda").to(dtype)
            one = same.clone()
            one[:, V // 2] = 0
            close = same.clone()
            close[:, ::3] = torch.nextafter(close[:, ::3].float(), torch.zeros((), device="cuda")).to(dtype)
            for T in (0.1, 1.0, 1.3):
                for x in (same, one, close):
                    check(x.clone(), t, min(4, V), T=T)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", SHORT + [2000])
def test_masks_of_the_lowest_value_alone(V, dtype):
    """A third and all but three symbols masked by finite values; no infinity or NaN anywhere."""
    print("logprobs lowest", V, dtype, flush=True)
    for low in (torch.finfo(dtype).min, -1e9, -1e30, -3e38):
        if not fits(low, dtype):
            continue
        some, t = make(70, V, dtype, seed=V)
        some[:, ::3] = low
        few = torch.full_like(some, low)
        few[:, [0, V // 2, V - 1]] = torch.tensor([0.5, 2.0, 1.0], device="cuda", dtype=dtype)
        for T in (0.25, 1.0, 2.0):
            for x in (some, few):
                check(x.clone(), t, min(5, V), T=T)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", SHORT + [2000, 9001])
def test_temperatures(V, dtype):
    """From nearly one symbol to nearly all alike; what is past a row's end counts nowhere."""
    print("logprobs temperatures", V, dtype, flush=True)
    x, t = make(70, V, dtype, seed=V + 1)
    wide = (x.float() * (1e37 if fits(1e38, dtype) else 1e4)).to(dtype)
    wide = torch.where(torch.isfinite(wide), wide, torch.zeros_like(wide))
    for T in (1e-30, 1e-10, 1e-3, 1e3, 1e10, 1e25):
        check(x.clone(), t, min(4, V), T=T)
    for T in (1e30, 1e34, 1e36, 2.0 ** 120):
        check(x.clone(), t, min(4, V), T=T, grad=False)
        check(wide.clone(), t, min(4, V), T=T, grad=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [33, 256, 2000])
def test_both_ends_of_the_type(V, dtype):
    """A log probability past the type's largest difference is finite where the temperature makes it so."""
    print("logprobs both ends", V, dtype, flush=True)
    big = torch.finfo(dtype).max
    x = torch.full((70, V), -big, dtype=dtype, device="cuda")
    x[:, V // 3] = big
    x[1::2, 0] = 0
    t = torch.arange(70, device="cuda") % V
    for T in (1.0, 10.0, 1e20):
        check(x.clone(), t, min(3, V), T=T)
    for T in (1e36, 2.0 ** 120):
        check(x.clone(), t, min(3, V), T=T, grad=False)


def test_temperatures_out_of_range():
    x, t = make(4, 33, torch.float32)
    for T in (2.0 ** -128, 2.0 ** 121, 1e38):
        with pytest.raises(ValueError, match="temperature must be from"):
            ops().token_logprobs(x, t, temperature=T)
