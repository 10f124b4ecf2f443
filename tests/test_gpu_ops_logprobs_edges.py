"""token_logprobs where its arithmetic has its ends: values at both ends of the type, and
temperatures far from 1. A call holds rows of one kind only, so that no other row of a wave sends them down a more careful path. Definitions
and tolerances are those of test_gpu_ops_logprobs.py, of which what no longer fits a result's type is infinite."""
import math

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
@pytest.mark.parametrize("V", [2000, 9001])
def test_temperatures_of_long_rows(V, dtype):
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
    for T in (1.0, 10.0):
        check(x.clone(), t, min(3, V), T=T)
