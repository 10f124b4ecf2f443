"""token_logprobs and its gradient against the definitions in 64 bits: sizes from one symbol to rows split over the chip, odd ones,
types, strides, ties, masked and empty rows, lowest values, infinities, NaN, ignored and impossible tokens.

Tolerances, with u = 2^-24 (a 32-bit rounding): (x - m) k and its factors are four roundings of it, so a log probability lp is off by
at most 4 u |lp| and the logarithm of the sum by the sum's relative error; a lane adds at most V / 64 terms in order, each from an
exponential of 2 u and an argument off by 3 u |d| (|d| e^d < 1), and joining lanes, waves and blocks adds below 50 roundings: (V / 64 + 64) u.
The entropy's second sum has terms of up to |d| e^d and is off by the same times its size. A gradient p a is off by p's relative error, (4 |lp| + V / 64 + 64) u,
times its terms, and by its own type's rounding."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F16_TINY = 2.0 ** -25


def ops():
    from neural_block_textures_amd import ops as o
    return o


def reference(x, tokens, top, T, ignore, g=None):
    """the definitions in 64 bits, for [N, V] and [N], with rows that are empty or hold NaN or +inf as documented"""
    x, T = x.double(), float(torch.tensor(T, dtype=torch.float32))
    V = x.shape[1]
    y = x / T
    empty = (x == -math.inf).all(1)
    bad = torch.isnan(x).any(1) | (x == math.inf).any(1)
    logp = torch.log_softmax(torch.where(empty[:, None], 0.0, y), 1)
    p = torch.exp(logp)
    fin = torch.where(p > 0, logp, 0.0)
    H = -(p * fin).sum(1)
    p, fin, logp = (torch.where(empty[:, None], v, t) for v, t in ((0.0, p), (0.0, fin), (-math.inf, logp)))
    H = torch.where(empty, 0.0, H)
    logp, H = torch.where(bad[:, None], math.nan, logp), torch.where(bad, math.nan, H)
    ignored = tokens == ignore
    inside = (tokens >= 0) & (tokens < V)
    at = torch.where(inside, tokens, 0).long()[:, None]
    lp = torch.where(ignored, 0.0, torch.where(inside, logp.gather(1, at)[:, 0], math.nan))
    order = torch.sort(torch.where(torch.isnan(x), -math.inf, x), dim=1, descending=True, stable=True).indices[:, :top]
    out = {"logprob": lp, "entropy": H, "ids": order, "top": logp.gather(1, order)}
    if g is not None:
        glp, gh, gt = (t.double() for t in g)
        glp = torch.where(ignored, 0.0, glp)
        glp = torch.where(~ignored & ~inside, math.nan, glp)
        hot = torch.zeros_like(x).scatter_add_(1, at, torch.where(inside, glp, 0.0)[:, None]).scatter_add_(1, order, gt)
        total = glp + gt.sum(1)
        dx = (hot - p * (total[:, None] + gh[:, None] * (fin + H[:, None]))) / T
        dx = torch.where(bad[:, None], math.nan, dx)
        out["dx"] = torch.where(empty[:, None], 0.0, dx)
        size = p * (total.abs()[:, None] + gh.abs()[:, None] * (fin.abs() + H.abs()[:, None])) / T
        out["dx_err"] = size * U * (8 * fin.abs() + V / 64 + 128) + hot.abs() / T * 8 * U
    return out


def close(got, want, err, what):
    got = got.double()
    same = (torch.isnan(got) & torch.isnan(want)) | (got == want)
    fine = torch.isfinite(want) & torch.isfinite(got) & ((got - want).abs() <= err)
    bad = ~(same | fine)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:4].tolist(), want[bad][:4].tolist())


def check(x, tokens, top, T=1.0, ignore=-100, grad=True):
    o = ops()
    V, flat, flat_tokens = x.shape[-1], x.reshape(-1, x.shape[-1]), tokens.reshape(-1)
    gen = torch.Generator(device="cuda").manual_seed(5)
    rnd = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    g = (rnd(*tokens.shape), rnd(*tokens.shape), rnd(*tokens.shape, top))
    x.requires_grad_(grad)
    r = o.token_logprobs(x, tokens, top=top, temperature=T, ignore_index=ignore)
    if grad:
        outs = [r.logprob, r.entropy] + ([r.top_logprobs] if top else [])
        dx = torch.autograd.grad(outs, x, list(g[:len(outs)]))[0]
        assert dx.shape == x.shape and dx.dtype == x.dtype
    x.requires_grad_(False)
    w = reference(flat, flat_tokens, top, T, ignore, (g[0].reshape(-1), g[1].reshape(-1), g[2].reshape(len(flat), top)))
    assert r.logprob.shape == tokens.shape and r.entropy.shape == tokens.shape
    base = U * (V / 64 + 64)
    close(r.logprob.reshape(-1), w["logprob"], 4 * U * w["logprob"].abs() + base, "logprob")
    close(r.entropy.reshape(-1), w["entropy"], base * (2 + w["entropy"].abs()), "entropy")
    if top:
        assert r.top_ids.shape == (*tokens.shape, top)
        assert torch.equal(r.top_ids.reshape(-1, top), w["ids"])
        close(r.top_logprobs.reshape(-1, top), w["top"], 4 * U * w["top"].abs() + base, "top")
    if grad:
        tiny = F16_TINY if x.dtype == torch.float16 else 2.0 ** -133
        close(dx.reshape(-1, V), w["dx"], w["dx_err"] + w["dx"].abs() * HALF[x.dtype] * 1.01 + tiny, "dx")
    return r


def make(N, V, dtype, seed=1, scale=3.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn((N, V), generator=gen, device="cuda") * scale).to(dtype)
    return x, torch.randint(0, V, (N,), generator=gen, device="cuda")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,V,top", [(1, 1, 1), (3, 2, 2), (5, 31, 4), (9, 64, 32), (66, 100, 3), (7, 255, 8), (130, 256, 4), (33, 257, 0), (4, 1000, 16),
                                     (5, 1024, 5), (3, 1025, 32), (2, 4099, 7), (1, 8193, 8), (300, 33, 1), (1, 70001, 32), (2, 131075, 16)])
def test_sizes(N, V, top, dtype):
    print("logprobs", N, V, top, dtype, flush=True)
    check(*make(N, V, dtype), top, T=0.7 if V % 2 else 1.3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [16, 17, 47, 64, 65, 128, 129, 200, 257, 512, 513, 1024])
def test_short_rows_with_many_alternatives(V, dtype):
    """Groups of every size, more rows than a block takes and not a multiple of it, alternatives that one lane holds most of."""
    print("logprobs short", V, dtype, flush=True)
    x, t = make(149, V, dtype, seed=V)
    x[1] = torch.arange(V, device="cuda").to(dtype)             # the best are all at the end, neighbours
    x[2] = -torch.arange(V, device="cuda").to(dtype)
    x[3, : min(V, 16)] += 50
    x[4, V // 2:] = -math.inf
    x[5, ::5] = math.nan
    for top in (0, 1, 5, min(32, V)):
        check(x, t, top, T=0.9)


@pytest.mark.parametrize("N,V", [(1100, 2048), (1030, 5000), (520, 20001), (300, 40000), (40, 100000), (9, 200003)])
def test_more_rows(N, V):
    print("logprobs rows", N, V, flush=True)
    check(*make(N, V, torch.bfloat16, seed=N), 6)


@pytest.mark.parametrize("V", [48, 256, 700, 3001, 50001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ties_go_to_the_lowest_index(V, dtype):
    print("logprobs ties", V, dtype, flush=True)
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randint(-2, 3, (6, V), generator=gen, device="cuda").to(dtype)
    x[1] = 0
    x[2] = -0.0
    x[2, ::3] = 0.0                                               # equal as numbers
    x[3] = torch.linspace(-8, 8, V, device="cuda").to(dtype)      # ascending: every value a new best
    x[4] = torch.linspace(8, -8, V, device="cuda").to(dtype)
    check(x, torch.arange(6, device="cuda"), 32)


@pytest.mark.parametrize("V", [40, 256, 2000, 9001, 140001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_masks_and_values_at_the_ends(V, dtype):
    print("logprobs masks", V, dtype, flush=True)
    x, t = make(12, V, dtype, seed=7)
    low = torch.finfo(dtype).min
    x[0] = -math.inf                                  # nothing left
    x[1] = -math.inf
    x[1, V - 1] = 1.0                                 # one symbol left, fewer than the alternatives asked for
    x[2, ::2] = -math.inf
    x[3] = low                                        # masks of the lowest value: all, and all but three
    x[4] = low
    x[4, [1, V // 2, V - 2]] = torch.tensor([0.5, 2.0, 1.0], device="cuda", dtype=dtype)
    x[5, V // 3] = math.nan
    x[6, V // 2] = math.inf
    x[7] = torch.finfo(dtype).max
    x[8, : V - 5] = -math.inf
    x[9] = -math.inf
    x[9, 3] = math.nan
    t[1], t[2], t[8] = 0, 0, 1                        # given tokens that the mask excludes
    t[10], t[11] = -100, V                            # ignored; impossible
    # a row of the largest value has sums of V equal terms and y far outside exp's range; temperature 1 keeps y finite in the reference
    check(x, t, 8)
    check(x, t.to(torch.int32), 0)


def test_ignored_and_impossible_tokens():
    x, t = make(5, 300, torch.float32)
    t[:] = torch.tensor([-1, 7, -100, 300, -2 ** 31], device="cuda")
    r = check(x, t, 2, ignore=7)
    assert r.logprob[1] == 0 and torch.isnan(r.logprob[[0, 2, 3, 4]]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [37, 256, 1000, 5003])
def test_strides(V, dtype):
    print("logprobs strides", V, dtype, flush=True)
    gen = torch.Generator(device="cuda").manual_seed(2)
    whole = torch.randn((3, 5, V + 9), generator=gen, device="cuda").to(dtype)
    tokens = torch.randint(0, V, (3, 6), generator=gen, device="cuda")
    check(whole[:, :-1, 4:V + 4], tokens[:, 1:5], 3)                  # rows cut out, shifted against their tokens
    check(whole.transpose(0, 1)[..., 1:V + 1], tokens.t()[:5], 3)      # rows in another order
    check(whole[0, 0, 3:V + 3], tokens[0, 0], 3)                       # a single row
    check(whole[:, :1, :V].expand(3, 4, V), tokens[:, :4], 2)          # one row read by several tokens
    check(whole.view(3, 5, 1, V + 9)[..., :V], tokens[:, :5, None], 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,V", [(2049, 3001), (4100, 9001), (500, 9001), (1300, 6000)])
def test_rows_in_order_and_in_ties(N, V, dtype):
    """Rows whose best come last, first, all at once or from few values, for one wave a row, four, and blocks a row."""
    print("logprobs order", N, V, dtype, flush=True)
    x, t = make(N, V, dtype, seed=V)
    up = torch.linspace(-8, 8, V, device="cuda")
    x[:64] = up.to(dtype)
    x[64:128] = -up.to(dtype)
    x[128:192] = (up * 64).round().remainder(7).to(dtype)
    x[192:256] = 100 + x[192:256] / 64                                # (a 16-bit type has few values there)
    x[256:300, : V // 2] = -math.inf
    x[300:310, 40:] = -math.inf
    x[310:320, 7:] = -math.inf                                        # fewer values than alternatives
    x[320:330, -3:] = 50
    for top in (1, 8, 32):
        check(x, t, top, grad=False)


def test_more_rows_than_threads_of_a_grid():
    print("logprobs 2^26 rows", flush=True)
    N, V = 2 ** 26 + 77, 2
    x = torch.zeros((N, V), dtype=torch.float16, device="cuda")
    t = torch.zeros(N, dtype=torch.int32, device="cuda")
    few = torch.cat([torch.arange(50), torch.arange(N - 120, N)]).cuda()
    src, few_t = make(len(few), V, torch.float16, seed=4)
    x[few], t[few] = src, few_t.int()
    x.requires_grad_(True)
    r = ops().token_logprobs(x, t)
    r.logprob.backward(torch.ones(N, device="cuda"))
    one = torch.ones(len(few), device="cuda")
    w = reference(src, few_t, 0, 1.0, -100, (one, 0 * one, torch.zeros((len(few), 0), device="cuda")))
    close(r.logprob[few], w["logprob"], 4 * U * w["logprob"].abs() + 65 * U, "logprob")
    close(x.grad[few], w["dx"], w["dx_err"] + w["dx"].abs() * HALF[torch.float16] * 1.01 + F16_TINY, "dx")
    assert bool((r.logprob[50:-120] == r.logprob[50]).all()) and bool((x.grad[50:-120, 0] == 0.5).all())


def test_rows_past_32_bit_offsets():
    print("logprobs far rows", flush=True)
    V, step = 1001, 2 ** 30 + 12345
    whole = torch.empty(2 * step + 2 * V, dtype=torch.bfloat16, device="cuda")
    x = whole.as_strided((3, V), (step, 1))
    src, t = make(3, V, torch.bfloat16, seed=9)
    x.copy_(src)
    r = ops().token_logprobs(x, t, top=4)
    s = ops().token_logprobs(src, t, top=4)
    assert all(torch.equal(a, b) for a, b in zip(r, s))


def test_gradient_against_differences():
    gen = torch.Generator(device="cuda").manual_seed(4)
    x, t = make(4, 300, torch.float32, scale=1.5)
    w = [torch.randn(s, generator=gen, device="cuda") for s in ((4,), (4,), (4, 3))]
    ids = ops().token_logprobs(x, t, top=3).top_ids

    def f(z):                                          # the weighted sum of outputs in 64 bits, alternatives held
        lp = torch.log_softmax(z / 0.8, 1)
        H = -(lp.exp() * lp).sum(1)
        return (w[0].double() * lp.gather(1, t[:, None])[:, 0]).sum() + (w[1].double() * H).sum() + (w[2].double() * lp.gather(1, ids)).sum()

    x.requires_grad_(True)
    r = ops().token_logprobs(x, t, top=3, temperature=0.8)
    dx = torch.autograd.grad([r.logprob, r.entropy, r.top_logprobs], x, w)[0].double()
    T = float(torch.tensor(0.8, dtype=torch.float32)) / 0.8
    for _ in range(8):
        v = torch.randn((4, 300), generator=gen, device="cuda", dtype=torch.float64)
        h = 1e-5                                       # the cubic term is below 1e-9 of the sum, the rounding of f below 1e-10
        d = (f(x.double() + h * v) - f(x.double() - h * v)) / (2 * h)
        size = (dx * v).abs().sum()
        assert abs((dx * v).sum() - d) <= size * (64 * U + abs(T - 1) * 4) + 1e-8


def test_partial_gradients_and_broadcast_ones():
    """Only some outputs used; gradients expanded from one number, as a sum gives them."""
    x, t = make(6, 500, torch.bfloat16)
    x.requires_grad_(True)
    r = ops().token_logprobs(x, t, top=2)
    (r.logprob.sum() + 0.5 * r.top_logprobs.sum()).backward()
    one = torch.ones(6, device="cuda")
    w = reference(x.detach(), t, 2, 1.0, -100, (one, 0 * one, torch.full((6, 2), 0.5, device="cuda")))
    close(x.grad, w["dx"], w["dx_err"] + w["dx"].abs() * HALF[torch.bfloat16] * 1.01, "dx")
    y = x.detach().clone().requires_grad_(True)
    ops().token_logprobs(y, t).entropy.mean().backward()
    w = reference(x.detach(), t, 0, 1.0, -100, (0 * one, one / 6, torch.zeros((6, 0), device="cuda")))
    close(y.grad, w["dx"], w["dx_err"] + w["dx"].abs() * HALF[torch.bfloat16] * 1.01, "dx")


def test_no_rows_and_other_streams():
    o = ops()
    r = o.token_logprobs(torch.empty((0, 50), device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda"), top=3)
    assert r.logprob.shape == (0,) and r.top_ids.shape == (0, 3)
    x, t = make(3, 90000, torch.bfloat16)
    want = o.token_logprobs(x, t, top=5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [o.token_logprobs(x, t, top=5) for _ in range(3)]
    side.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


@pytest.mark.parametrize("N,V", [(1, 131072), (3, 70000), (64, 300)])
def test_repeats_bit_for_bit(N, V):
    x, t = make(N, V, torch.bfloat16, seed=11)
    a = ops().token_logprobs(x, t, top=16)
    for _ in range(5):
        b = ops().token_logprobs(x, t, top=16)
        assert all(torch.equal(p, q) for p, q in zip(a, b))
