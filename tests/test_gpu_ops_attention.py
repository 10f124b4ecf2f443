"""attention and its gradients against the definition in 64 bits: packed sequences, caches, grouped heads, odd sizes, layouts, what is masked."""
import pytest
import torch

from tests.attention_reference import check, reference
from neural_block_textures_amd import ops

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def randn(seed, *shape):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def ends(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return at


def on_gpu(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def run(q, k, v, do, **kw):
    for t in (q, k, v):
        t.requires_grad_(True)
    o = ops.attention(q, k, v, **kw)
    return dict(zip(("o", "dq", "dk", "dv"), (o, *torch.autograd.grad(o, (q, k, v), do))))


def compare(got, want):
    for name, (values, tol) in want.items():
        if name in got:
            check(got[name].reshape(values.shape), values, tol, name)


# lengths of queries and keys, heads, width
CASES = [([1], [1], 1, 1, 8), ([5], [5], 2, 2, 32), ([33, 1, 64], [33, 1, 64], 4, 2, 64), ([200], [200], 3, 1, 96), ([129, 31], [129, 31], 4, 4, 128), ([0, 7, 0, 90, 0], [0, 7, 0, 90, 0], 2, 1, 16),
         ([1, 2, 3], [300, 64, 65], 8, 2, 72), ([70, 5], [3, 0], 2, 2, 40), ([100, 40, 1], [0, 200, 17], 6, 2, 104), ([500], [500], 5, 1, 128), ([257] * 5, [257] * 5, 2, 2, 24), ([1] * 70, [1] * 70, 2, 2, 64),
         ([3] * 150, [40] * 150, 16, 1, 32), ([1000], [77], 2, 1, 64), ([64], [1025], 4, 2, 128)]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("nq,nk,Hq,Hk,D", CASES)
def test_packed(nq, nk, Hq, Hk, D, dtype, causal):
    print("attention", len(nq), max(nq), max(nk), Hq, Hk, D, dtype, causal, flush=True)
    t, eq, ek = TYPES[dtype], ends(nq), ends(nk)
    q, do = randn(1, eq[-1], Hq, D).to(t), (0.01 * randn(2, eq[-1], Hq, D)).to(t)
    k, v = randn(3, ek[-1], Hk, D).to(t), (0.5 + randn(4, ek[-1], Hk, D)).to(t)
    got = run(q, k, v, do, causal=causal, cu_q=on_gpu(eq), cu_k=on_gpu(ek))
    compare(got, reference(q, k, v, do, list(zip(eq[:-1], eq[1:], ek[:-1], ek[1:])), causal))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("B,Lq,T,lens,Hq,Hk,D", [(3, 1, 700, [1, 0, 700], 8, 2, 128), (2, 5, 130, [130, 64], 4, 4, 64), (4, 1, 90, [3, 17, 64, 65], 3, 1, 80), (1, 130, 200, [199], 2, 1, 32),
                                                  (16, 1, 1030, list(range(0, 1024, 64)), 16, 1, 64)])
def test_cache(B, Lq, T, lens, Hq, Hk, D, dtype):
    """Rows past a sequence's length hold NaN, and are not read; they have gradients of 0."""
    t = TYPES[dtype]
    q, do = randn(1, B, Lq, Hq, D).to(t), (0.1 * randn(2, B, Lq, Hq, D)).to(t)
    k, v = randn(3, B, T, Hk, D).to(t), randn(4, B, T, Hk, D).to(t)
    for b, n in enumerate(lens):
        k[b, n:] = v[b, n:] = float("nan")
    got = run(q, k, v, do, k_lens=on_gpu(lens))
    flat = lambda x: torch.nan_to_num(x.detach()).reshape(-1, *x.shape[2:])  # noqa: E731
    spans = [(b * Lq, (b + 1) * Lq, b * T, b * T + n) for b, n in enumerate(lens)]
    compare(got, reference(flat(q), flat(k), flat(v), flat(do), spans))
    with torch.no_grad():
        assert torch.equal(ops.attention(q, k, v, k_lens=on_gpu(lens)), got["o"])


def test_mixed_forms():
    """Packed queries against keys in equal room, with lengths; batched queries against packed keys."""
    Hq, Hk, D, T = 4, 2, 64, 100
    nq, lens = [3, 50, 1], [100, 50, 7]
    eq, ek = ends(nq), ends(lens)
    q, k, v = randn(1, eq[-1], Hq, D).bfloat16(), randn(2, 3, T, Hk, D).bfloat16(), randn(3, 3, T, Hk, D).bfloat16()
    do = randn(4, *q.shape).bfloat16()
    got = run(q, k, v, do, cu_q=on_gpu(eq), k_lens=on_gpu(lens))
    compare(got, reference(q, k.flatten(0, 1), v.flatten(0, 1), do, [(eq[b], eq[b + 1], b * T, b * T + n) for b, n in enumerate(lens)]))
    q, k, v = randn(1, 3, 6, Hq, D).bfloat16(), randn(2, ek[-1] + 5, Hk, D).bfloat16(), randn(3, ek[-1] + 5, Hk, D).bfloat16()
    do = randn(4, *q.shape).bfloat16()
    got = run(q, k, v, do, cu_k=on_gpu(ek))
    compare(got, reference(q.flatten(0, 1), k, v, do.flatten(0, 1), [(6 * b, 6 * b + 6, ek[b], ek[b + 1]) for b in range(3)]))
    lens = [60, 50, 0]                                    # packed keys, each with room
    got = run(q, k, v, do, cu_k=on_gpu(ek), k_lens=on_gpu(lens))
    compare(got, reference(q.flatten(0, 1), k, v, do.flatten(0, 1), [(6 * b, 6 * b + 6, ek[b], ek[b] + n) for b, n in enumerate(lens)]))


def test_rows_behind_the_last_sequence():
    """... have outputs and gradients of 0, whatever they hold, and touch nothing."""
    e = [0, 40, 90]
    x = randn(1, 300, 2, 64).bfloat16()
    x[90:] = float("nan")
    do = randn(2, 300, 2, 64).bfloat16()
    got = run(x.clone(), x.clone(), x.clone(), do, cu_q=on_gpu(e), cu_k=on_gpu(e))
    assert all(not got[n][90:].any() for n in got)
    y = torch.nan_to_num(x)
    compare(got, reference(y, y, y, do, [(0, 40, 0, 40), (40, 90, 40, 90)]))


@pytest.mark.parametrize("count", [1, 63, 64, 65, 200, 5000])
def test_many_sequences(count):
    """The search for a tile's sequence, over any number of them and through empty ones."""
    nq = [(7 * i) % 5 for i in range(count)]
    e = ends(nq)
    q, k, v = (randn(s, e[-1], 1, 16).half() for s in (1, 2, 3))
    do = randn(4, *q.shape).half()
    got = run(q, k, v, do, cu_q=on_gpu(e), cu_k=on_gpu(e))
    alone = [run(*(t.detach()[a:b].clone() for t in (q, k, v)), do[a:b]) for a, b in list(zip(e[:-1], e[1:]))[-7:] if b > a]
    for name in got:
        if alone:
            whole = torch.cat([x[name].detach() for x in alone])
            assert (got[name][-len(whole):] - whole).abs().max() <= 2e-3 * whole.abs().max()   # (float16 rounding, and its gradients' power of two, which goes by all sequences)
    first = [(a, b, a, b) for a, b in zip(e[:-1], e[1:])][:60]
    n = first[-1][1]
    compare({m: x[:n] for m, x in got.items()}, reference(q[:n], k[:n], v[:n], do[:n], first))


@pytest.mark.parametrize("layout", ["fused", "heads first", "every other", "odd start", "shared keys", "gradient strided", "short rows"])
def test_layouts(layout):
    N, H, D = 150, 4, 64
    whole = randn(1, N, 3 * H, D).bfloat16()
    q, k, v = whole[:, :H], whole[:, H:2 * H], whole[:, 2 * H:]
    do = randn(2, N, H, D).bfloat16()
    if layout == "heads first":
        q, k, v = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v))
    elif layout == "every other":
        q = randn(3, N, H, 2 * D).bfloat16()[..., ::2]
    elif layout == "odd start":
        k = torch.empty(N * H * D + 1, dtype=torch.bfloat16, device="cuda")[1:].view(N, H, D).copy_(k)
    elif layout == "shared keys":
        k, v = k[:, :1].expand(N, H, D), v[:, :1].expand(N, H, D)
    elif layout == "gradient strided":
        do = randn(2, H, N, 2 * D).bfloat16()[..., ::2].transpose(0, 1)
    elif layout == "short rows":
        q, k, v = (randn(s, N, H * 65).bfloat16()[:, :H * 64].unflatten(1, (H, 64)) for s in (4, 5, 6))
    q, k, v = (t.detach() for t in (q, k, v))
    compare(run(q, k, v, do), reference(q, k, v, do, [(0, N, 0, N)]))
    b = [t.detach().unflatten(0, (3, 50)) for t in (q, k, v)]
    got = run(*b, do.unflatten(0, (3, 50)))
    compare(got, reference(q, k, v, do, [(50 * i, 50 * i + 50, 50 * i, 50 * i + 50) for i in range(3)]))


def test_gradients_of_some():
    q, k, v = (randn(s, 90, 2, 32).bfloat16() for s in (1, 2, 3))
    do = randn(4, 90, 2, 32).bfloat16()
    whole = run(q.clone(), k.clone(), v.clone(), do)
    for which in range(3):
        x = [t.clone().requires_grad_(i == which) for i, t in enumerate((q, k, v))]
        g, = torch.autograd.grad(ops.attention(*x), x[which], do)
        assert torch.equal(g, whole[("dq", "dk", "dv")[which]])


@pytest.mark.parametrize("scale", [1e-6, 0.03, 1.0, 30.0])
def test_scales(scale):
    """From all keys alike to one key alone."""
    q, k, v, do = (randn(s, 200, 2, 64).half() for s in (1, 2, 3, 4))
    compare(run(q, k, v, do, scale=scale), reference(q, k, v, do, [(0, 200, 0, 200)], scale=scale))


@pytest.mark.parametrize("size", [1e-6, 1.0, 1e3])
def test_sizes_of_gradients(size):
    """float16: scores' gradients far below its normal range, and large ones."""
    q, k, v = (randn(s, 700, 2, 64).half() for s in (1, 2, 3))
    do = (size * randn(4, 700, 2, 64)).half()
    compare(run(q, k, v, do), reference(q, k, v, do, [(0, 700, 0, 700)]))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_large_scores(dtype):
    """Scores of thousands: the largest is taken off before the exponential, and a row's maximum rises late and far."""
    t = TYPES[dtype]
    q, v, do = randn(1, 300, 1, 64).to(t), randn(2, 300, 1, 64).to(t), randn(3, 300, 1, 64).to(t)
    k = (randn(4, 300, 1, 64) * torch.linspace(0.1, 60, 300, device="cuda")[:, None, None]).to(t)
    compare(run(q, k, v, do, causal=False), reference(q, k, v, do, [(0, 300, 0, 300)], causal=False))


def test_not_finite():
    """What is not finite makes the queries that see it NaN, and no other sequence's."""
    e = [0, 100, 230, 300]
    q, k, v = (randn(s, 300, 2, 64).bfloat16() for s in (1, 2, 3))
    plain = ops.attention(q, k, v, cu_q=on_gpu(e), cu_k=on_gpu(e))
    for t, at in ((q, 150), (k, 150), (v, 150)):
        for bad in (float("nan"), float("inf")):
            x = t.clone()
            x[at, 0, 5] = bad
            o = ops.attention(*(x if t is z else z for z in (q, k, v)), cu_q=on_gpu(e), cu_k=on_gpu(e))
            assert torch.equal(o[:100], plain[:100]) and torch.equal(o[230:], plain[230:]) and torch.equal(o[:, 1], plain[:, 1])
            if bad != bad:
                seen = slice(150, 151) if t is q else slice(150, 230)
                assert o[seen, 0].isnan().any(-1).all()
    k[150, 0, 5] = -float("inf")                          # a score of minus infinity leaves its key out, one of plus infinity is NaN
    o = ops.attention(q, k, v, cu_q=on_gpu(e), cu_k=on_gpu(e))
    below = q[150:230, 0, 5] > 0
    kept = torch.cat([torch.arange(100, 150, device="cuda"), torch.arange(151, 230, device="cuda")])
    want = ops.attention(q[150:230], k[kept], v[kept], causal=False)
    assert o[150:230, 0][~below].isnan().any(-1).all() and o[150:230, 0][below].isfinite().all()
    assert (o[229, 0] - want[79, 0]).abs().max() < 2e-2 or not below[79]


def test_far_cache():
    """Rows past 2^32 bytes from the first, of a batch and within a sequence."""
    T, Hk, D = 5000, 2, 128
    step = 2 ** 20                                        # elements from row to row: 10 GB of keys
    buf = torch.empty(T * step, dtype=torch.bfloat16, device="cuda")
    k = buf.as_strided((1, T, Hk, D), (T * step, step, D, 1))
    v = buf[Hk * D:].as_strided((1, T, Hk, D), (T * step, step, D, 1))
    k.copy_(randn(1, 1, T, Hk, D))
    v.copy_(randn(2, 1, T, Hk, D))
    q, lens = randn(3, 1, 1, 4, D).bfloat16(), on_gpu([T - 3])
    o = ops.attention(q, k, v, k_lens=lens)
    assert torch.equal(o, ops.attention(q, k.clone(), v.clone(), k_lens=lens))
    del k, v
    shape, strides = (3, 10, Hk, D), (1_500_000_000, Hk * D, D, 1)
    k = buf.as_strided(shape, strides)
    k.copy_(randn(4, *shape))
    q = randn(5, 3, 10, 4, D).bfloat16()
    assert torch.equal(ops.attention(q, k, k), ops.attention(q, k.clone(), k.clone()))


def test_repeats():
    q, k, v, do = (randn(s, 1000, 8, 64).half() for s in (1, 2, 3, 4))
    a, b = run(q, k, v, do), run(q, k, v, do)
    assert all(torch.equal(a[n], b[n]) for n in a)


def test_gradient_along_directions():
    q, k, v, do = (randn(s, 60, 2, 32).half() for s in (1, 2, 3, 4))
    got = run(q, k, v, do)

    def f(q, k, v):
        s = torch.matmul(q.transpose(0, 1), k.transpose(0, 1).transpose(1, 2).contiguous()) * 32 ** -0.5
        s = s.masked_fill(~torch.ones(60, 60, dtype=torch.bool, device="cuda").tril(), float("-inf"))
        return float((torch.matmul(torch.softmax(s, -1), v.transpose(0, 1)).transpose(0, 1) * do.double()).sum())

    x = [t.detach().double() for t in (q, k, v)]
    for n in range(4):
        step = [randn(10 * n + i, 60, 2, 32).double() for i in range(3)]
        diff = (f(*(a + 1e-5 * b for a, b in zip(x, step))) - f(*(a - 1e-5 * b for a, b in zip(x, step)))) / 2e-5
        mine = sum(float((got[m].double() * b).sum()) for m, b in zip(("dq", "dk", "dv"), step))
        size = sum(float((got[m].double() * b).norm()) for m, b in zip(("dq", "dk", "dv"), step))
        assert abs(diff - mine) <= 6 * 2 * 2.0 ** -11 * size      # 6 deviations of independent roundings, two of half a step each


@pytest.mark.parametrize("shape", [(0, 2, 8), (3, 0, 2, 8), (0, 5, 2, 8)])
def test_empty(shape):
    q, k = torch.zeros(shape, dtype=torch.float16, device="cuda"), torch.zeros(shape, dtype=torch.float16, device="cuda")
    got = run(q, k, k.clone(), torch.zeros_like(q))
    assert all(got[n].shape == q.shape for n in got)


def test_no_sequences_no_keys():
    q, k = torch.randn(5, 2, 16, device="cuda").half(), torch.randn(7, 2, 16, device="cuda").half()
    got = run(q, k, k.clone(), torch.ones_like(q), cu_q=on_gpu([0]), cu_k=on_gpu([0]))     # every row is behind the last sequence
    assert all(not x.any() for x in got.values())
    got = run(q[:0].detach(), k.detach(), k.detach().clone(), torch.ones_like(q[:0]))     # no queries
    assert not got["dk"].any() and not got["dv"].any() and got["dk"].shape == k.shape
    got = run(q, k[:0], k[:0].clone(), torch.ones_like(q))
    assert not got["o"].any() and not got["dq"].any()


def test_wrong_lengths_stay_inside():
    """Ends and lengths that leave the tensors, or go backwards: wrong results, no access out of bounds (these are cut off before any address)."""
    q, k, v = (randn(s, 100, 2, 32).half() for s in (1, 2, 3))
    for e in ([0, 50, 5000], [0, -7, 100], [30, 60, 100], [0, 90, 20, 100], [0, 2 ** 31 - 1, 2 ** 31 - 1]):
        got = run(q, k, v, torch.ones_like(q), cu_q=on_gpu(e), cu_k=on_gpu(e))
        assert got["o"].shape == q.shape
    for lens in ([-5], [10 ** 9]):
        run(q[None].detach(), k[None].detach(), v[None].detach(), torch.ones_like(q[None]), k_lens=on_gpu(lens))
    torch.cuda.synchronize()


def test_refusals():
    q, k = torch.zeros(6, 4, 16, dtype=torch.float16, device="cuda"), torch.zeros(6, 2, 16, dtype=torch.float16, device="cuda")
    e = on_gpu([0, 6])
    for call, reason in ((lambda: ops.attention(q.float(), k, k), "q is Float"), (lambda: ops.attention(q, k.bfloat16(), k), "k must have q's type"), (lambda: ops.attention(q, k[:, :, :8], k), "one shape"),
                         (lambda: ops.attention(q[:, :3], k, k), "3 heads"), (lambda: ops.attention(q[..., :12], k[..., :12], k[..., :12]), "multiple of 8"),
                         (lambda: ops.attention(*(torch.zeros(6, 2, 136, dtype=torch.float16, device="cuda"),) * 3), "up to 128"), (lambda: ops.attention(q, k, k, scale=0.0), "scale"),
                         (lambda: ops.attention(q, k, k, scale=float("nan")), "scale"), (lambda: ops.attention(q, k, k, scale=-1.0), "scale"), (lambda: ops.attention(q, k, k, cu_q=e.long()), "cu_q must be a vector of int32"),
                         (lambda: ops.attention(q, k, k, cu_q=on_gpu([0, 3, 6])), "1 sequences, others of 2"), (lambda: ops.attention(q[None], k[None], k[None], cu_q=e), "cu_q goes with q"),
                         (lambda: ops.attention(q, k, k, k_lens=on_gpu([3, 3])), "k_lens is of 2"), (lambda: ops.attention(q, k, k, cu_q=e[:0]), "each sequence's end"), (lambda: ops.attention(q, k, k, cu_q=e.cpu()), "cu_q must be a tensor on the GPU"),
                         (lambda: ops.attention(q[0], k, k), "must be \\[rows"), (lambda: ops.attention(q, k.cpu(), k), "k must be a tensor on the GPU")):
        with pytest.raises(ValueError, match=reason):
            call()
    o = ops.attention(q.requires_grad_(True), k, k)
    g, = torch.autograd.grad((o * o).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()
