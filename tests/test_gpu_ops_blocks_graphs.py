"""Layer norm, rotary positions and attention in captured graphs (every replay on new values is what the eager calls give, with eager work between), on other
streams, with tangents, and one after another as a model runs them."""
import pytest
import torch
from torch.autograd import forward_ad

from neural_block_textures_amd import ops

pytestmark = pytest.mark.gpu


def fill(tensors, seed):
    with torch.no_grad():
        for i, t in enumerate(tensors):
            t.copy_(torch.randn(t.shape, generator=torch.Generator(device="cuda").manual_seed(100 * seed + i), device="cuda"))


def captured(call, pool=None):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, pool=pool):
        out = call()
    return graph, out


def replays(call, inputs, before=lambda k: None):
    graph, out = captured(call)
    for k in range(4):
        fill(inputs, k)
        before(k)
        want = [y.detach().clone() for y in call()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k


def zeros(*shape, grad=True, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype, device="cuda", requires_grad=grad)


@pytest.mark.parametrize("N,C", [(1, 512), (4096, 256), (37, 1000), (3, 40000), (9000, 2048)])
def test_layer_norm(N, C):
    x, w, b, dy = zeros(N, C), zeros(C), zeros(C), zeros(N, C, grad=False)

    def call():
        y = ops.layer_norm(x, w, b)
        return [y, *torch.autograd.grad(y, (x, w, b), dy)]

    replays(call, (x, w, b, dy))


@pytest.mark.parametrize("N,H", [(1, 8), (3000, 4)])
def test_rotary(N, H):
    q, k, dq, dk = zeros(N, H, 64), zeros(N, 1, 64), zeros(N, H, 64, grad=False), zeros(N, 1, 64, grad=False)
    at = torch.zeros(N, 3, dtype=torch.int32, device="cuda")

    def call():
        y = ops.rotary(at, q, k, sections=(10, 10, 12))
        return [*y, *torch.autograd.grad(y, (q, k), (dq, dk))]

    replays(call, (q, k, dq, dk), lambda i: at.copy_(torch.arange(3 * N, device="cuda").view(N, 3) * (i + 1)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nq,nk,Hq,Hk,D", [([300, 0, 41], [300, 0, 41], 4, 2, 64), ([1500], [1500], 2, 1, 128), ([9], [6000], 4, 1, 32), ([128] * 60, [128] * 60, 8, 8, 32)])
def test_attention(nq, nk, Hq, Hk, D, dtype):
    """... whose sequences' ends change between replays as well."""
    q, k, v, do = zeros(sum(nq), Hq, D, dtype=dtype), zeros(sum(nk), Hk, D, dtype=dtype), zeros(sum(nk), Hk, D, dtype=dtype), zeros(sum(nq), Hq, D, grad=False, dtype=dtype)
    ends = lambda n: torch.tensor([0, *n], device="cuda").cumsum(0).int()  # noqa: E731
    eq, ek = ends(nq), ends(nk)
    first_q, first_k = eq.clone(), ek.clone()

    def call():
        o = ops.attention(q, k, v, cu_q=eq, cu_k=ek)
        return [o, *torch.autograd.grad(o, (q, k, v), do)]

    def move(i):
        eq.copy_(torch.clamp(first_q - i, min=0))            # the last rows are behind the last sequence then
        ek.copy_(torch.clamp(first_k - 2 * i, min=0))

    replays(call, (q, k, v, do), move)


def test_two_graphs_of_tokens():
    """Steps for single tokens from caches that fill up: two graphs, from one pool, replayed in turn."""
    B, T, Hq, Hk, D = 3, 2000, 8, 2, 64
    q = [torch.zeros(B, 1, Hq, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    k, v = (torch.zeros(B, T, Hk, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    lens = [torch.zeros(B, dtype=torch.int32, device="cuda") for _ in range(2)]
    calls = [lambda i=i: ops.attention(q[i], k, v, k_lens=lens[i]) for i in range(2)]
    with torch.no_grad():
        one, first = captured(calls[0])
        two, second = captured(calls[1], one.pool())
        for n in range(5):
            fill((*q, k, v), n)
            for i in range(2):
                lens[i].copy_(torch.tensor([n, 100 * n + i, min(T, 600 * n + 1)], device="cuda"))
            want = [call().clone() for call in calls]
            one.replay()
            got = [first.clone()]
            two.replay()
            got.append(second.clone())
            torch.cuda.synchronize()
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), n


def block(x, w, b, at, ends, H):
    """What a layer of a model does with them: (tokens, 3 H D) -> (tokens, H, D)."""
    q, k, v = ops.layer_norm(x, w, b).view(x.shape[0], 3, H, -1).unbind(1)
    q, k = ops.rotary(at, q, k, sections=(8, 8))
    return ops.attention(q, k, v, cu_q=ends, cu_k=ends)


def block_inputs():
    N, H, D = 333, 4, 40
    ends = torch.tensor([0, 100, 101, 101, 320], dtype=torch.int32, device="cuda")
    at = torch.stack((torch.arange(N) // 16, torch.arange(N) % 16), 1).cuda()
    return zeros(N, 3 * H * D), zeros(3 * H * D), zeros(3 * H * D), at, ends, H, zeros(N, H, D, grad=False)


def test_one_after_another_in_a_graph():
    x, w, b, at, ends, H, do = block_inputs()

    def call():
        o = block(x, w, b, at, ends, H)
        return [o, *torch.autograd.grad(o, (x, w, b), do)]

    replays(call, (x, w, b, do))


def test_streams():
    """Two streams at once, each with work that the other's must not disturb; tensors made on a third."""
    x, w, b, at, ends, H, do = block_inputs()
    fill((x, w, b, do), 1)

    def call(scale):
        o = block(x * scale, w, b, at, ends, H)
        return [o.detach(), *torch.autograd.grad(o, (x, w, b), do)]

    want = [call(s) for s in (1, 2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for n in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(i + 1))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, c) for r in got[i] for a, c in zip(r, want[i]))


@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(grad):
    x, w = torch.randn(4, 64, device="cuda"), torch.randn(64, device="cuda")
    q = torch.randn(4, 2, 32, device="cuda").bfloat16()
    at = torch.zeros(4, 1, dtype=torch.int64, device="cuda")
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t.clone().requires_grad_(grad), torch.ones_like(t))  # noqa: E731
        dx, dw, dq = dual(x), dual(w), dual(q)
        for call in (lambda: ops.layer_norm(dx), lambda: ops.layer_norm(x, dw), lambda: ops.layer_norm(x, w, dw), lambda: ops.rotary(at, dq, sections=(16,)), lambda: ops.rotary(at, q, dq, sections=(16,)),
                     lambda: ops.attention(dq, q, q), lambda: ops.attention(q, dq, q), lambda: ops.attention(q, q, dq)):
            with pytest.raises(ValueError, match="no forward-mode derivative"):
                call()
        plain = ops.attention(q, q, q)
    assert torch.equal(plain, ops.attention(q, q, q))


def test_changed_in_between():
    """What a gradient needs and has been written over since is an error of torch's, not a wrong gradient."""
    q = torch.randn(6, 2, 32, device="cuda").bfloat16().requires_grad_()
    ends = torch.tensor([0, 6], dtype=torch.int32, device="cuda")
    o = ops.attention(q, q, q, cu_q=ends, cu_k=ends)
    ends[1] = 3
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()
    at = torch.zeros(6, 1, dtype=torch.int32, device="cuda")
    y = ops.rotary(at, q, sections=(16,))
    at += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    x = torch.randn(6, 32, device="cuda", requires_grad=True)
    t = x * 1
    y = ops.layer_norm(t)
    t += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_broadcast_inputs():
    """Rows, heads and keys that are one in memory: their gradients are the sums over where they are read."""
    x = torch.randn(40, device="cuda", requires_grad=True)
    dy = torch.randn(5, 7, 40, device="cuda")
    g, = torch.autograd.grad(ops.layer_norm(x.expand(5, 7, 40)), x, dy)
    h, = torch.autograd.grad(ops.layer_norm(x.expand(5, 7, 40).contiguous()), x, dy)
    assert torch.equal(g, h)
    q = torch.randn(5, 1, 32, device="cuda").bfloat16().requires_grad_()
    at = torch.arange(5, device="cuda").view(5, 1)
    for turn in (lambda y: ops.rotary(at, y, sections=(9,)), lambda y: ops.attention(y, y[:1].expand(5, 4, 32), y), lambda y: ops.rotary(at[:1].expand(5, 1), y, sections=(9,))):
        do = torch.randn(5, 4, 32, device="cuda").bfloat16()
        g, = torch.autograd.grad(turn(q.expand(5, 4, 32)), q, do)
        h, = torch.autograd.grad(turn(q.expand(5, 4, 32).contiguous()), q, do)
        assert torch.equal(g, h)


def test_sizes_of_nothing():
    at = torch.zeros(0, 1, dtype=torch.int32, device="cuda")
    q = torch.zeros(0, 3, 16, device="cuda", requires_grad=True)
    y, z = ops.rotary(at, q, q, sections=(8,))
    (y.sum() + z.sum()).backward()
    assert q.grad.shape == q.shape
    at = torch.zeros(4, 1, dtype=torch.int32, device="cuda")
    q, k = torch.randn(4, 0, 16, device="cuda"), torch.randn(4, 2, 16, device="cuda", requires_grad=True)
    y, z = ops.rotary(at, q, k, sections=(8,))
    assert y.shape == q.shape and torch.equal(z, k)
    y, z = ops.rotary(at, k, q, sections=(8,))
    y.sum().backward()
    assert torch.equal(k.grad, torch.ones_like(k))
    w = torch.randn(7, device="cuda", requires_grad=True)
    y = ops.layer_norm(torch.zeros(3, 0, 7, device="cuda", requires_grad=True), w, w)
    y.sum().backward()
    assert y.shape == (3, 0, 7) and not w.grad.any()
    x = torch.randn(5, 1, device="cuda", requires_grad=True)
    y = ops.layer_norm(x)
    y.sum().backward()
    assert not y.any() and not x.grad.any()
