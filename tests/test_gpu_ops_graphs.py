"""The operators in a captured graph: every replay on new values is what the eager calls give, with eager work between. What a replay of an optimizer's
step is, is stated with it: the step that was captured, with its step count and random bits, on what the gradients hold by then."""
import pytest
import torch

from neural_block_textures_amd import ops

pytestmark = pytest.mark.gpu


def captured(call):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    return graph, out


@pytest.mark.parametrize("N,V,top", [(300, 256, 4), (2, 90000, 8), (700, 3000, 0)])
def test_token_logprobs(N, V, top):
    print("graph logprobs", N, V, top, flush=True)
    x = torch.zeros((N, V), dtype=torch.bfloat16, device="cuda", requires_grad=True)
    t = torch.zeros(N, dtype=torch.int64, device="cuda")

    def call():
        r = ops.token_logprobs(x, t, top=top)
        g, = torch.autograd.grad([r.logprob, r.entropy], x, [torch.ones_like(r.logprob), torch.ones_like(r.entropy)])
        return [y for y in r if y is not None] + [g]

    graph, out = captured(call)
    for k in range(4):
        with torch.no_grad():
            x.copy_(torch.randn((N, V), generator=torch.Generator(device="cuda").manual_seed(k), device="cuda"))
            t.fill_(k)
        want = [y.clone() for y in call()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k


@pytest.mark.parametrize("M,N,K", [(3, 300, 500), (300, 200, 520), (4096, 64, 64)])
def test_fp8_linear(M, N, K):
    print("graph fp8", M, N, K, flush=True)
    x, w = (torch.zeros(s, dtype=torch.bfloat16, device="cuda", requires_grad=True) for s in ((M, K), (N, K)))
    dy = torch.zeros((M, N), dtype=torch.bfloat16, device="cuda")

    def call():
        y = ops.fp8_linear(x, w)
        return [y, *torch.autograd.grad(y, (x, w), dy)]

    graph, out = captured(call)
    for k in range(4):
        with torch.no_grad():
            for i, v in enumerate((x, w, dy)):
                v.copy_(torch.randn(v.shape, generator=torch.Generator(device="cuda").manual_seed(10 * k + i), device="cuda"))
        want = [y.detach().clone() for y in call()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_repeats_the_captured_step(bits):
    p, g = torch.ones(1000, device="cuda"), torch.ones(1000, device="cuda")
    opt = ops.AdamW([p], state_bits=bits, seed=3)
    graph, _ = captured(lambda: opt.step([g]))              # steps 1 and 2, and the captured one, 3
    assert opt.calls == 3 and opt.steps.tolist() == [3]
    state = {k: v.clone() if torch.is_tensor(v) else v for k, v in opt.state_dict().items()}
    start = p.clone()
    for k in range(3):
        g.copy_(torch.randn(1000, generator=torch.Generator(device="cuda").manual_seed(k), device="cuda"))
        graph.replay()
    assert opt.calls == 3                                    # replays are not counted
    q = start.clone()
    eager = ops.AdamW([q], state_bits=bits, seed=3)
    eager.load_state_dict(state)
    for k in range(3):
        eager.load_state_dict({**eager.state_dict(), "step": 2, "calls": 2})
        eager.step([torch.randn(1000, generator=torch.Generator(device="cuda").manual_seed(k), device="cuda")])
    torch.cuda.synchronize()
    assert torch.equal(p, q) and all(torch.equal(a, b) for a, b in zip(opt.moments(), eager.moments()))
