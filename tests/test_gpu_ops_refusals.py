"""What the operators refuse of tensors that are on the GPU."""
import pytest
import torch

from neural_block_textures_amd import ops as O

pytestmark = pytest.mark.gpu


def z(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype, device="cuda")


def test_logprobs():
    t = z(4, dtype=torch.int64)
    for logits, tokens, kw, reason in [
            (z(4, 9), z(3, dtype=torch.int64), {}, "shape of logits"), (z(4, 9, dtype=torch.float64), t, {}, "logits is"), (z(4, 9), z(4), {}, "tokens is"),
            (z(9, 4).t(), t, {}, "contiguous"), (z(4, 0), t, {}, "at least one value"), (z(4, 9), t, {"top": 10}, "top is 0 to 9"), (z(4, 40), t, {"top": 33}, "top is 0 to 32"),
            (z(4, 9), t, {"temperature": 0.0}, "temperature"), (z(4, 9), t, {"temperature": float("nan")}, "temperature"), (z(4, 9), t.cpu(), {}, "on the GPU"),
            (z(2, 2, 2, 9).transpose(0, 1), z(2, 2, 2, dtype=torch.int64), {}, "two strides")]:
        with pytest.raises(ValueError, match=reason):
            O.token_logprobs(logits, tokens, **kw)


def test_adamw():
    p = z(300)
    for params, kw, reason in [([z(4, 5).t()], {}, "contiguous"), ([p, p], {}, "overlap"), ([p[:200], p[100:]], {}, "overlap"), ([p], {"state_bits": 4}, "8 or 32"),
                               ([p], {"betas": (1.0, 0.9)}, "betas"), ([p], {"lr": -1.0}, "negative"), ([z(3, dtype=torch.float64)], {}, "a parameter is")]:
        with pytest.raises(ValueError, match=reason):
            O.AdamW(params, **kw)
    opt = O.AdamW([p, z(5)], state_bits=8)
    for grads, reason in [([p], "1 gradients for 2"), ([z(300), z(6)], "gradient 1"), ([z(300), z(5, dtype=torch.float64)], "gradient 1"), ([z(300).cpu(), None], "gradient 0")]:
        with pytest.raises(ValueError, match=reason):
            opt.step(grads)
    assert opt.calls == 0 and not opt.steps.any()                  # a refused step is none
    with pytest.raises(ValueError, match="a state has 768"):
        opt.set_moments(z(300), z(300))
    with pytest.raises(ValueError, match="exp_avg must be"):
        opt.load_state_dict({"step": 1, "exp_avg": z(3), "exp_avg_sq": z(3)})
    q = torch.nn.Parameter(z(10))
    opt = O.AdamW([q])
    q.data = z(10)
    with pytest.raises(ValueError, match="moved"):
        opt.step([z(10)])


def test_fp8():
    with pytest.raises(ValueError, match="a matrix"):
        O.fp8_quantize(z(4))
    with pytest.raises(ValueError, match="1 or 128 rows"):
        O.fp8_quantize(z(4, 4), 64)
    a, b = O.fp8_quantize(z(4, 200)), O.fp8_quantize(z(6, 300), 128)
    with pytest.raises(ValueError, match="as many columns"):
        O.fp8_matmul(a, b)
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        O.fp8_matmul(a, a, torch.float64)
    with pytest.raises(ValueError, match="b.exps must be"):
        O.fp8_matmul(O.fp8_quantize(z(4, 600)), b._replace(shape=(6, 600), codes=z(6, 640, dtype=torch.uint8)))
    with pytest.raises(ValueError, match="a.codes must be"):
        O.fp8_matmul(a._replace(codes=a.codes[:, :200]), a)
    with pytest.raises(ValueError, match="w's 300 columns"):
        O.fp8_linear(z(2, 200), b)
    with pytest.raises(ValueError, match="for inference"):
        O.fp8_linear(z(2, 300).requires_grad_(True), b)
    with pytest.raises(ValueError, match="must be a matrix"):
        O.fp8_linear(z(2, 300), z(5, 301))
