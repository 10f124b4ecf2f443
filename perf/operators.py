"""The operators that a learned prior over a texture's symbols is made of, as timed and checked cases.

Three operators and their gradients: the log probabilities of given tokens with the entropy and the best alternatives
(`op: logprobs`; the bits an arithmetic coder would spend on each symbol, and a training step's loss), an AdamW step over
many tensors with its state in 32 or 8 bits (`op: adamw`), and linear layers whose products run in 8-bit floating point
with a power-of-two scale for each block of 128 (`op: linear`). prepare() gives what a program holds before the call, run()
makes the call - in the framework's kernels where `own` is true, else in elementary torch operations in 32 bits - and
exact() is the same result in 64 bits from the definitions.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 256                 # values that share one scale of an 8-bit optimizer state
LR, BETAS, EPS, DECAY, STEP, ADAM_SEED = 2e-3, (0.9, 0.999), 1e-8, 0.05, 40, 11
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
IGNORE = -100
MOST_LOGITS, MOST_PARAMS, MOST_MACS = 4096 * 131072, 2 ** 28, 2 ** 39


def listed():
    return [
        # one position of a large symbol alphabet, as a decoder asks for it: latency
        {"name": "lp_one", "op": "logprobs", "path": "score", "N": 1, "V": 131072, "dtype": "bf16", "top": 8, "temperature": 1.0, "masked": 0.0, "shifted": False},
        # a 512 x 512 latent level of 8-bit symbols: the bits of every texel, four alternatives each
        {"name": "lp_symbols", "op": "logprobs", "path": "score", "N": 262144, "V": 256, "dtype": "bf16", "top": 4, "temperature": 1.0, "masked": 0.0, "shifted": False},
        # the largest: whole sequences over a large alphabet, sharpened, many alternatives
        {"name": "lp_large", "op": "logprobs", "path": "score", "N": 4096, "V": 131072, "dtype": "bf16", "top": 16, "temperature": 0.7, "masked": 0.0, "shifted": False},
        # a training step: odd sizes, logits shifted against their tokens, a tenth of the alphabet masked, an entropy bonus
        {"name": "lp_train_odd", "op": "logprobs", "path": "train", "N": 8190, "V": 50001, "dtype": "bf16", "top": 0, "temperature": 1.0, "masked": 0.1, "shifted": True},
        # the decoder of this framework's headline workload (8-32-32-12): six small tensors, launches and latency
        {"name": "adamw_decoder", "op": "adamw", "sizes": "256,32,1024,32,384,12", "dtype": "fp32", "bits": 32, "master": False, "odd": False},
        # a model of 240 tensors of ragged sizes (norms, biases, matrices), 8-bit state
        {"name": "adamw8_ragged", "op": "adamw", "sizes": "ragged:240:1:400000", "dtype": "bf16", "bits": 8, "master": False, "odd": False},
        # 2^28 weights in 16 bits with a 32-bit copy and 32-bit state
        {"name": "adamw_large", "op": "adamw", "sizes": "equal:16:16777216", "dtype": "bf16", "bits": 32, "master": True, "odd": False},
        # the same with an 8-bit state and no copy: a quarter of the bytes
        {"name": "adamw8_large", "op": "adamw", "sizes": "equal:16:16777216", "dtype": "bf16", "bits": 8, "master": False, "odd": False},
        # one row through a prepared layer: a texel at a time, bound by the weights' bytes
        {"name": "linear_one", "op": "linear", "path": "infer", "M": 1, "K": 4096, "N": 4096, "dtype": "bf16"},
        # a 256-wide layer of the prior on 65536 texels: the layer, and both gradients
        {"name": "linear_prior", "op": "linear", "path": "train", "M": 65536, "K": 256, "N": 256, "dtype": "bf16"},
        # everything ragged
        {"name": "linear_odd", "op": "linear", "path": "train", "M": 1003, "K": 1500, "N": 2077, "dtype": "fp16"},
        # the largest product
        {"name": "linear_large", "op": "linear", "path": "infer", "M": 8192, "K": 8192, "N": 8192, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more call: alphabets of 32 to 200 thousand symbols, 1 to 2^28 weights in 1 to 400 tensors, layers of 1 to 65536 rows."""
    op = rng.choice(["logprobs", "adamw", "linear"])
    if op == "logprobs":
        V = _log(rng, 32, 200000)
        path = rng.choice(["score", "train"])
        shifted = rng.random() < 0.3
        N = _log(rng, 1, min(400000, MOST_LOGITS // (8 * V)))
        return {"op": op, "path": path, "N": 2 * -(-N // 2) if shifted else N, "V": V, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "top": rng.choice([0, 1, 4, 8, 16, 32]),
                "temperature": rng.choice([0.6, 1.0, 1.0, 1.3]), "masked": rng.choice([0.0, 0.0, 0.2]), "shifted": shifted}
    if op == "adamw":
        count = _log(rng, 1, 400)
        most = _log(rng, 64, min(2 ** 25, MOST_PARAMS // (2 * count)))
        return {"op": op, "sizes": "ragged:%d:%d:%d" % (count, rng.choice([1, max(1, most // 50)]), most), "dtype": rng.choice(["bf16", "fp16", "fp32"]),
                "bits": rng.choice([8, 32]), "master": rng.random() < 0.4, "odd": rng.random() < 0.3}
    path = rng.choice(["infer", "train"])
    M, K = _log(rng, 1, 65536), _log(rng, 64, 12000)
    N = _log(rng, 64, min(12000, max(65, MOST_MACS // (4 * M * K))))
    return {"op": op, "path": path, "M": M, "K": K, "N": N, "dtype": rng.choice(["bf16", "bf16", "fp16"])}


# ---------------------------------------------------------------- inputs
def _device():
    return torch.device("cuda") if torch.cuda.is_available() else torch.device("cpu")


def _gen(seed):
    return torch.Generator(device=_device()).manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device=_device())


def _tensor_sizes(spec):
    if ":" not in spec:
        return [int(x) for x in spec.split(",")]
    kind, count, *rest = spec.split(":")
    count = int(count)
    if kind == "equal":
        return [int(rest[0])] * count
    lo, hi = int(rest[0]), int(rest[1])
    # sizes spread over the logarithm, in no order, odd ones among them; the largest and the smallest are there
    return [int(round(lo * (hi / lo) ** (((k * 7919) % count) / max(1, count - 1)))) for k in range(count)]


def _offsets(case):
    """Where each tensor's state starts (a multiple of 256 values), and their end."""
    sizes, at = _tensor_sizes(case["sizes"]), [0]
    for n in sizes:
        at.append(at[-1] + -(-n // BLOCK) * BLOCK)
    return sizes, at[:-1], at[-1]


def _prepare_logprobs(case, seed):
    gen, N, V = _gen(seed), case["N"], case["V"]
    dtype = TYPES[case["dtype"]]
    # a trained model's logits: a few symbols well above the rest; in two sequences where rows are shifted against tokens
    rows = N + 2 if case["shifted"] else N
    logits = torch.empty(rows, V, dtype=dtype, device=_device())
    for r in range(0, rows, max(1, 2 ** 27 // V)):
        part = logits[r:r + max(1, 2 ** 27 // V)]
        x = _randn(gen, *part.shape) * 2.5
        x += 4 * (torch.rand(part.shape, generator=gen, device=x.device) < 4 / V)
        part.copy_(x)
    tokens = torch.randint(0, V, (rows,), generator=gen, device=_device())
    likely = torch.rand(rows, generator=gen, device=_device()) < 0.7
    tokens = torch.where(likely, logits[:, : min(V, 4096)].argmax(1), tokens)
    if case["masked"]:  # symbols that cannot follow
        logits[:, torch.rand(V, generator=gen, device=_device()) < case["masked"]] = -math.inf
        tokens[torch.rand(rows, generator=gen, device=_device()) < 0.05] = IGNORE
    if case["shifted"]:  # the logits of each position but a sequence's last, the tokens of each but its first
        logits, tokens = logits.view(2, rows // 2, V)[:, :-1], tokens.view(2, rows // 2)[:, 1:]
    s = {"logits": logits, "tokens": tokens}
    if case["path"] == "train":
        shape = tokens.shape
        s["g_logprob"] = -torch.rand(shape, generator=gen, device=_device()) / N
        s["g_entropy"] = -0.01 * torch.rand(shape, generator=gen, device=_device()) / N
        s["g_top"] = _randn(gen, *shape, case["top"]) * (0.1 / N)
        logits.requires_grad_(True)
    return s


def _prepare_adamw(case, seed):
    gen, dtype = _gen(seed), TYPES[case["dtype"]]
    sizes, at, total = _offsets(case)
    live = torch.zeros(total, dtype=torch.bool, device=_device())
    for n, o in zip(sizes, at):
        live[o:o + n] = True
    first = 1 if case["odd"] else 0     # weights that start at an odd element of their buffer

    def flat(x):
        whole = torch.zeros(total + first, dtype=dtype, device=_device())
        whole[first:] = x
        return whole[first:]

    # gradients of very different size from tensor to tensor and from weight to weight, as a network has
    size = 10 ** (-2 - 2 * torch.rand(total // BLOCK, generator=gen, device=_device())).repeat_interleave(BLOCK)
    w = _randn(gen, total) * 0.05 * live
    s = {"case": case, "step": STEP, "p": flat(w), "g": flat(_randn(gen, total) * size * live),
         "master": w.clone() if case["master"] else None}
    m = _randn(gen, total) * size * 0.3 * live
    v = (_randn(gen, total) * size).square_().mul_(0.04) * live
    if case["bits"] == 8:
        half = torch.full((total,), 32768, dtype=torch.int32, device=_device())
        s["m"], s["m_exp"] = _encode(m, 15, half)
        s["v"], s["v_exp"] = _encode(v, 31, half)
    else:
        s["m"], s["v"] = m, v
    if own:  # the optimizer a program keeps: built once over its tensors, and the state put back into it
        from neural_block_textures_amd import ops
        cut = lambda x: [x[o:o + n] for n, o in zip(sizes, at)]  # noqa: E731
        s["params"], s["grads"] = cut(s["p"]), cut(s["g"])
        s["opt"] = ops.AdamW(s["params"], lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=case["bits"], master=case["master"], seed=ADAM_SEED)
        state = {"step": STEP, "exp_avg": s.pop("m"), "exp_avg_sq": s.pop("v"), "master": s.pop("master")}
        if case["bits"] == 8:
            state.update(exp_avg_exp=s.pop("m_exp"), exp_avg_sq_exp=s.pop("v_exp"))
        s["opt"].load_state_dict(state)
    return s


def _prepare_linear(case, seed):
    gen, dtype = _gen(seed), TYPES[case["dtype"]]
    M, N, K = case["M"], case["N"], case["K"]
    x = _randn(gen, M, K) * (0.3 + 2 * torch.rand(K, generator=gen, device=_device()))  # channels of different size, some rows' outliers
    x[:, :: max(1, K // 7)] *= 8
    w = _randn(gen, N, K) * K ** -0.5
    s = {"case": case, "x": x.to(dtype), "w": w.to(dtype)}
    if case["path"] == "infer":  # the weights are laid out once
        s["w_codes"], s["w_exps"] = _quantize(s.pop("w").float(), 128)
    else:
        s["x"].requires_grad_(True)
        s["w"].requires_grad_(True)
        s["dy"] = (_randn(gen, M, N) * (1e-3 * (0.2 + torch.rand(M, 1, generator=gen, device=_device())))).to(dtype)
    return s


def prepare(case, seed):
    s = {"logprobs": _prepare_logprobs, "adamw": _prepare_adamw, "linear": _prepare_linear}[case["op"]](case, seed)
    s["case"] = case
    return s


# ---------------------------------------------------------------- the plain forms
def _plain_logprobs(s):
    c = s["case"]
    V = c["V"]
    x = s["logits"].detach().float().reshape(-1, V)
    tokens = s["tokens"].reshape(-1)
    y = x / c["temperature"]
    best = y.amax(1, keepdim=True)
    d = y - torch.where(best == -math.inf, 0.0, best)
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    lse = best + torch.log(total)
    entropy = (torch.log(total) - (e * d.clamp_min(-1e30)).sum(1, keepdim=True) / total)[:, 0]
    entropy = torch.where(best[:, 0] == -math.inf, 0.0, entropy)
    given = tokens != IGNORE
    at = torch.where(given, tokens, 0)[:, None]
    logprob = torch.where(given, (y.gather(1, at) - lse.clamp_min(-3e38))[:, 0], 0.0)
    out = {"logprob": logprob.view(s["tokens"].shape), "entropy": entropy.view(s["tokens"].shape)}
    if c["top"]:
        bits = (x + 0.0).view(torch.int32).long()
        order = torch.where(bits < 0, -2147483648 - bits, bits)    # integers in the floats' order
        order = (order << 32) | (0xffffffff - torch.arange(V, device=x.device))
        ids = 0xffffffff - (torch.topk(order, c["top"], dim=1).values & 0xffffffff)
        out["top_ids"] = ids.view(*s["tokens"].shape, -1)
        out["top_logprobs"] = (y.gather(1, ids) - lse.clamp_min(-3e38)).view(*s["tokens"].shape, -1)
    if c["path"] == "train":
        logp = d - torch.log(total)
        p = e / total
        g = torch.where(given, s["g_logprob"].reshape(-1), 0.0)[:, None]
        gh = s["g_entropy"].reshape(-1, 1)
        dx = -p * (g + gh * (logp.clamp_min(-1e30) + entropy[:, None]))
        dx.scatter_add_(1, at, g)
        if c["top"]:
            gt = s["g_top"].reshape(-1, c["top"])
            dx -= p * gt.sum(1, keepdim=True)
            dx.scatter_add_(1, ids, gt)
        dx = torch.where(best == -math.inf, 0.0, dx) / c["temperature"]
        out["dlogits"] = dx.to(s["logits"].dtype).view(s["logits"].shape)
    return out


_TABLES = {}


def _table(top):
    """The values of the 128 (top 15) or 256 (top 31) codes whose largest exponent stands for [1, 2)."""
    key = (top, _device())
    if key not in _TABLES:
        values = [(8 + n % 8) * 2.0 ** (n // 8 - top - 3) if n >= 8 else n * 2.0 ** (-2 - top) for n in range(8 * (top + 1))]
        _TABLES[key] = torch.tensor(values, device=_device())
    return _TABLES[key]


def _power(byte):
    """2^(byte - 127)"""
    byte = byte.to(torch.int32)
    return torch.where(byte > 0, byte << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _encode(x, top, r16):
    """Codes (a sign bit where top is 15, exponents to `top`, 3 bits of mantissa) and a power of two for each 256 values, from
    16 random bits a value: rounded up as often as it is above the lower code. A positive value never becomes 0."""
    a = x.abs().view(-1, BLOCK)
    most = a.amax(1).view(torch.int32)
    byte = (most >> 23) + ((most & 0x7fffff) > 0x700000).int()
    y = (a * _power(254 - byte)[:, None]).view(-1)
    normal = ((y.view(torch.int32) + (r16 << 4)) >> 20) - 8 * (127 - top)
    small = torch.floor(y * 2.0 ** (top + 2) + r16.float() * 2.0 ** -16).int()
    code = torch.where(y >= 2.0 ** (1 - top), normal, small)
    if top == 31:
        code = torch.where((y > 0) & (code == 0), 1, code)
    else:
        code = code | torch.where(x < 0, 128, 0)
    return code.to(torch.uint8), byte.to(torch.uint8)


def _decode(code, byte, top):
    c = code.int()
    v = _table(top)[c if top == 31 else c & 127]
    if top == 15:
        v = torch.where(c >= 128, -v, v)
    return (v.view(-1, BLOCK) * _power(byte)[:, None]).view(-1)


def _mix(x):
    """splitmix64's output function of 64-bit counters, as the framework draws its random numbers."""
    x = x + -7046029254386353131
    x = (x ^ ((x >> 30) & ((1 << 34) - 1))) * -4658895280553007687
    x = (x ^ ((x >> 27) & ((1 << 37) - 1))) * -7723592293110705685
    return x ^ ((x >> 31) & ((1 << 33) - 1))


def _random16(n, step, device):
    head = ADAM_SEED ^ (5 << 56) ^ (step << 32)
    head = _mix(torch.tensor([head], device=device))
    bits = _mix(head + torch.arange((n + 1) // 2, device=device) * -7046029254386353131)
    bits = torch.stack([bits & 0xffff, (bits >> 16) & 0xffff, (bits >> 32) & 0xffff, (bits >> 48) & 0xffff], 1).to(torch.int32)
    return bits[:, 0::2].reshape(-1)[:n], bits[:, 1::2].reshape(-1)[:n]


def _plain_adamw(s):
    c = s["case"]
    s["step"] += 1
    t, (b1, b2) = s["step"], BETAS
    g = s["g"].float()
    p = (s["master"] if c["master"] else s["p"]).float()
    m, v = s["m"], s["v"]
    if c["bits"] == 8:
        m, v = _decode(m, s["m_exp"], 15), _decode(v, s["v_exp"], 31)
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    p = p * (1 - LR * DECAY) - (LR / (1 - b1 ** t)) * (m / (torch.sqrt(v) * (1 / math.sqrt(1 - b2 ** t)) + EPS))
    if c["bits"] == 8:
        rm, rv = _random16(m.numel(), t, m.device)
        s["m"], s["m_exp"] = _encode(m, 15, rm)
        s["v"], s["v_exp"] = _encode(v, 31, rv)
        m, v = _decode(s["m"], s["m_exp"], 15), _decode(s["v"], s["v_exp"], 31)
    else:
        s["m"], s["v"] = m, v
    if c["master"]:
        s["master"] = p
    s["p"].copy_(p)
    return {"p": s["p"], "m": m, "v": v, "master": s["master"]}


def _exponents(amax):
    """The smallest power of two s with amax / s <= 448, as its exponent + 127 (0 at least)."""
    bits = amax.view(torch.int32)
    return ((bits >> 23) - 8 + ((bits & 0x7fffff) > 0x600000).int()).clamp_min(0)


def _quantize(x, rows):
    """8-bit codes and one exponent for each `rows` x 128 values: columns padded with zeros to whole blocks, the
    exponents' to a multiple of four."""
    R, K = x.shape
    x = torch.nn.functional.pad(x, (0, -K % 128, 0, -R % rows))
    b = x.view(x.shape[0] // rows, rows, -1, 128)
    byte = _exponents(b.abs().amax(dim=(1, 3)))
    codes = (b * _power(254 - byte)[:, None, :, None]).to(torch.float8_e4m3fn).view(x.shape)[:R]
    return codes.view(torch.uint8), torch.nn.functional.pad(byte.to(torch.uint8), (0, -byte.shape[1] % 4))


def _values(codes, byte, rows):
    x = codes.view(torch.float8_e4m3fn).float()
    scale = _power(byte[:, : x.shape[1] // 128]).repeat_interleave(128, 1)
    return x * (scale.repeat_interleave(rows, 0)[: x.shape[0]] if rows > 1 else scale)


def _plain_linear(s):
    c = s["case"]
    dtype, K = TYPES[c["dtype"]], c["K"]
    x = s["x"].detach().float()
    if c["path"] == "infer":
        return {"y": (_values(*_quantize(x, 1), 1) @ _values(s["w_codes"], s["w_exps"], 128).T).to(dtype)}
    dy = s["dy"].float()
    w = _values(*_quantize(s["w"].detach().float(), 128), 128)[:, :K]
    y = _values(*_quantize(x, 1), 1)[:, :K] @ w.T
    dx = _values(*_quantize(dy, 1), 1)[:, : c["N"]] @ w
    dw = _values(*_quantize(dy.T.contiguous(), 1), 1) @ _values(*_quantize(x.T.contiguous(), 1), 1).T
    return {"y": y.to(dtype), "dx": dx.to(dtype), "dw": dw.to(dtype)}


# ---------------------------------------------------------------- the framework's calls
def _own_logprobs(s):
    from neural_block_textures_amd import ops
    c = s["case"]
    r = ops.token_logprobs(s["logits"], s["tokens"], top=c["top"], temperature=c["temperature"], ignore_index=IGNORE)
    out = {"logprob": r.logprob, "entropy": r.entropy}
    if c["top"]:
        out.update(top_ids=r.top_ids, top_logprobs=r.top_logprobs)
    if c["path"] == "train":
        outs, gs = [r.logprob, r.entropy], [s["g_logprob"], s["g_entropy"]]
        if c["top"]:
            outs, gs = outs + [r.top_logprobs], gs + [s["g_top"]]
        out["dlogits"] = torch.autograd.grad(outs, s["logits"], gs)[0]
    return out


def _own_adamw(s):
    opt = s["opt"]
    opt.step(s["grads"])
    m, v = opt.moments()
    return {"p": s["p"], "m": m, "v": v, "master": opt.master}


def _own_linear(s):
    from neural_block_textures_amd import ops
    c = s["case"]
    if c["path"] == "infer":
        return {"y": ops.fp8_linear(s["x"], ops.Fp8Tensor(s["w_codes"], s["w_exps"], (c["N"], c["K"]), 128))}
    y = ops.fp8_linear(s["x"], s["w"])
    dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
    return {"y": y, "dx": dx, "dw": dw}


def run(s):
    kind = s["case"]["op"]
    if own:
        return {"logprobs": _own_logprobs, "adamw": _own_adamw, "linear": _own_linear}[kind](s)
    return {"logprobs": _plain_logprobs, "adamw": _plain_adamw, "linear": _plain_linear}[kind](s)


def work(case):
    if case["op"] == "logprobs":
        size = 4 if case["dtype"] == "fp32" else 2
        N, V, K = case["N"], case["V"], case["top"]
        b = N * V * size + N * (8 + 8) + N * K * 12
        if case["path"] == "train":
            return {"bytes": b + N * V * size + N * (8 + 4 * K), "flops": 14 * N * V}
        return {"bytes": b, "flops": 6 * N * V}
    if case["op"] == "adamw":
        size = 4 if case["dtype"] == "fp32" else 2
        n = sum(_tensor_sizes(case["sizes"]))
        state = 4 + 4 / BLOCK + 8 if case["bits"] == 8 else 16    # 8-bit states are also given back as the values they stand for
        p = size + 8 if case["master"] else 2 * size
        return {"bytes": int(n * (p + size + state)), "flops": 16 * n}
    M, N, K = case["M"], case["N"], case["K"]
    if case["path"] == "infer":
        return {"bytes": 2 * M * K + N * K + 2 * M * N, "flops": 2 * M * N * K}
    return {"bytes": 2 * (2 * M * K + 2 * N * K + 2 * M * N), "flops": 6 * M * N * K}


# ---------------------------------------------------------------- the definitions in 64 bits
def _two(e):
    """2^e in 64 bits, exactly"""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _binade(x):
    """the e of 2^e <= x < 2^(e+1)"""
    return torch.frexp(x).exponent - 1


def _exact_logprobs(s):
    c = s["case"]
    shape, V, T = s["tokens"].shape, c["V"], c["temperature"]
    tokens = s["tokens"].reshape(-1)
    rows = s["logits"].detach().reshape(-1, V)
    parts = []
    for r in range(0, len(tokens), max(1, 2 ** 28 // V)):
        some = slice(r, r + max(1, 2 ** 28 // V))
        y, tok = rows[some].double() / T, tokens[some]
        logp = torch.log_softmax(y, 1)
        p = torch.exp(logp)
        finite = torch.where(p > 0, logp, 0.0)
        entropy = -(p * finite).sum(1)
        given = tok != IGNORE
        at = torch.where(given, tok, 0)[:, None]
        o = {"logprob": torch.where(given, logp.gather(1, at)[:, 0], 0.0), "entropy": entropy}
        if c["top"]:
            o["top_logprobs"], _ = torch.topk(logp, c["top"], dim=1)
        if c["path"] == "train":
            g = torch.where(given, s["g_logprob"].reshape(-1)[some].double(), 0.0)[:, None]
            gsum, gh = g, s["g_entropy"].reshape(-1)[some].double()[:, None]
            dx = torch.zeros_like(y).scatter_(1, at, g)
            if c["top"]:
                gt = s["g_top"].reshape(len(tokens), -1)[some].double()
                order = torch.sort(y, dim=1, descending=True, stable=True).indices[:, : c["top"]]
                dx.scatter_add_(1, order, gt)
                gsum = g + gt.sum(1, keepdim=True)
            o["dlogits"] = (dx - p * gsum - gh * p * (finite + entropy[:, None])) / T
        parts.append(o)
    out = {k: torch.cat([o[k] for o in parts]) for k in parts[0]}
    out = {k: v.view(*shape, *v.shape[1:]) for k, v in out.items()}
    if c["top"]:
        out["top_ids"] = None
    return out


def _exact_adamw(s):
    c = s["case"]
    t, (b1, b2) = s["step"] + 1, BETAS
    g = s["g"].double()
    p = (s["master"] if c["master"] else s["p"]).double()

    def value(code, byte, top):
        n = code.long()
        sign = torch.where(n >= 128, -1.0, 1.0) if top == 15 else 1.0
        n = n & 127 if top == 15 else n
        e, f = n >> 3, (n & 7).double()
        x = torch.where(e > 0, (8 + f) * _two(e - top - 3), f * 2 ** (-2.0 - top))
        return sign * x * _two(byte.long() - 127).repeat_interleave(BLOCK)

    def stored(x, top, r):
        most = x.abs().view(-1, BLOCK).amax(1)
        scale = torch.where(most > 0, _two(_binade(most)), 1.0)
        scale = torch.where(most > 1.875 * scale, 2 * scale, scale).repeat_interleave(BLOCK)
        y = x.abs() / scale
        unit = _two(_binade(y.clamp_min(2.0 ** (1 - top))) - 3)
        k = torch.floor(y / unit + r.double() / 65536)
        if top == 31:
            k = torch.where((y > 0) & (k == 0), 1.0, k)
        return torch.sign(x) * k * unit * scale

    if c["bits"] == 8:
        m, v = value(s["m"], s["m_exp"], 15), value(s["v"], s["v_exp"], 31)
    else:
        m, v = s["m"].double(), s["v"].double()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p = p * (1 - LR * DECAY) - LR * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + EPS)
    if c["bits"] == 8:
        rm, rv = _random16(m.numel(), t, m.device)
        m, v = stored(m, 15, rm), stored(v, 31, rv)
    return {"p": p, "m": m, "v": v, "master": p if c["master"] else None}


def _exact_quantized(x, rows):
    """x as it stands in 8 bits, in 64: each `rows` x 128 block over its power of two, rounded to four significant bits."""
    R, K = x.shape
    b = torch.nn.functional.pad(x.double(), (0, -K % 128, 0, -R % rows)).view(-(-R // rows), rows, -1, 128)
    most = b.abs().amax(dim=(1, 3), keepdim=True)
    scale = torch.where(most > 0, _two(_binade(most) - 8), 1.0)
    scale = torch.where(most > 448 * scale, 2 * scale, scale).clamp_min(2.0 ** -127)
    y = b / scale
    unit = _two(_binade(y.abs().clamp_min(2.0 ** -6)) - 3)
    return (torch.round(y / unit) * unit * scale).view(-(-R // rows) * rows, -1)[:R, :K]


def _exact_linear(s):
    c = s["case"]
    x = _exact_quantized(s["x"].detach(), 1)
    if c["path"] == "infer":
        codes = s["w_codes"].view(torch.float8_e4m3fn).double()
        scale = _two(s["w_exps"].long() - 127).repeat_interleave(128, 0).repeat_interleave(128, 1)
        return {"y": x @ (codes * scale[: c["N"], : codes.shape[1]])[:, : c["K"]].T}
    w = _exact_quantized(s["w"].detach(), 128)
    dy, dyt, xt = _exact_quantized(s["dy"], 1), _exact_quantized(s["dy"].T, 1), _exact_quantized(s["x"].detach().T, 1)
    return {"y": x @ w.T, "dx": dy @ w, "dw": dyt @ xt.T}


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
        return {"logprobs": _exact_logprobs, "adamw": _exact_adamw, "linear": _exact_linear}[case["op"]](s)
    finally:
        own = was
