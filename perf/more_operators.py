"""The operators that a sequence model of a texture's symbols is made of, as timed and checked cases.

Three operators and their gradients: layer norm with its weight's and bias's gradient (`op: norm`), rotary positions of several axes
on queries and keys (`op: rotary`; a texel's channel, row and column, or time, height and width), and causal attention with grouped heads over
packed sequences or a cache (`op: attention`). prepare() gives what a program holds before the call, run() makes the call - in the framework's
kernels where `own` is true, else in elementary torch operations in 32 bits - and exact() is the same result in 64 bits from the
definitions.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5
MOST_NORM, MOST_TURNED, MOST_SCORES = 16384 * 8192, 50176 * 32 * 128, 2 ** 32


def listed():
    return [
        # one symbol's row, as a decoder asks for it: latency
        {"name": "norm_one", "op": "norm", "path": "infer", "N": 1, "C": 256, "dtype": "bf16", "weights": "bf16"},
        # a training step's rows in a 256-wide model of 65536 symbols
        {"name": "norm_symbols", "op": "norm", "path": "train", "N": 65536, "C": 256, "dtype": "bf16", "weights": "bf16"},
        # ragged rows, 32-bit weights beside 16-bit values
        {"name": "norm_odd", "op": "norm", "path": "train", "N": 5003, "C": 1601, "dtype": "fp16", "weights": "fp32"},
        # the largest: a wide model's values, with their gradient
        {"name": "norm_wide", "op": "norm", "path": "train", "N": 16384, "C": 8192, "dtype": "bf16", "weights": "bf16"},
        # one token's queries and keys at a far time: latency
        {"name": "turn_one", "op": "rotary", "path": "infer", "grid": "1,1,1", "far": 1000003, "Hq": 32, "Hk": 8, "D": 128, "sections": "16,24,24", "one_ladder": True, "interleaved": False, "dtype": "bf16"},
        # 128 x 128 texels of four channels: channel, row and column, each with frequencies of its own, and both gradients
        {"name": "turn_texels", "op": "rotary", "path": "train", "grid": "128,128,4", "far": 0, "Hq": 8, "Hk": 8, "D": 32, "sections": "6,6,4", "one_ladder": False, "interleaved": False, "dtype": "bf16"},
        # the largest: frames of a clip, neighbouring elements paired, a part of each head left as it is
        {"name": "turn_frames", "op": "rotary", "path": "infer", "grid": "49,32,32", "far": 100000, "Hq": 24, "Hk": 8, "D": 128, "sections": "16,20,20", "one_ladder": False, "interleaved": True, "dtype": "bf16"},
        # a token for each of 16 sequences against a cache of up to 8192 rows: bound by the cache's bytes
        {"name": "attend_token", "op": "attention", "path": "infer", "form": "cache", "q": "1", "k": "16:900:8192", "Hq": 32, "Hk": 8, "D": 128, "dtype": "bf16"},
        # a training step over 64 tiles of at most 16 x 16 texels of four channels, those of the edges smaller
        {"name": "attend_tiles", "op": "attention", "path": "train", "form": "packed", "q": "64:600:1024", "k": "", "Hq": 8, "Hk": 8, "D": 32, "dtype": "bf16"},
        # prompts of different lengths, four query heads to a key head
        {"name": "attend_prompts", "op": "attention", "path": "infer", "form": "packed", "q": "7:300:4096", "k": "", "Hq": 32, "Hk": 8, "D": 128, "dtype": "bf16"},
        # everything ragged: queries and keys of other lengths (none, one, more queries than keys), 72 wide heads, groups of three
        {"name": "attend_odd", "op": "attention", "path": "train", "form": "cross", "q": "13:1:777", "k": "13:0:1301", "Hq": 6, "Hk": 2, "D": 72, "dtype": "fp16"},
        # the largest: one long sequence with its gradients
        {"name": "attend_long", "op": "attention", "path": "train", "form": "packed", "q": "1:8192:8192", "k": "", "Hq": 16, "Hk": 4, "D": 128, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more call: rows of 8 to 20000 values, grids of 1 to 65536 tokens, sequences of 1 to 16384 tokens in batches of 1 to 100."""
    op = rng.choice(["norm", "rotary", "attention", "attention"])
    if op == "norm":
        C = _log(rng, 8, 20000)
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        return {"op": op, "path": rng.choice(["infer", "train"]), "N": _log(rng, 1, min(300000, MOST_NORM // (2 * C))), "C": C, "dtype": dtype,
                "weights": rng.choice([dtype, "fp32"])}
    if op == "rotary":
        D = rng.choice([16, 32, 64, 80, 128, 256])
        cut = [rng.randint(1, D // 8) for _ in range(rng.choice([1, 2, 3, 3, 4]))]
        Hk = rng.choice([1, 2, 3, 4, 8])
        Hq = Hk * rng.choice([1, 1, 2, 4])
        grid, most = [], max(1, MOST_TURNED // (2 * D * (Hq + Hk)))
        for _ in cut:
            grid.append(_log(rng, 1, max(1, min(300, most))))
            most = max(1, most // grid[-1])
        return {"op": op, "path": rng.choice(["infer", "train"]), "grid": ",".join(map(str, grid)), "far": rng.choice([0, 0, 5000, 2000000]), "Hq": Hq, "Hk": Hk, "D": D,
                "sections": ",".join(map(str, cut)), "one_ladder": rng.random() < 0.5, "interleaved": rng.random() < 0.5, "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    form = rng.choice(["packed", "packed", "cross", "cache"])
    path = "infer" if form == "cache" else rng.choice(["infer", "train"])
    Hk = rng.choice([1, 2, 3, 4, 8])
    Hq = Hk * rng.choice([1, 1, 2, 3, 4, 8])
    count = _log(rng, 1, 100)
    most = MOST_SCORES // (8 if path == "train" else 3) // (count * Hq)
    least = 16 if path == "train" else 1    # (where every query has one key its gradient is 0, and all that a result holds is rounding)
    case = {"op": op, "path": path, "form": form, "Hq": Hq, "Hk": Hk, "D": rng.choice([8, 16, 32, 40, 64, 64, 72, 96, 128, 128]), "dtype": rng.choice(["bf16", "bf16", "fp16"])}
    if form == "packed":
        hi = _log(rng, least, min(16384, math.isqrt(most), 200000 // count))
        return {**case, "q": "%d:%d:%d" % (count, max(1, hi // rng.choice([1, 4, 30])), hi), "k": ""}
    if form == "cross":
        hq = _log(rng, least, min(8192, math.isqrt(most), 200000 // count))
        hk = _log(rng, least, min(16384, most // hq, 200000 // count))
        return {**case, "q": "%d:%d:%d" % (count, rng.randint(0, hq), hq), "k": "%d:%d:%d" % (count, rng.randint(0, hk), hk)}
    hk = _log(rng, 1, min(65536, 2 ** 28 // (count * Hk * case["D"])))
    return {**case, "q": str(rng.choice([1, 1, 1, 2, 5])), "k": "%d:%d:%d" % (count, rng.randint(0, hk), hk)}


# ---------------------------------------------------------------- inputs
def _device():
    return torch.device("cuda") if torch.cuda.is_available() else torch.device("cpu")


def _gen(seed):
    return torch.Generator(device=_device()).manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device=_device())


def _lengths(spec):
    """count:lo:hi as lengths spread evenly from lo to hi, in no order; the longest and the shortest are there."""
    count, lo, hi = map(int, spec.split(":"))
    return [hi - (hi - lo) * ((i * 7919) % count) // max(1, count - 1) if count > 1 else hi for i in range(count)]


def _ends(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return at


def _prepare_norm(case, seed):
    gen, N, C = _gen(seed), case["N"], case["C"]
    dtype, wtype = TYPES[case["dtype"]], TYPES[case["weights"]]
    x = _randn(gen, N, C) * (0.5 + torch.rand(C, generator=gen, device=_device())) + 0.3 * _randn(gen, 1, C) + 0.5 * _randn(gen, N, 1)
    x[:, :: max(1, C // 5)] *= 6     # a few channels far larger than the rest
    s = {"x": x.to(dtype), "w": (1 + 0.2 * _randn(gen, C)).to(wtype), "b": (0.1 * _randn(gen, C)).to(wtype)}
    if case["path"] == "train":
        for k in ("x", "w", "b"):
            s[k].requires_grad_(True)
        s["dy"] = (_randn(gen, N, C) * (1e-2 * (0.2 + torch.rand(N, 1, generator=gen, device=_device())))).to(dtype)
    return s


def _ints(text):
    return [int(x) for x in text.split(",")]


def _prepare_rotary(case, seed):
    gen, dtype = _gen(seed), TYPES[case["dtype"]]
    grid, Hq, Hk, D = _ints(case["grid"]), case["Hq"], case["Hk"], case["D"]
    N = math.prod(grid)
    at = torch.arange(N, device=_device())
    axes = []
    for n in reversed(grid):
        axes.insert(0, at % n)
        at = at // n
    axes[0] = axes[0] + case["far"] + seed % 13    # the first axis goes on from what came before
    qkv = _randn(gen, N, Hq + 2 * Hk, D).to(dtype)  # as one projection gives them
    s = {"positions": torch.stack(axes, 1), "q": qkv[:, :Hq], "k": qkv[:, Hq:Hq + Hk]}
    if case["path"] == "train":
        s["q"].requires_grad_(True)
        s["k"].requires_grad_(True)
        s["dq"], s["dk"] = (1e-2 * _randn(gen, N, Hq, D)).to(dtype), (1e-2 * _randn(gen, N, Hk, D)).to(dtype)
    return s


def _prepare_attention(case, seed):
    gen, dtype = _gen(seed), TYPES[case["dtype"]]
    Hq, Hk, D = case["Hq"], case["Hk"], case["D"]

    def made(n, h):
        x = _randn(gen, n, h, D)
        return (x * (0.5 + torch.rand(D, generator=gen, device=_device())) + 0.4 * _randn(gen, 1, h, D)).to(dtype)

    on = lambda v: torch.tensor(v, dtype=torch.int32, device=_device())  # noqa: E731
    if case["form"] == "packed":      # queries, keys and values as one projection gives them
        ends = _ends(_lengths(case["q"]))
        qkv = made(ends[-1], Hq + 2 * Hk)
        s = {"q": qkv[:, :Hq], "k": qkv[:, Hq:Hq + Hk], "v": qkv[:, Hq + Hk:], "cu_q": on(ends)}
        s["cu_k"] = s["cu_q"]
    elif case["form"] == "cross":
        eq, ek = _ends(_lengths(case["q"])), _ends(_lengths(case["k"])[::-1])
        s = {"q": made(eq[-1], Hq), "k": made(ek[-1], Hk), "v": made(ek[-1], Hk), "cu_q": on(eq), "cu_k": on(ek)}
    else:                             # a cache with room behind each sequence
        lens = _lengths(case["k"])
        room = max(1, int(max(lens) * 1.1))
        s = {"q": made(len(lens) * int(case["q"]), Hq).view(len(lens), -1, Hq, D), "k": made(len(lens) * room, Hk).view(len(lens), room, Hk, D),
             "v": made(len(lens) * room, Hk).view(len(lens), room, Hk, D), "k_lens": on(lens)}
    if case["path"] == "train":
        for k in ("q", "k", "v"):
            s[k].requires_grad_(True)
        s["do"] = (1e-2 * _randn(gen, *s["q"].shape)).to(dtype)
    return s


def prepare(case, seed):
    s = {"norm": _prepare_norm, "rotary": _prepare_rotary, "attention": _prepare_attention}[case["op"]](case, seed)
    s["case"] = case
    return s


# ---------------------------------------------------------------- the plain forms
def _plain_norm(s):
    x, w, b = s["x"].detach().float(), s["w"].detach().float(), s["b"].detach().float()
    d = x - x.mean(1, keepdim=True)
    r = torch.rsqrt((d * d).mean(1, keepdim=True) + EPS)
    h = d * r
    out = {"y": (h * w + b).to(s["x"].dtype)}
    if s["case"]["path"] == "train":
        g = s["dy"].float()
        gw = g * w
        dx = r * (gw - gw.mean(1, keepdim=True) - h * (gw * h).mean(1, keepdim=True))
        out.update(dx=dx.to(s["x"].dtype), dw=(g * h).sum(0).to(s["w"].dtype), db=g.sum(0).to(s["b"].dtype))
    return out


_LADDERS = {}


def _ladder(sections, one_ladder):
    """Each pair's axis and frequency, in 64 bits; a table that a program makes once."""
    key = (sections, one_ladder, _device())
    if key not in _LADDERS:
        n, base, pairs = _ints(sections), 10000.0, sum(_ints(sections))
        axis = [a for a, c in enumerate(n) for _ in range(c)]
        freq = [base ** (-p / pairs) for p in range(pairs)] if one_ladder else [base ** (-j / c) for c in n for j in range(c)]
        _LADDERS[key] = torch.tensor(axis, device=_device()), torch.tensor(freq, dtype=torch.float64, device=_device())
    return _LADDERS[key]


def _turned(x, cos, sin, interleaved):
    y = x.float()
    pairs = cos.shape[-1]
    if interleaved:
        a, b = y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2]
        both = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = y[..., :pairs], y[..., pairs:2 * pairs]
        both = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([both, y[..., 2 * pairs:]], -1).to(x.dtype)


def _plain_rotary(s):
    c = s["case"]
    axis, freq = _ladder(c["sections"], c["one_ladder"])
    angle = s["positions"][:, axis].double() * freq     # far positions need 64 bits
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    out = {n: _turned(s[n].detach(), cos, sin, c["interleaved"]) for n in ("q", "k")}
    if c["path"] == "train":
        out.update({n: _turned(s[n], cos, -sin, c["interleaved"]) for n in ("dq", "dk")})
    return out


def _padded(cu, lens, rows, longest):
    """[sequences, longest] row numbers, `rows` where there is none, from ends or from lengths in equal room."""
    at = torch.arange(longest, device=_device())
    if cu is not None:
        start, n = cu[:-1].long(), (cu[1:] - cu[:-1]).long()
    else:
        start, n = torch.arange(len(lens), device=_device()) * (rows // len(lens)), lens.long()
    return torch.where(at < n[:, None], start[:, None] + at, rows), n


def _plain_attention(s):
    c = s["case"]
    Hq, Hk, D = c["Hq"], c["Hk"], c["D"]
    G, scale = Hq // Hk, D ** -0.5
    q, k, v = (s[n].detach().reshape(-1, h, D) for n, h in (("q", Hq), ("k", Hk), ("v", Hk)))
    N, M = len(q), len(k)
    B = len(s["k_lens"]) if c["form"] == "cache" else len(s["cu_q"]) - 1
    Lq = int(c["q"]) if c["form"] == "cache" else max(_lengths(c["q"]))
    Lk = max(_lengths(c["k"] or c["q"]))
    if c["form"] == "cache":
        qi, nq = torch.arange(N, device=_device()).view(B, Lq), torch.full((B,), Lq, device=_device())
        ki, nk = _padded(None, s["k_lens"], M, Lk)
    else:
        (qi, nq), (ki, nk) = _padded(s["cu_q"], None, N, Lq), _padded(s["cu_k"], None, M, Lk)

    def rows(x, index, heads):     # [sequences, key heads, (the group's heads and) rows, width]
        y = torch.cat([x, x.new_zeros(1, *x.shape[1:])])[index].float()
        return y.view(B, -1, Hk, heads // Hk, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, -1, D)

    def back(y, index, like, heads):
        y = y.view(B, Hk, heads // Hk, -1, D).permute(0, 3, 1, 2, 4).reshape(-1, heads, D).to(like.dtype)
        out = like.new_zeros(len(like) + 1, heads, D)
        out[index.reshape(-1)] = y
        return out[:-1]

    Q, K, V = rows(q, qi, Hq), rows(k, ki, Hk), rows(v, ki, Hk)
    S = torch.matmul(Q, K.transpose(2, 3).contiguous()).mul_(scale).view(B, Hk, G, Lq, Lk)
    i, j = torch.arange(Lq, device=_device())[:, None], torch.arange(Lk, device=_device())
    seen = (j <= i + (nk - nq)[:, None, None]) & (j < nk[:, None, None]) & (i < nq[:, None, None])
    S.masked_fill_(~seen[:, None, None], -math.inf)
    best = S.amax(-1, keepdim=True)
    P = S.sub_(torch.where(best == -math.inf, 0.0, best)).exp_()
    total = P.sum(-1, keepdim=True)
    P = P.div_(torch.where(total == 0, 1.0, total)).view(B, Hk, G * Lq, Lk)
    O = torch.matmul(P, V)
    out = {"o": back(O, qi, q, Hq).view(s["q"].shape)}
    if c["path"] == "train":
        dO = rows(s["do"], qi, Hq)
        dV = torch.matmul(P.transpose(2, 3), dO)
        dS = torch.matmul(dO, V.transpose(2, 3).contiguous()).sub_((dO * O).sum(-1, keepdim=True)).mul_(P).mul_(scale)
        out.update(dq=back(torch.matmul(dS, K), qi, q, Hq), dk=back(torch.matmul(dS.transpose(2, 3), Q), ki, k, Hk), dv=back(dV, ki, v, Hk))
    return out


# ---------------------------------------------------------------- the framework's calls
def _own_norm(s):
    from neural_block_textures_amd import ops
    y = ops.layer_norm(s["x"], s["w"], s["b"], EPS)
    if s["case"]["path"] == "infer":
        return {"y": y}
    return {"y": y, **dict(zip(("dx", "dw", "db"), torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])))}


def _own_rotary(s):
    from neural_block_textures_amd import ops
    c = s["case"]
    q, k = ops.rotary(s["positions"], s["q"], s["k"], sections=_ints(c["sections"]), one_ladder=c["one_ladder"], interleaved=c["interleaved"])
    if c["path"] == "infer":
        return {"q": q, "k": k}
    dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
    return {"q": q, "k": k, "dq": dq, "dk": dk}


def _own_attention(s):
    from neural_block_textures_amd import ops
    o = ops.attention(s["q"], s["k"], s["v"], cu_q=s.get("cu_q"), cu_k=s.get("cu_k"), k_lens=s.get("k_lens"))
    if s["case"]["path"] == "infer":
        return {"o": o}
    return {"o": o, **dict(zip(("dq", "dk", "dv"), torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])))}


def run(s):
    kind = s["case"]["op"]
    if own:
        return {"norm": _own_norm, "rotary": _own_rotary, "attention": _own_attention}[kind](s)
    return {"norm": _plain_norm, "rotary": _plain_rotary, "attention": _plain_attention}[kind](s)


def _pairs(case):
    """Queries, keys, and the pairs of them that the mask leaves."""
    if case["form"] == "packed":
        nq = nk = _lengths(case["q"])
    else:
        nk = _lengths(case["k"])[::-1]
        nq = _lengths(case["q"]) if case["form"] == "cross" else [int(case["q"])] * len(nk)
    seen = 0
    for a, b in zip(nq, nk):
        n = min(a, b)               # the last n queries see b - n + 1 .. b keys
        seen += n * (b - n) + n * (n + 1) // 2
    return sum(nq), sum(nk), seen


def work(case):
    if case["op"] == "norm":
        N, C, size, w = case["N"], case["C"], 4 if case["dtype"] == "fp32" else 2, 4 if case["weights"] == "fp32" else 2
        if case["path"] == "infer":
            return {"bytes": 2 * N * C * size + 2 * C * w, "flops": 7 * N * C}
        return {"bytes": 4 * N * C * size + 4 * C * w, "flops": 20 * N * C}
    if case["op"] == "rotary":
        size = 4 if case["dtype"] == "fp32" else 2
        grid = _ints(case["grid"])
        N, row = math.prod(grid), (case["Hq"] + case["Hk"]) * case["D"]
        times = 1 if case["path"] == "infer" else 2
        return {"bytes": times * 2 * N * row * size + 8 * N * len(grid), "flops": times * 3 * N * row}
    nq, nk, seen = _pairs(case)
    Hq, Hk, D = case["Hq"], case["Hk"], case["D"]
    q, k = 2 * nq * Hq * D, 2 * nk * Hk * D
    if case["path"] == "infer":
        return {"bytes": 2 * q + 2 * k, "flops": 4 * D * Hq * seen}
    return {"bytes": 4 * q + 4 * k, "flops": 14 * D * Hq * seen}


# ---------------------------------------------------------------- the definitions in 64 bits
def _exact_norm(s):
    x, w = s["x"].detach().double(), s["w"].detach().double()
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    sd = torch.sqrt(var + EPS)
    h = (x - mean) / sd
    out = {"y": torch.addcmul(s["b"].detach().double(), h, w)}
    if "dy" in s:
        g = s["dy"].double()
        t = g * w / sd
        dx = t - t.mean(1, keepdim=True)
        dx -= h * (t * h).mean(1, keepdim=True)
        out.update(dx=dx, dw=torch.einsum("nc,nc->c", g, h), db=g.sum(0))
    return out


def _exact_rotary(s):
    c = s["case"]
    n, total = _ints(c["sections"]), sum(_ints(c["sections"]))
    angle, done = [], 0
    for a, pairs in enumerate(n):
        j = torch.arange(pairs, dtype=torch.float64, device=_device())
        exponent = (j + done) / total if c["one_ladder"] else j / pairs
        angle.append(s["positions"][:, a:a + 1].double() * torch.pow(10000.0, -exponent))
        done += pairs
    angle = torch.cat(angle, 1)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]

    def turned(x, t):
        x = x.detach().double()
        held, rest = x[..., :2 * total], x[..., 2 * total:]
        held = held.unflatten(-1, (total, 2)) if c["interleaved"] else held.unflatten(-1, (2, total)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(held.contiguous()) * t)
        z = z.flatten(-2) if c["interleaved"] else z.transpose(-1, -2).flatten(-2)
        return torch.cat([z, rest], -1)

    out = {k: turned(s[k], turn) for k in ("q", "k")}
    if c["path"] == "train":
        out.update({k: turned(s[k], turn.conj()) for k in ("dq", "dk")})
    return out


def _exact_attention(s):
    c = s["case"]
    Hq, Hk, D = c["Hq"], c["Hk"], c["D"]
    train = c["path"] == "train"
    q, k, v = (s[n].detach().double().reshape(-1, h, D) for n, h in (("q", Hq), ("k", Hk), ("v", Hk)))
    do = s["do"].double() if train else None
    if c["form"] == "cache":
        lens = s["k_lens"].tolist()
        room, step = s["k"].shape[1], s["q"].shape[1]
        spans = [(b * step, (b + 1) * step, b * room, b * room + n) for b, n in enumerate(lens)]
    else:
        a, b = s["cu_q"].tolist(), s["cu_k"].tolist()
        spans = list(zip(a[:-1], a[1:], b[:-1], b[1:]))
    o, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for q0, q1, k0, k1 in spans:
        n, m = q1 - q0, k1 - k0
        if not n or not m:
            continue
        seen = torch.ones(n, m, dtype=torch.bool, device=q.device).tril(m - n)
        for h in range(Hq):
            e = h // (Hq // Hk)
            a, kk, vv = q[q0:q1, h], k[k0:k1, e], v[k0:k1, e]
            z = (a @ kk.T / math.sqrt(D)).masked_fill(~seen, -math.inf)
            p = torch.nan_to_num(torch.softmax(z, 1), nan=0.0)
            o[q0:q1, h] = p @ vv
            if train:
                g = do[q0:q1, h]
                dv[k0:k1, e] += p.T @ g
                t = g @ vv.T
                t = p * (t - (p * t).sum(1, keepdim=True)) / math.sqrt(D)
                dq[q0:q1, h] = t @ kk
                dk[k0:k1, e] += t.T @ a
    out = {"o": o.view(s["q"].shape)}
    if train:
        out.update(dq=dq, dk=dk, dv=dv)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "rotary": _exact_rotary, "attention": _exact_attention}[case["op"]](s)
