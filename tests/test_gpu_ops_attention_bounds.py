"""attention's C entry points inside their buffers: ends and lengths that leave the rows, go backwards or overlap are cut off before any address. What surrounds the operands is NaN, and shows in no result; what
surrounds results and workspaces is as it was."""
import ctypes as C

import pytest
import torch

from neural_block_textures_amd import ops

pytestmark = pytest.mark.gpu
TYPES = {"bf16": (torch.bfloat16, 1), "fp16": (torch.float16, 2)}
PAD = 4096                                                # elements before and behind


class Inside:
    """A buffer in the midst of `around`"""

    def __init__(self, n, dtype, around, fill):
        self.whole = torch.full((n + 2 * PAD,), around, dtype=dtype, device="cuda")
        self.own, self.n = self.whole[PAD:PAD + n], n
        self.own.fill_(fill) if not isinstance(fill, torch.Tensor) else self.own.copy_(fill.reshape(-1))
        self.before = self.whole.clone()

    def untouched(self):
        a, b = (torch.cat([x[:PAD], x[PAD + self.n:]]).view(torch.uint8) for x in (self.whole, self.before))
        return torch.equal(a, b)


def randn(seed, *shape):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def run(entry, d, backward):
    size = ops.library().ntc_op_attention_workspace(C.byref(d), backward)
    work = Inside(max(16, size), torch.uint8, 0xA5, 0)
    d.workspace = work.own.data_ptr()
    why = C.create_string_buffer(256)
    assert entry(C.byref(d), torch.cuda.current_stream().cuda_stream, why, 256) == 0, why.value
    torch.cuda.synchronize()
    assert work.untouched()


def both(rows, keys, Hq, Hk, D, dtype, sequences, causal, finite=("o", "o_rest", "dq", "dk", "dv"), **ends):
    t, code = TYPES[dtype]
    nan = float("nan")
    given = {n: Inside(m * h * D, t, nan, randn(i, m * h * D).to(t)) for i, (n, m, h) in enumerate((("q", rows, Hq), ("k", keys, Hk), ("v", keys, Hk), ("d_o", rows, Hq)))}
    made = {n: Inside(m * h * D, t, 77.0, 0.0) for n, m, h in (("o", rows, Hq), ("o_rest", rows, Hq), ("dq", rows, Hq), ("dk", keys, Hk), ("dv", keys, Hk))}
    made["lse"] = Inside(rows * Hq, torch.float32, 77.0, 0.0)
    ints = {n: torch.tensor(e, dtype=torch.int32, device="cuda") for n, e in ends.items()}
    d = ops.AttentionDesc(sequences=sequences, q_rows=rows, k_rows=keys, q_heads=Hq, k_heads=Hk, head_dim=D, dtype=code, causal=causal, scale=D ** -0.5,
                          **{n: x.own.data_ptr() for n, x in {**given, **made}.items()}, **{n: x.data_ptr() for n, x in ints.items()})
    for n, m, h in (("q", rows, Hq), ("k", keys, Hk), ("v", keys, Hk), ("do", rows, Hq)):
        setattr(d, n + "_row_stride", h * D)
        setattr(d, n + "_head_stride", D)
        setattr(d, n + "_batch_stride", m // max(1, sequences) * h * D)
    run(ops.library().ntc_op_attention, d, 0)
    run(ops.library().ntc_op_attention_backward, d, 1)
    for n, x in {**given, **made}.items():
        assert x.untouched(), n
    for n in finite:
        assert not made[n].own.isnan().any(), n


BIG = 2 ** 31 - 1
ENDS = [[0, 50, 5000], [0, -7, 100], [30, 60, 100], [0, BIG, BIG], [0, 0, 0], [BIG, BIG, BIG], [-5, -5, -5], [0, 40, 70], [0, 99, 99, 100, 99, BIG, 3]]
# (Rows of two sequences have the log sum of either: float16's probabilities may pass its range then, and where a row sees no key in one of them, causal with fewer keys than rows, it is -inf, which makes its
# probabilities in the other infinite.)
OVERLAPS = [[0, 90, 20, 100], [0, 100, 0, 100, 0, 100], [0, 64, 1, 96]]


@pytest.mark.parametrize("causal", [1, 0])
@pytest.mark.parametrize("Hq,Hk,D", [(2, 1, 32), (2, 2, 72), (4, 2, 128)])
@pytest.mark.parametrize("dtype,ends", [(t, e) for t in TYPES for e in ENDS] + [("bf16", e) for e in OVERLAPS])
@pytest.mark.parametrize("rows,keys", [(100, 100), (100, 3000), (2500, 100)])
def test_ends(rows, keys, dtype, ends, Hq, Hk, D, causal):
    finite = ("o", "o_rest") if ends in OVERLAPS and causal and rows > keys else ("o", "o_rest", "dq", "dk", "dv")
    both(rows, keys, Hq, Hk, D, dtype, len(ends) - 1, causal, finite, cu_q=[e * rows // 100 if abs(e) < BIG else e for e in ends], cu_k=[e * keys // 100 if abs(e) < BIG else e for e in ends])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", [[-5, 0], [10 ** 9, BIG], [-2 ** 31, 50], [51, 49]])
@pytest.mark.parametrize("rows,keys", [(2, 100), (200, 100), (2, 9000)])
def test_lengths(rows, keys, lens, dtype):
    both(rows, keys, 4, 2, 64, dtype, 2, 1, k_lens=lens)
    both(rows, keys, 4, 2, 64, dtype, 2, 1, k_lens=lens, cu_k=[0, keys // 3, keys])
    both(rows, keys, 4, 2, 64, dtype, 2, 1, k_lens=lens, cu_q=[0, rows // 3, rows])
