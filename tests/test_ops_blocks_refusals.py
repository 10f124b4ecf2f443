"""What layer_norm, rotary and attention refuse, without a GPU: Python's checks of tensors, and the C entry points' of their descriptions (a refusal comes before any
device call); the mirrors have the compiled layouts."""
import ctypes as C

import pytest
import torch

from neural_block_textures_amd import ops as O

AT = 1 << 20


def refused(fn, d):
    why = C.create_string_buffer(256)
    rc = fn(C.byref(d) if d is not None else None, None, why, 256)
    return rc, why.value.decode()


@pytest.mark.parametrize("name,size", [("ntc_layer_norm_desc", C.sizeof(O.LayerNormDesc)), ("ntc_rotary_desc", C.sizeof(O.RotaryDesc)), ("ntc_attention_desc", C.sizeof(O.AttentionDesc))])
def test_struct_layouts(name, size):
    from neural_block_textures_amd import trainer
    assert trainer.library().ntc_abi_sizeof(name.encode()) == size


def test_tensors_that_are_not_on_the_gpu():
    x = torch.zeros(2, 4, 8, dtype=torch.float16)
    with pytest.raises(ValueError, match="x must be a tensor on the GPU"):
        O.layer_norm(x)
    with pytest.raises(ValueError, match="positions must be a tensor on the GPU"):
        O.rotary(torch.zeros(2, 1, dtype=torch.int64), x, sections=(4,))
    with pytest.raises(ValueError, match="q must be a tensor on the GPU"):
        O.attention(x, x, x)


def norm(**kw):
    d = O.LayerNormDesc()
    d.x = d.y = d.stats = d.dy = d.dx = d.dweight = d.workspace = AT
    d.rows, d.C, d.x_stride, d.dy_stride, d.dtype, d.weight_type, d.eps = 4, 8, 8, 8, 1, 1, 1e-5
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,reason", [({"rows": -1}, "rows >= 0"), ({"C": 0}, "1 <= C"), ({"C": 2 ** 30}, "2^30"), ({"dtype": 3}, "values are"), ({"weight_type": 2}, "of the values' type"),
                                       ({"eps": -1.0}, "eps"), ({"eps": float("nan")}, "eps"), ({"eps": float("inf")}, "eps"), ({"x": None}, "null pointer"), ({"stats": AT + 4}, "multiple of 8")])
def test_layer_norm_refusals(kw, reason):
    for fn in (O.library().ntc_op_layer_norm, O.library().ntc_op_layer_norm_backward):
        rc, why = refused(fn, norm(**kw))
        assert rc == 1 and reason in why, why


def test_layer_norm_pointers():
    lib = O.library()
    assert refused(lib.ntc_op_layer_norm, norm(y=None)) == (1, "null pointer")
    assert refused(lib.ntc_op_layer_norm_backward, norm(stats=None)) == (1, "null pointer")
    assert refused(lib.ntc_op_layer_norm_backward, norm(workspace=None)) == (1, "null workspace")
    assert refused(lib.ntc_op_layer_norm, None)[0] == 1
    assert refused(lib.ntc_op_layer_norm, norm(rows=0)) == (0, "")
    assert refused(lib.ntc_op_layer_norm_backward, norm(rows=0, dweight=None)) == (0, "")


def rotary(sections=(4,), **kw):
    d = O.RotaryDesc()
    d.positions = AT
    for t in range(2):
        d.x[t] = d.y[t] = AT
        d.heads[t], d.token_stride[t], d.head_stride[t] = 2, 32, 16
    d.position_stride, d.tokens, d.head_dim, d.axes, d.position_bytes, d.dtype, d.base = 1, 3, 16, len(sections), 8, 1, 10000.0
    for a, n in enumerate(sections):
        d.sections[a] = n
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("sections,kw,reason", [((4,), {"tokens": -1}, "tokens and heads"), ((4,), {"head_dim": 15}, "even number"), ((4,), {"head_dim": 0}, "even number"), ((4,), {"axes": 0}, "1 to 8 axes"),
                                                ((4,), {"axes": 9}, "1 to 8 axes"), ((9,), {}, "pairs"), ((0,), {}, "pairs"), ((-1, 3), {}, "0 pairs or more"), ((64, 65), {"head_dim": 512}, "128 pairs"),
                                                ((4,), {"base": 0.9}, "base"), ((4,), {"base": float("nan")}, "base"), ((4,), {"base": float("inf")}, "base"), ((4,), {"dtype": 3}, "values are"),
                                                ((4,), {"position_bytes": 2}, "4 or 8"), ((4,), {"heads": (1 << 14, 1), "head_dim": 1 << 14}, "2^28 elements"), ((4,), {"positions": None}, "null")])
def test_rotary_refusals(sections, kw, reason):
    rc, why = refused(O.library().ntc_op_rotary, rotary(sections, **kw))
    assert rc == 1 and reason in why, why


def test_rotary_pointers():
    fn = O.library().ntc_op_rotary
    d = rotary()
    d.x[1] = None
    assert refused(fn, d) == (1, "null pointer")
    d = rotary(tokens=0)
    d.x[1] = None
    assert refused(fn, d) == (0, "") and refused(fn, None)[0] == 1


def attention(**kw):
    d = O.AttentionDesc()
    for n in ("q", "k", "v", "o", "o_rest", "lse", "d_o", "dq", "dk", "dv", "workspace"):
        setattr(d, n, AT)
    d.sequences, d.q_rows, d.k_rows, d.q_heads, d.k_heads, d.head_dim, d.dtype, d.causal, d.scale = 2, 8, 8, 4, 2, 16, 1, 1, 0.25
    for n in ("q", "k", "v", "do"):
        setattr(d, n + "_row_stride", 64)
        setattr(d, n + "_head_stride", 16)
        setattr(d, n + "_batch_stride", 256)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,reason", [({"sequences": -1}, "from 0 on"), ({"q_rows": -1}, "from 0 on"), ({"sequences": 2 ** 30}, "2^30 sequences"), ({"dtype": 0}, "bfloat16 or float16"), ({"head_dim": 12}, "multiple of 8"), ({"head_dim": 136}, "up to 128"),
                                       ({"head_dim": 0}, "multiple of 8"), ({"k_heads": 3}, "times the key heads"), ({"k_heads": 0}, "times the key heads"), ({"q_heads": 65536 + 2}, "at most 65536"), ({"q_heads": 4096}, "1 to 1024"), ({"scale": 0.0}, "scale"),
                                       ({"scale": -1.0}, "scale"), ({"scale": float("nan")}, "scale"), ({"scale": float("inf")}, "scale"), ({"q_rows": 2 ** 29}, "2^30"), ({"k_rows": 2 ** 30}, "2^30"), ({"q_rows": 9}, "as many queries"),
                                       ({"k_rows": 9}, "as many keys"), ({"sequences": 0}, "without a sequence"), ({"q_row_stride": 60}, "multiples of 8"), ({"k_head_stride": -8}, "multiples of 8"), ({"v_row_stride": 2 ** 22 + 8}, "at most 2^22"),
                                       ({"q_head_stride": 2 ** 20 + 8}, "2^20"), ({"k_batch_stride": 4}, "multiples of 8"), ({"q": None}, "null pointer"), ({"o": None}, "null pointer"), ({"v": None}, "null pointer"), ({"k": AT + 8}, "multiple of 16")])
def test_attention_refusals(kw, reason):
    for fn in (O.library().ntc_op_attention, O.library().ntc_op_attention_backward):
        rc, why = refused(fn, attention(**kw))
        assert rc == 1 and reason in why, why


def test_attention_backward_refusals():
    fn = O.library().ntc_op_attention_backward
    for kw, reason in (({"d_o": None}, "null"), ({"lse": None}, "null"), ({"o_rest": None}, "null"), ({"workspace": None}, "null"), ({"do_row_stride": 4}, "multiples of 8"), ({"do_head_stride": 2 ** 20 + 8}, "2^20"), ({"dq": AT + 2}, "multiple of 16")):
        rc, why = refused(fn, attention(**kw))
        assert rc == 1 and reason in why, why
    assert refused(fn, attention(q_rows=0, k_rows=0)) == (0, "") and refused(O.library().ntc_op_attention, attention(q_rows=0)) == (0, "")
    assert refused(fn, None)[0] == 1 and refused(O.library().ntc_op_attention, None)[0] == 1
