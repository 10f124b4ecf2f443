"""What the operators refuse, without a GPU: Python's checks of tensors, and the C entry points' of their descriptions (a refusal comes
before any device call); every function of include/ntc_ops.h is exported, and the mirrors have the compiled layouts."""
import ctypes as C
import os
import re

import pytest
import torch

from neural_block_textures_amd import ops as O

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def refused(fn, *args):
    why = C.create_string_buffer(256)
    rc = fn(*args, None, why, 256)
    return rc, why.value.decode()


def test_every_declared_function_is_exported():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "ntc_ops.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(ntc_op_\w+)\s*\(", text)))
    assert len(names) >= 10
    assert not [n for n in names if not hasattr(O.library(), n)]


@pytest.mark.parametrize("name,size", [("ntc_logprobs_desc", C.sizeof(O.LogprobsDesc)), ("ntc_adamw_desc", C.sizeof(O.AdamwDesc)), ("ntc_adamw_tensor", O._TENSOR.itemsize),
                                       ("ntc_fp8_quantize_desc", C.sizeof(O.QuantizeDesc)), ("ntc_fp8_matmul_desc", C.sizeof(O.MatmulDesc))])
def test_struct_layouts(name, size):
    from neural_block_textures_amd import trainer
    assert trainer.library().ntc_abi_sizeof(name.encode()) == size


def test_tensors_that_are_not_on_the_gpu():
    x, t = torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="logits must be a tensor on the GPU"):
        O.token_logprobs(x, t)
    with pytest.raises(ValueError, match="a parameter must be a tensor on the GPU"):
        O.AdamW([x])
    with pytest.raises(ValueError, match="no parameters"):
        O.AdamW([])
    with pytest.raises(ValueError, match="x must be a tensor on the GPU"):
        O.fp8_quantize(x)
    with pytest.raises(ValueError, match="x must be a tensor on the GPU"):
        O.fp8_linear(x, x)
    with pytest.raises(ValueError, match="a must be an Fp8Tensor"):
        O.fp8_matmul(x, x)


def logprobs(**kw):
    d = O.LogprobsDesc()
    d.logits = d.tokens = d.logprob = d.entropy = d.stats = d.top_ids = d.top_logprobs = d.dlogits = 1 << 20
    d.rows = d.inner_rows = 4
    d.V, d.dtype, d.token_bytes, d.temperature = 10, 1, 8, 1.0
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,reason", [
    ({"rows": -1}, "rows >= 0"), ({"V": 0}, "V >= 1"), ({"inner_rows": 0}, "inner_rows >= 1"), ({"V": 2 ** 31}, "2^31"), ({"dtype": 3}, "logits are"),
    ({"token_bytes": 2}, "tokens are"), ({"top": 33}, "top is 0 to 32"), ({"top": 11}, "at most V"), ({"top": -1}, "top is"),
    ({"temperature": 0.0}, "temperature"), ({"temperature": float("nan")}, "temperature"), ({"temperature": float("inf")}, "temperature"),
    ({"logits": None}, "null"), ({"stats": None}, "null"), ({"top": 2, "top_ids": None}, "null")])
def test_logprobs_refusals(kw, reason):
    rc, why = refused(O.library().ntc_op_token_logprobs, C.byref(logprobs(**kw)))
    assert rc == 1 and reason in why, why


def test_logprobs_backward_refusals():
    fn = O.library().ntc_op_token_logprobs_backward
    for kw in ({"dlogits": None}, {"g_top": 1 << 20, "top": 2, "top_ids": None}, {"entropy": None}):
        rc, why = refused(fn, C.byref(logprobs(**kw)))
        assert rc == 1 and "null" in why
    assert refused(O.library().ntc_op_token_logprobs, None)[0] == 1
    assert refused(O.library().ntc_op_token_logprobs, C.byref(logprobs(rows=0))) == (0, "")


@pytest.mark.parametrize("kw,reason", [
    ({"n": -1}, "tensor count"), ({"state_bits": 16}, "8 or 32 bits"), ({"beta1": 1.0}, "betas"), ({"beta2": -0.1}, "betas"), ({"lr": -1.0}, "not negative"),
    ({"eps": float("nan")}, "not negative"), ({"tensors": None}, "null"), ({"state_bits": 8}, "exponents"), ({"steps": (C.c_int32 * 1)(0)}, "count from 1"),
    ({"grad_types": (C.c_int32 * 1)(3)}, "gradients are"), ({"first_chunk": (C.c_int64 * 2)(1, 0)}, "in order")])
def test_adamw_refusals(kw, reason):
    d = O.AdamwDesc()
    held = {"first_chunk": (C.c_int64 * 2)(0, 1), "grads": (C.c_void_p * 1)(1 << 20), "grad_types": (C.c_int32 * 1)(0), "steps": (C.c_int32 * 1)(1),
            "tensors": 1 << 20, "chunk_tensor": 1 << 20, "exp_avg": 1 << 20, "exp_avg_sq": 1 << 20, "n": 1, "state_bits": 32, "beta1": 0.9, "beta2": 0.9, **kw}
    for k, v in held.items():
        setattr(d, k, C.addressof(v) if isinstance(v, C.Array) else v)
    rc, why = refused(O.library().ntc_op_adamw, C.byref(d))
    assert rc == 1 and reason in why, why


def test_adamw_state_refusals():
    lib = O.library()
    rc, why = refused(lib.ntc_op_adamw_moments, 1, 1, 1, 1, 100, 1, 1)
    assert rc == 1 and "multiple of 256" in why
    rc, why = refused(lib.ntc_op_adamw_encode, 1, 1, 256, 1, None, 1, 1)
    assert rc == 1 and "null" in why


@pytest.mark.parametrize("kw,reason", [({"R": -1}, "not negative"), ({"dtype": 3}, "x is"), ({"block_rows": 64}, "blocks are"), ({"codes": None}, "nothing to write"),
                                       ({"x": None}, "null"), ({"exps": None}, "null")])
def test_quantize_refusals(kw, reason):
    d = O.QuantizeDesc()
    for k, v in {"x": 1 << 20, "R": 4, "K": 4, "row_stride": 4, "block_rows": 1, "codes": 1 << 20, "exps": 1 << 20, **kw}.items():
        setattr(d, k, v)
    rc, why = refused(O.library().ntc_op_fp8_quantize, C.byref(d))
    assert rc == 1 and reason in why, why


def test_quantize_pair_refusals():
    d, e = O.QuantizeDesc(), O.QuantizeDesc()
    for q, rows in ((d, 1), (e, 128)):
        for k, v in {"x": 1 << 20, "R": 4, "K": 4, "row_stride": 4, "block_rows": rows, "codes": 1 << 20, "exps": 1 << 20}.items():
            setattr(q, k, v)
    call = O.library().ntc_op_fp8_quantize_pair
    for a, b, reason in ((d, d, "pair's blocks"), (e, d, "pair's blocks")):
        rc, why = refused(call, C.byref(a), C.byref(b))
        assert rc == 1 and reason in why, why
    e.exps = None
    rc, why = refused(call, C.byref(d), C.byref(e))
    assert rc == 1 and "null" in why, why


@pytest.mark.parametrize("kw,reason", [({"M": -1}, "not negative"), ({"c_type": 3}, "C is"), ({"a_block_rows": 2}, "blocks are"), ({"b_block_rows": 0}, "blocks are"),
                                       ({"ldc": 3}, "overlap"), ({"b": None}, "null"), ({"c": None}, "null"), ({"a_exps": None}, "null"), ({"a_type": 4}, "A is")])
def test_matmul_refusals(kw, reason):
    d = O.MatmulDesc()
    for k, v in {"a": 1 << 20, "a_exps": 1 << 20, "b": 1 << 20, "b_exps": 1 << 20, "c": 1 << 20, "workspace": 1 << 20, "M": 4, "N": 4, "K": 4, "ldc": 4, "a_type": 3,
                 "a_block_rows": 1, "b_block_rows": 1, **kw}.items():
        setattr(d, k, v)
    rc, why = refused(O.library().ntc_op_fp8_matmul, C.byref(d))
    assert rc == 1 and reason in why, why
