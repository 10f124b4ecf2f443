"""The ends of what the operators' C entry points take, without a GPU."""
import ctypes as C

import pytest

from neural_block_textures_amd import ops as O
from tests.test_ops_refusals import logprobs, refused


@pytest.mark.parametrize("T", [2.0 ** -128, 1e-44, 2.0 ** 121, 3e38, -1.0])
def test_temperatures_out_of_range(T):
    rc, why = refused(O.library().ntc_op_token_logprobs, C.byref(logprobs(temperature=T)))
    assert rc == 1 and "temperature is from" in why, why


@pytest.mark.parametrize("T", [2.0 ** -127, 1.0, 2.0 ** 120])
def test_temperatures_in_range(T):
    assert refused(O.library().ntc_op_token_logprobs, C.byref(logprobs(temperature=T, rows=0))) == (0, "")


def test_a_step_of_tensors_without_values():
    d = O.AdamwDesc()
    held = {"first_chunk": (C.c_int64 * 3)(0, 0, 0), "grads": (C.c_void_p * 2)(1 << 20, None), "grad_types": (C.c_int32 * 2)(0, 0), "steps": (C.c_int32 * 2)(1, 1)}
    for k, v in held.items():
        setattr(d, k, C.addressof(v))
    d.n, d.state_bits, d.beta1, d.beta2 = 2, 8, 0.9, 0.9
    assert refused(O.library().ntc_op_adamw, C.byref(d)) == (0, "")
