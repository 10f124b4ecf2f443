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
