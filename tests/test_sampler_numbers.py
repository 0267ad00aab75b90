"""Plain numbers as settings of a TokenSampler that count something, on the CPU."""
import ctypes as C
import types

import pytest

from gpu_bpe_b200 import TokenSampler
from tests.test_next_token_refusals import Fake


@pytest.fixture
def sampler():
    s = TokenSampler.__new__(TokenSampler)
    s._engine, s.vocabSize, s._h = types.SimpleNamespace(device_index=0), 100, C.c_void_p(1)
    return s


@pytest.mark.parametrize("number", [0.9, 40.5, -0.5, float("nan"), float("inf"), 2**31, -2**31 - 1, 2.0**31])
def test_numbers_that_are_not_whole(sampler, number):
    """A setting that counts something is not rounded: a topK of 0.9 would be 0, which is all tokens."""
    rows = Fake([4])
    with pytest.raises(ValueError, match="topK: a whole number"):
        sampler.sample(Fake([4, 100]), rows, topK=number)
    history = Fake([4, 9], "int32")
    for call in (sampler.sample, sampler.adjustLogits):
        with pytest.raises(ValueError, match="lengths: a whole number"):
            call(Fake([4, 100]), history=history, lengths=number)
        with pytest.raises(ValueError, match="promptLengths: a whole number"):
            call(Fake([4, 100]), history=history, lengths=Fake([4], "int32"), promptLengths=number)
