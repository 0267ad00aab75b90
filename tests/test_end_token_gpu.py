"""The step of a grammar by an end token that is none: n_entries or more."""
import ctypes as C

import numpy as np
import pytest

from gpu_bpe_b200 import _lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("end", [2, 3, 77, 2**28, 2**32 - 2, 2**32 - 1])
def test_an_end_token_outside_the_vocabulary(engine, end):
    import torch
    L, h = _lib.lib(), C.c_void_p()
    text, off = np.frombuffer(b"ab", np.uint8), np.array([0, 1, 2], np.uint64)
    table, accepting = np.full((2, 256), 2, np.uint32), np.array([1, 1], np.uint8)
    table[0, ord("a")] = 1
    assert L.b200bpe_grammar_create(engine.ctx, text.ctypes.data, off.ctypes.data, 2, table.ctypes.data, accepting.ctypes.data, 2, end, C.byref(h)) == 0
    tokens = np.array([0, 1, 2, 3, 77, 2**28, end, 2**32 - 1], np.uint32)
    none = 0xFFFFFFFF
    want = [1] + [none] * 6 + [0]
    if end == none:
        want[6] = 0                     # (that is no token, which leaves a state as it is)
    states, t = torch.zeros(8, dtype=torch.int32, device="cuda"), torch.from_numpy(tokens.view(np.int32)).cuda()
    out = torch.full((8,), 9, dtype=torch.int32, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    assert L.b200bpe_grammar_advance(h, states.data_ptr(), t.data_ptr(), 8, out.data_ptr(), None, 0, 0, None, None, stream) == 0
    got = out.cpu().numpy().view(np.uint32).tolist()
    L.b200bpe_grammar_destroy(h)
    assert got == want
