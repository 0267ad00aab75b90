"""What a choice of tokens gives decodes, on the CPU: -1, no token, is an unknown id."""
import numpy as np
import pytest

from gpu_bpe_b200 import TrieTokenizer


@pytest.mark.parametrize("kind", [list, np.int32, np.int64])
def test_no_token(kind):
    t = TrieTokenizer.__new__(TrieTokenizer)
    t._vocab = [b"a", b"bc", b"d"]
    ids = [0, -1, 1, 3, -3, 2]
    assert t.decode(ids if kind is list else np.array(ids, kind)) == "a�bc��d".encode()
    assert t.decode(np.array(ids, np.int32).view(np.uint32)) == t.decode(ids)
