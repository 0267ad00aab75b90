"""Arguments of TokenGrammar that are no rows of states, on the CPU."""
import types

import pytest

from gpu_bpe_b200 import TokenGrammar
from tests.test_next_token_refusals import Fake


@pytest.fixture
def grammar(monkeypatch):
    g = TokenGrammar.__new__(TokenGrammar)
    g._engine, g.vocabSize, g._h, g.stateCount = types.SimpleNamespace(device_index=0), 100, None, 3      # (a call that is not refused finds no handle)
    monkeypatch.setattr(TokenGrammar, "_ready", lambda self: 0)
    return g


def test_states_without_rows(grammar):
    """One state is a tensor of one element, [1]."""
    one, row = Fake([], "int32"), Fake([1], "int32")
    for states in (one, Fake([1, 1], "int32"), [0], None, 3):
        with pytest.raises(ValueError, match="states: "):
            grammar.allowedTokens(states)
        with pytest.raises(ValueError, match="states: "):
            grammar.advance(states, one, out=one)
    with pytest.raises(ValueError, match="tokens: shape"):
        grammar.advance(row, one, out=row)
    for out in (one, [0]):
        with pytest.raises(ValueError, match="out: "):
            grammar.advance(row, row, out=out)
