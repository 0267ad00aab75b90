"""What TokenSampler, TokenGrammar and their C entry points refuse, and the plain model they are tested against, on the CPU."""
import ctypes as C
import types

import numpy as np
import pytest

from gpu_bpe_b200 import TokenGrammar, TokenSampler, TrieTokenizer, _lib
from tests import next_token_model as model


class Fake:
    """As much of a torch tensor as the checks look at."""

    def __init__(self, shape, dtype="float32", strides=None, device=("cuda", 0)):
        self.shape, self.dtype = tuple(shape), "torch." + dtype
        dense = [int(np.prod(shape[i + 1:])) for i in range(len(shape))]
        self._strides = tuple(strides or dense)
        self.device = types.SimpleNamespace(type=device[0], index=device[1])

    def stride(self, i=None):
        return self._strides if i is None else self._strides[i]

    @property
    def ndim(self):
        return len(self.shape)

    def size(self, i):
        return self.shape[i]

    def is_contiguous(self):
        return len(self.shape) == 1 and self._strides == (1,)

    def get_device(self):
        return self.device.index if self.device.type == "cuda" else -1

    def data_ptr(self):
        return 4096


def _sampler(vocab=100):
    s = TokenSampler.__new__(TokenSampler)
    s._engine, s.vocabSize, s._h = types.SimpleNamespace(device_index=0), vocab, C.c_void_p(1)
    return s


def _grammar(vocab=100):
    g = TokenGrammar.__new__(TokenGrammar)
    g._engine, g.vocabSize, g._h, g.stateCount = types.SimpleNamespace(device_index=0), vocab, C.c_void_p(1), 3
    g._ready = lambda: 0
    return g


ROW, IDS = Fake([4]), Fake([4], "int32")
HISTORY = dict(history=Fake([4, 9], "int32"), lengths=IDS)


@pytest.mark.parametrize("arguments, text", [
    (dict(logits=Fake([4, 99])), "99 columns"),
    (dict(logits=Fake([4, 100], "float64")), "logits: a tensor of"),
    (dict(logits=np.zeros((4, 100), np.float32)), "logits: a tensor of"),
    (dict(logits=Fake([400])), "logits: shape"),
    (dict(logits=Fake([4, 100], strides=[1, 4])), "next to one another"),
    (dict(logits=Fake([4, 100], device=("cpu", None))), "the engine is on cuda:0"),
    (dict(logits=Fake([4, 100], device=("cuda", 1))), "the engine is on cuda:0"),
    (dict(lengths=IDS), "history: needed"),
    (dict(repetition=ROW), "history: needed"),
    (dict(history=Fake([4, 9], "int32")), "lengths: needed"),
    (dict(history=Fake([4, 9], "int64"), lengths=IDS), "history: a tensor of"),
    (dict(history=Fake([3, 9], "int32"), lengths=IDS), "history: shape"),
    (dict(HISTORY, lengths=Fake([4], "int64")), "lengths: a tensor of"),
    (dict(HISTORY, lengths=Fake([5], "int32")), "lengths: shape"),
    (dict(HISTORY, promptLengths=ROW), "promptLengths: a tensor of"),
    (dict(HISTORY, presence=Fake([4, 1])), "presence: shape"),
    (dict(HISTORY, frequency=Fake([4], strides=[2])), "frequency: elements"),
    (dict(biasTokens=Fake([4, 3], "int32")), "one without the other"),
    (dict(biasTokens=Fake([4, 3], "int32"), biases=Fake([4, 2])), "biases: shape"),
    (dict(biasTokens=Fake([4, 1025], "int32"), biases=Fake([4, 1025])), "1,024"),
    (dict(biasTokens=Fake([4, 3], "int32"), biases=Fake([4, 3], strides=[4, 1])), "another distance"),
    (dict(mask=Fake([4, 3], "int32")), "mask: 3 words"),
    (dict(mask=Fake([3, 4], "int32")), "no maskRows"),
    (dict(mask=Fake([3, 4], "int32"), maskRows=Fake([3], "int32")), "maskRows: shape"),
    (dict(maskRows=IDS), "needs a mask"),
])
def test_logits_are_checked(arguments, text):
    s = _sampler()
    arguments = dict({"logits": Fake([4, 100])}, **arguments)
    with pytest.raises(ValueError, match=text):
        s.sample(**arguments)
    with pytest.raises(ValueError, match=text):
        s.adjustLogits(**arguments)


@pytest.mark.parametrize("arguments, text", [
    (dict(temperature=ROW), "uniform: needed"),
    (dict(uniform=Fake([3])), "uniform: shape"),
    (dict(uniform=ROW, topK=ROW), "topK: a tensor of"),
    (dict(uniform=ROW, topP=IDS), "topP: a tensor of"),
    (dict(uniform=ROW, minP=Fake([4], device=("cuda", 2))), "the engine is on cuda:0"),
])
def test_choice_is_checked(arguments, text):
    with pytest.raises(ValueError, match=text):
        _sampler().sample(Fake([4, 100]), **arguments)


@pytest.mark.parametrize("out, text", [
    (Fake([4, 100], "float16"), "out: a tensor of"), (Fake([4, 99]), "out: 99 columns"), (Fake([3, 100]), "out: shape"),
    (Fake([4, 100], strides=[64, 1]), "rows overlap"),
])
def test_output_is_checked(out, text):
    with pytest.raises(ValueError, match=text):
        _sampler().adjustLogits(Fake([4, 100]), out=out)


def test_grammar_calls_are_checked():
    g, states = _grammar(), Fake([4], "int32")
    for text, call in [("states: a tensor", lambda: g.allowedTokens(ROW)), ("states: shape", lambda: g.allowedTokens(Fake([4, 1], "int32"))),
                       ("out: 3 words", lambda: g.allowedTokens(states, out=Fake([4, 3], "int32"))),
                       ("rows overlap", lambda: g.allowedTokens(states, out=Fake([4, 4], "int32", strides=[3, 1]))),
                       ("tokens: shape", lambda: g.advance(states, Fake([5], "int32"))),
                       ("lengths: without", lambda: g.advance(states, states, out=states, lengths=states)),
                       ("lengths: needed", lambda: g.advance(states, states, out=states, history=Fake([4, 9], "int32"))),
                       ("rows overlap", lambda: g.advance(states, states, out=states, lengths=states, history=Fake([4, 9], "int32", strides=[8, 1]))),
                       ("out: shape", lambda: g.advance(states, states, out=Fake([3], "int32")))]:
        with pytest.raises(ValueError, match=text):
            call()


def test_a_destroyed_handle():
    s, g = _sampler(), TokenGrammar.__new__(TokenGrammar)
    s._h = g._h = None
    with pytest.raises(RuntimeError, match="destroyed"):
        s.sample(Fake([4, 100]))
    with pytest.raises(RuntimeError, match="destroyed"):
        g.allowedTokens(IDS)
    s.destroy()
    g.destroy()


def test_what_makes_no_handle():
    engine = types.SimpleNamespace(ctx=None, device_index=0)
    for n in (0, -1, 327681):
        with pytest.raises(ValueError, match="327,680"):
            TokenSampler(engine, n)
    table, ends = np.full((2, 256), -1), [0, 1]
    for arguments, text in [((table[:, :255], ends), "transitions"), ((table.astype(float), ends), "transitions"), ((table, [1]), "accepting"),
                            ((np.zeros((0, 256), int), []), "65,535"), ((np.zeros((65536, 256), np.int8), np.zeros(65536)), "65,535"),
                            ((table, ends, 3), "endToken"), ((table, ends, -1), "endToken")]:
        with pytest.raises(ValueError, match=text):
            TokenGrammar(engine, [b"a", b"b", b"c"], *arguments)
    with pytest.raises(ValueError, match="no entries"):
        TokenGrammar(engine, [], table, ends)
    assert callable(TrieTokenizer.sampler) and callable(TrieTokenizer.grammar)


def _refused(status, text):
    assert _lib.STATUS[status] == "BAD_ARG" and text in _lib.lib().b200bpe_last_error().decode(), _lib.lib().b200bpe_last_error()


def test_c_entry_points():
    """Arguments are looked at before the handles, so that a machine without a GPU can tell."""
    L, h = _lib.lib(), C.c_void_p()
    _refused(L.b200bpe_sampler_create(None, 0, C.byref(h)), "327,680")
    _refused(L.b200bpe_sampler_create(None, 327681, C.byref(h)), "327,680")
    _refused(L.b200bpe_sampler_create(None, 5, C.byref(h)), "null")
    p, c = _lib.Logits(), _lib.Choice()
    p.struct_size, c.struct_size = C.sizeof(_lib.Logits), C.sizeof(_lib.Choice)

    def both(text, **fields):
        q = _lib.Logits.from_buffer_copy(p)
        for k, v in dict({"logits": 4096, "n_rows": 1}, **fields).items():
            setattr(q, k, v)
        _refused(L.b200bpe_sampler_adjust(None, C.byref(q), 4096, 0, None), text)
        _refused(L.b200bpe_sampler_sample(None, C.byref(q), C.byref(c), None), text)
    both("struct_size", struct_size=8)
    both("unknown dtype", dtype=3)
    both("rows", n_rows=1 << 28)
    both("misaligned", logits=4098)
    both("without lengths", history=4096)
    both("without a history", lengths=4096)
    both("without a history", frequency=4096)
    both("1,024", n_bias=1025, biases=4096, bias_tokens=4096)
    both("null list", n_bias=2, biases=4096)
    both("mask_rows without", mask_rows=4096)
    both("fewer rows of the mask", mask=4096)
    for field in ("history", "repetition", "biases", "mask", "mask_rows", "lengths"):
        both("misaligned", **{field: 4098})
    c.tokens_out = c.logprobs_out = 4096
    both("null handle")
    off, table = np.array([0, 1, 3], np.uint64), np.zeros((2, 256), np.uint32)
    ends, text = np.zeros(2, np.uint8), np.zeros(3, np.uint8)
    make = lambda off=off, n=2, states=2, blob=text.ctypes.data: L.b200bpe_grammar_create(  # noqa: E731
        None, blob, off.ctypes.data, n, table.ctypes.data, ends.ctypes.data, states, 0, C.byref(h))
    _refused(make(states=0), "states")
    _refused(make(states=65536), "states")
    _refused(make(n=0), "entries")
    _refused(make(off=np.array([1, 1, 3], np.uint64)), "begin at 0")
    _refused(make(off=np.array([0, 3, 1], np.uint64)), "fall")
    _refused(make(blob=None), "null bytes")
    _refused(make(), "null context")
    _refused(L.b200bpe_grammar_mask(None, None, 1, None, 0, None), "null handle")
    _refused(L.b200bpe_grammar_advance(None, None, None, 1, None, None, 0, 0, None, None, None), "null handle")
    L.b200bpe_sampler_destroy(None)
    L.b200bpe_grammar_destroy(None)


def test_the_model_by_hand():
    x = np.log(np.array([1.0, 4.0, 2.0, 1.0]))
    assert [model.choice(x, u)[0] for u in (0, 0.12, 0.13, 0.6, 0.63, 0.87, 0.88, 1)] == [0, 0, 1, 1, 2, 2, 3, 3]
    assert model.choice(x)[0] == 1 and abs(model.choice(x)[1] - np.log(0.5)) < 1e-15
    assert [model.choice(x, 0.999, k=k)[0] for k in (1, 2, 3, 4, 9)] == [1, 2, 2, 3, 3]
    assert [model.choice(x, 0.0, k=k)[0] for k in (1, 2, 3, 4)] == [1, 1, 0, 0]
    assert [model.choice(x, 0.999, p=p)[0] for p in (0.0, 0.4, 0.6, 0.8, 0.9)] == [1, 1, 2, 2, 3]
    assert model.choice(x, 0.999, m=0.4)[0] == 2 and model.choice(x, 0.0, m=0.4)[0] == 1
    assert model.choice(np.full(3, -np.inf), 0.5)[:2] == (-1, -np.inf) and model.choice(np.array([np.nan, 1.0]), 0.5)[0] == 1
    x, _ = model.adjusted(np.array([[2.0, -2.0, 1.0]]), np.float64, np.array([[0, 1, 1, 7, -1]]), [5], [1], [2.0], [0.5], [0.25], np.array([[2, 2]]),
                          np.array([[1.0, 3.0]]), model.packed([[1, 1, 0]]))
    assert x.tolist() == [[1.0, -5.0, -np.inf]]
    table, ends = model.literals([b"ab", b"abc"])
    assert model.allowed([b"a", b"abc", b"b", b"", b"x", b"e"], table, ends, 5, 0).tolist() == [True, True, False, False, False, False]
    assert model.allowed([b"c", b"cc", b"e"], table, ends, 2, 2).tolist() == [True, False, True]


def test_packed_structures():
    """What the calls pack is what the header's structures are."""
    for packed, of in ((_lib.PACKED_LOGITS, _lib.Logits), (_lib.PACKED_CHOICE, _lib.Choice)):
        assert packed.size == C.sizeof(of)
        values = list(range(1, len(of._fields_) + 1))
        got = of.from_buffer_copy(packed.pack(*values))
        assert [getattr(got, name) for name, _ in of._fields_] == values
