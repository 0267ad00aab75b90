"""TokenGrammar — the tokens of a vocabulary that a byte automaton allows, and its step behind a token, on a B200.

No counterpart in the reference.  The masks are those that TokenSampler takes.  As there, tensors are torch's on the engine's
GPU, and the work is enqueued on torch's current stream.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib
from .token_sampler import IDS, _refuse, raw_stream, row_of, table_of


class TokenGrammar:
    def __init__(self, engine, vocab, transitions, accepting, endToken: int | None = None):
        """transitions [states, 256] of whole numbers: the state behind a byte; what is no state (-1, say) means that the byte is not allowed.
        accepting [states]: whether a text may end there, with endToken.  The vocabulary is taken as it is now."""
        self._engine, self._h = engine, None
        table, ends = np.asarray(transitions), np.asarray(accepting)
        if table.ndim != 2 or table.shape[1] != 256 or table.dtype.kind not in "iu":
            raise ValueError("transitions: whole numbers of shape [states, 256]")
        if not 1 <= table.shape[0] <= 65535:
            raise ValueError("transitions: 1 to 65,535 states")
        if ends.shape != (table.shape[0],):
            raise ValueError("accepting: one value a state")
        entries = vocab if isinstance(vocab, list) and set(map(type, vocab)) == {bytes} else [bytes(e) for e in vocab]
        if not entries:
            raise ValueError("vocab: no entries")
        if endToken is not None and not 0 <= endToken < len(entries):
            raise ValueError("endToken: outside the vocabulary")
        self.stateCount, self.vocabSize = table.shape[0], len(entries)
        table = np.where((table >= 0) & (table < table.shape[0]), table, 0xFFFFFFFF).astype(np.uint32)
        ends = np.ascontiguousarray(ends != 0).astype(np.uint8)
        blob = np.frombuffer(b"".join(entries) or b"\0", np.uint8)
        off = np.zeros(len(entries) + 1, np.uint64)
        np.cumsum(np.fromiter(map(len, entries), np.uint64, len(entries)), out=off[1:])
        h = C.c_void_p()
        _lib.check(_lib.lib().b200bpe_grammar_create(engine.ctx, blob.ctypes.data, off.ctypes.data, len(entries), table.ctypes.data, ends.ctypes.data,
                                                     self.stateCount, 0xFFFFFFFF if endToken is None else endToken, C.byref(h)), "b200bpe_grammar_create")
        self._h = h

    def _ready(self):
        if self._h is None:
            raise RuntimeError("TokenGrammar is destroyed")
        return raw_stream(self._engine.device_index)

    def allowedTokens(self, states, out=None):
        """states [rows] → mask int32 [rows, (vocabSize + 31) // 32] (or `out`, at least as wide): the tokens with bytes, all of which the automaton
        takes from the row's state, and the end token in an accepting state.  A state that is none (-1) allows nothing."""
        stream, at = self._ready(), self._engine.device_index
        shape, words = getattr(states, "shape", ())[:1], (self.vocabSize + 31) >> 5
        if not shape:
            _refuse(states, "states", at, IDS, (None,))
        address = row_of(states, "states", at, IDS, shape)
        rows = shape[0]
        if out is None:
            import torch
            out = states.new_empty((rows, words), dtype=torch.int32)
            p_out, stride = out.data_ptr(), words
        else:
            p_out, stride, columns = table_of(out, "out", at, IDS, rows)
            if columns < words:
                raise ValueError(f"out: {columns} words, the vocabulary needs {words}")
            if rows > 1 and stride < words:
                raise ValueError("out: rows overlap")
        status = _lib.lib().b200bpe_grammar_mask(self._h, address, rows, p_out, stride, stream)
        if status:
            _lib.check(status, "b200bpe_grammar_mask")
        return out

    def advance(self, states, tokens, history=None, lengths=None, out=None, lengthsOut=None):
        """The states behind tokens [rows] → states int32 [rows] (or `out`, which may be states): -1 where the automaton does not take the token's
        bytes; the end token leaves an accepting state as it is, and no token (-1) any state.

        With history [rows, room] and lengths: tokens are also written behind each row's history, and → (states, new lengths) (or
        `lengthsOut`, which may be lengths).  No token, and a full row, changes neither."""
        stream, at = self._ready(), self._engine.device_index
        shape = getattr(states, "shape", ())[:1]
        if not shape:
            _refuse(states, "states", at, IDS, (None,))
        rows = shape[0]
        p_states, p_tokens = row_of(states, "states", at, IDS, shape), row_of(tokens, "tokens", at, IDS, shape)
        if out is None:
            import torch
            out = states.new_empty(rows, dtype=torch.int32)
            p_out = out.data_ptr()
        else:
            p_out = row_of(out, "out", at, IDS, shape)
        p_history = p_lengths = p_new = None
        stride = room = 0
        if history is not None:
            if lengths is None:
                raise ValueError("lengths: needed with a history")
            p_lengths = row_of(lengths, "lengths", at, IDS, shape)
            p_history, stride, room = table_of(history, "history", at, IDS, rows)
            if rows > 1 and stride < room:
                raise ValueError("history: rows overlap")
            if lengthsOut is None:
                import torch
                lengthsOut = lengths.new_empty(rows, dtype=torch.int32)
                p_new = lengthsOut.data_ptr()
            else:
                p_new = row_of(lengthsOut, "lengthsOut", at, IDS, shape)
            if rows and not room:             # (an empty tensor has no address)
                p_history = p_lengths
        elif lengths is not None or lengthsOut is not None:
            raise ValueError("lengths: without a history")
        status = _lib.lib().b200bpe_grammar_advance(self._h, p_states, p_tokens, rows, p_out, p_history, stride, room, p_lengths, p_new, stream)
        if status:
            _lib.check(status, "b200bpe_grammar_advance")
        return out if history is None else (out, lengthsOut)

    def destroy(self):
        if self._h is not None:
            _lib.lib().b200bpe_grammar_destroy(self._h)
            self._h = None
