"""TokenSampler — from a model's logits over a vocabulary to the next token of every request, on a B200.

No counterpart in the reference, whose tokens end in decode.  Inputs and outputs are torch tensors on the engine's GPU; the
work is enqueued on torch's current stream and nothing is waited for, so calls can be captured into CUDA graphs.
Token ids are int32 (or uint32), as encodeBatchDevice leaves them; -1 stands for no token.  Results carry no gradients.
"""
from __future__ import annotations

import ctypes as C

from . import _lib

# Types by name; a dtype object joins its name when it is met first (its name takes as long to make as the rest of a check).
LOGITS = {"torch.float32": 0, "torch.float16": 1, "torch.bfloat16": 2}
IDS = {"torch.int32": 0, "torch.uint32": 0}
FLOATS = {"torch.float32": 0}
MAX_VOCAB, MAX_BIASES = 327680, 1024


def _refuse(t, name, index, kinds, shape):
    """What is wrong with a tensor that row_of or table_of did not take at sight; nothing, if it is its type's first."""
    kind = getattr(t, "dtype", None)
    if kind not in kinds:
        if str(kind) not in kinds:
            raise ValueError(f"{name}: a tensor of {' or '.join(k for k in kinds if isinstance(k, str))} is needed")
        kinds[kind] = kinds[str(kind)]
    if len(t.shape) != len(shape) or any(want is not None and want != got for want, got in zip(shape, t.shape)):
        raise ValueError(f"{name}: shape {tuple(t.shape)} where {tuple(shape)} is needed")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}: elements of a row must lie next to one another")
    if t.get_device() != index:
        raise ValueError(f"{name}: on {t.device}, the engine is on cuda:{index}")


def row_of(t, name, index, kinds, shape):
    """Address of a dense tensor of this shape, (rows,), of one of these types on GPU `index`."""
    try:
        if t.dtype in kinds and t.shape == shape and t.get_device() == index and t.is_contiguous():
            return t.data_ptr()
    except AttributeError:
        pass
    _refuse(t, name, index, kinds, shape)
    return t.data_ptr()


def table_of(t, name, index, kinds, rows):
    """Address, distance between rows, and columns of a tensor [rows (None: any number), any number]; its rows may be at any distance."""
    try:
        if t.dtype in kinds and t.get_device() == index:
            shape, strides = t.shape, t.stride()
            if len(shape) == 2 and strides[1] == 1 and (rows is None or shape[0] == rows):
                return t.data_ptr(), strides[0], shape[1]
    except AttributeError:
        pass
    _refuse(t, name, index, kinds, (rows, None))
    return t.data_ptr(), t.stride(0), t.shape[1]


_stream_of = None


def raw_stream(index):
    """Torch's current stream on GPU `index`, as a number."""
    global _stream_of
    if _stream_of is None:
        import torch
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)       # (a tenth of a microsecond; the stream as an object takes two)
        _stream_of = raw or (lambda i: torch.cuda.current_stream(i).cuda_stream)
    return _stream_of(index)


class TokenSampler:
    def __init__(self, engine, vocabSize: int):
        self._engine, self.vocabSize = engine, int(vocabSize)
        self._h = None
        if not 1 <= self.vocabSize <= MAX_VOCAB:
            raise ValueError(f"vocabSize: 1 to {MAX_VOCAB:,} tokens")
        h = C.c_void_p()
        _lib.check(_lib.lib().b200bpe_sampler_create(engine.ctx, self.vocabSize, C.byref(h)), "b200bpe_sampler_create")
        self._h = h

    def _row(self, keep, value, name, shape, kinds):
        """Address of one value a row; None has none (0), a plain number stands for all rows."""
        if value is None:
            return 0
        index = self._engine.device_index
        if isinstance(value, (int, float)):
            import torch
            if kinds is IDS and not (-2**31 <= value < 2**31 and value == int(value)):
                raise ValueError(f"{name}: a whole number of 32 bits is needed")
            value = torch.full(shape, value, dtype=torch.int32 if kinds is IDS else torch.float32, device=f"cuda:{index}")
            keep.append(value)
        return row_of(value, name, index, kinds, shape)

    def _logits(self, keep, logits, history, lengths, promptLengths, repetition, presence, frequency, biasTokens, biases, mask, maskRows):
        if self._h is None:
            raise RuntimeError("TokenSampler is destroyed")
        at = self._engine.device_index
        p_logits, row_stride, columns = table_of(logits, "logits", at, LOGITS, None)
        shape = logits.shape[:1]
        rows = shape[0]
        if columns < self.vocabSize:
            raise ValueError(f"logits: {columns} columns, the vocabulary has {self.vocabSize} tokens")
        p_history = p_lengths = p_prompt = p_rep = p_pres = p_freq = p_ids = p_biases = p_mask = p_which = 0
        history_stride = room = n_bias = bias_stride = mask_stride = mask_rows = 0
        if history is not None:
            if lengths is None:
                raise ValueError("lengths: needed with a history")
            p_history, history_stride, room = table_of(history, "history", at, IDS, rows)
            p_lengths = self._row(keep, lengths, "lengths", shape, IDS)
            p_prompt = self._row(keep, promptLengths, "promptLengths", shape, IDS)
            p_rep = self._row(keep, repetition, "repetition", shape, FLOATS)
            p_pres = self._row(keep, presence, "presence", shape, FLOATS)
            p_freq = self._row(keep, frequency, "frequency", shape, FLOATS)
            if not room:
                p_history = p_lengths = p_prompt = p_rep = p_pres = p_freq = 0
        elif not (lengths is None and promptLengths is None and repetition is None and presence is None and frequency is None):
            raise ValueError("history: needed for lengths and penalties")
        if biasTokens is not None or biases is not None:
            if biasTokens is None or biases is None:
                raise ValueError("biasTokens and biases: one without the other")
            p_ids, bias_stride, n_bias = table_of(biasTokens, "biasTokens", at, IDS, rows)
            if n_bias > MAX_BIASES:
                raise ValueError(f"biasTokens: at most {MAX_BIASES:,} a row")
            p_biases, other, n = table_of(biases, "biases", at, FLOATS, rows)
            if n != n_bias:
                raise ValueError(f"biases: shape {tuple(biases.shape)} where {(rows, n_bias)} is needed")
            if other != bias_stride and rows > 1 and n_bias:
                raise ValueError("biases: another distance between rows than biasTokens")
        if mask is not None:
            p_mask, mask_stride, words = table_of(mask, "mask", at, IDS, None)
            mask_rows = mask.shape[0]
            if words < (self.vocabSize + 31) >> 5:
                raise ValueError(f"mask: {words} words, the vocabulary needs {(self.vocabSize + 31) // 32}")
            if maskRows is not None:
                p_which = row_of(maskRows, "maskRows", at, IDS, shape)
                if rows and not mask_rows:
                    raise ValueError("mask: no rows")
            elif mask_rows != rows:
                raise ValueError(f"mask: {mask_rows} rows for {rows} rows of logits, and no maskRows")
        elif maskRows is not None:
            raise ValueError("maskRows: needs a mask")
        return rows, _lib.PACKED_LOGITS.pack(LOGITS_BYTES, LOGITS[logits.dtype], rows, n_bias, p_logits, row_stride, p_history, history_stride, p_lengths,
                                             p_prompt, room, mask_rows, p_rep, p_pres, p_freq, p_ids, p_biases, bias_stride, p_mask, mask_stride, p_which)

    def adjustLogits(self, logits, out=None, history=None, lengths=None, promptLengths=None, repetition=None, presence=None, frequency=None,
                     biasTokens=None, biases=None, mask=None, maskRows=None):
        """Penalties for tokens of the history, biases and masks on logits [rows, at least vocabSize] (float32, float16 or bfloat16), in `out`
        (may be logits; of the same type; columns behind the vocabulary are left as they are) or a new tensor [rows, vocabSize].

        history [rows, room] holds each row's tokens so far, lengths says how many, promptLengths how many of them were given (they count for
        repetition, not for presence and frequency).  repetition, presence, frequency: one number a row, or one for all (which makes a tensor, a kernel
        of its own, in every call: a loop keeps tensors).
        biasTokens, biases [rows, n]: ids (-1: unused place) and what is added.  mask [rows, words]: bit v & 31 of word v >> 5 allows token v, as
        TokenGrammar.allowedTokens makes them; with maskRows, row maskRows[r] of it is row r's, and none allows anything."""
        keep = []
        rows, p = self._logits(keep, logits, history, lengths, promptLengths, repetition, presence, frequency, biasTokens, biases, mask, maskRows)
        if out is None:
            out = logits.new_empty((rows, self.vocabSize))
        address, stride, columns = table_of(out, "out", self._engine.device_index, LOGITS, rows)
        if out.dtype != logits.dtype:
            raise ValueError(f"out: a tensor of {logits.dtype} is needed")
        if columns < self.vocabSize:
            raise ValueError(f"out: {columns} columns, the vocabulary has {self.vocabSize} tokens")
        if stride < self.vocabSize and rows > 1:
            raise ValueError("out: rows overlap")
        status = _lib.lib().b200bpe_sampler_adjust(self._h, p, address, stride, raw_stream(self._engine.device_index))
        if status:
            _lib.check(status, "b200bpe_sampler_adjust")
        return out

    def sample(self, logits, uniform=None, temperature=None, topK=None, topP=None, minP=None, history=None, lengths=None, promptLengths=None,
               repetition=None, presence=None, frequency=None, biasTokens=None, biases=None, mask=None, maskRows=None):
        """→ (tokens int32 [rows], logprobs float32 [rows]): adjustLogits and the choice of a token in one kernel.

        Without uniform every row takes its largest adjusted logit.  With uniform [rows] in [0, 1): of the topK largest (0: all), of those the shortest
        run from the largest on that has topP of their weight exp(x / temperature), of those the ones with at least minP times the largest weight,
        the first in order of ids at which the running sum of weights is above uniform times their sum.  temperature below
        2^-16: the largest.  Each but uniform is one number a row, or one for all, as in adjustLogits.  logprobs are under the weights of all allowed tokens (at temperature 1
        where the largest is taken).  A row without an allowed token gives -1 and -inf (TrieTokenizer.decode counts
        negative ids from the vocabulary's end: it is not given a -1); a NaN is never chosen."""
        keep = []
        rows, p = self._logits(keep, logits, history, lengths, promptLengths, repetition, presence, frequency, biasTokens, biases, mask, maskRows)
        shape = logits.shape[:1]
        p_uniform = p_warm = p_k = p_p = p_m = 0
        if uniform is not None:
            p_uniform = row_of(uniform, "uniform", self._engine.device_index, FLOATS, shape)
            p_warm = self._row(keep, temperature, "temperature", shape, FLOATS)
            p_k = self._row(keep, topK, "topK", shape, IDS)
            p_p = self._row(keep, topP, "topP", shape, FLOATS)
            p_m = self._row(keep, minP, "minP", shape, FLOATS)
        elif not (temperature is None and topK is None and topP is None and minP is None):
            raise ValueError("uniform: needed to draw")
        import torch
        tokens, logprobs = logits.new_empty(rows, dtype=torch.int32), logits.new_empty(rows, dtype=torch.float32)
        c = _lib.PACKED_CHOICE.pack(CHOICE_BYTES, 0, p_uniform, p_warm, p_k, p_p, p_m, tokens.data_ptr(), logprobs.data_ptr())
        status = _lib.lib().b200bpe_sampler_sample(self._h, p, c, raw_stream(self._engine.device_index))
        if status:
            _lib.check(status, "b200bpe_sampler_sample")
        return tokens, logprobs

    def destroy(self):
        if self._h is not None:
            _lib.lib().b200bpe_sampler_destroy(self._h)
            self._h = None


LOGITS_BYTES, CHOICE_BYTES = C.sizeof(_lib.Logits), C.sizeof(_lib.Choice)
