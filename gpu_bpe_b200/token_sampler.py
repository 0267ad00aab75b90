"""TokenSampler — from a model's logits over a vocabulary to the next token of every request, on a B200.

No counterpart in the reference, whose tokens end in decode.  Inputs and outputs are torch tensors on the engine's GPU; the
work is enqueued on torch's current stream and nothing is waited for, so calls can be captured into CUDA graphs.
Token ids are int32 (or uint32), as encodeBatchDevice leaves them; -1 stands for no token.
"""
from __future__ import annotations

import ctypes as C

from . import _lib

DTYPES = {"torch.float32": 0, "torch.float16": 1, "torch.bfloat16": 2}
IDS, FLOATS = ("torch.int32", "torch.uint32"), ("torch.float32",)


def device_of(t, name, index, kinds, shape):
    """Refuses a tensor that is not of these types and this shape (None: any size), dense within its rows, on GPU `index`; its address."""
    if str(getattr(t, "dtype", None)) not in kinds:
        raise ValueError(f"{name}: a tensor of {' or '.join(kinds)} is needed")
    if len(t.shape) != len(shape) or any(want is not None and want != got for want, got in zip(shape, t.shape)):
        raise ValueError(f"{name}: shape {tuple(t.shape)} where {tuple(shape)} is needed")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}: elements of a row must lie next to one another")
    if t.device.type != "cuda" or t.device.index != index:
        raise ValueError(f"{name}: on {t.device}, the engine is on cuda:{index}")
    return t.data_ptr()


class TokenSampler:
    def __init__(self, engine, vocabSize: int):
        self._engine, self.vocabSize = engine, int(vocabSize)
        self._h = None
        if not 1 <= self.vocabSize <= 327680:
            raise ValueError("vocabSize: 1 to 327,680 tokens")
        h = C.c_void_p()
        _lib.check(_lib.lib().b200bpe_sampler_create(engine.ctx, self.vocabSize, C.byref(h)), "b200bpe_sampler_create")
        self._h = h

    def _row(self, value, name, rows, kinds, like):
        """Address of one value a row; a plain number stands for all rows (the tensor that holds it is returned, too)."""
        if isinstance(value, (int, float)):
            import torch
            value = torch.full((rows,), value, dtype=torch.int32 if kinds is IDS else torch.float32, device=like.device)
        return device_of(value, name, self._engine.device_index, kinds, (rows,)), value

    def _logits(self, keep, logits, history, lengths, promptLengths, repetition, presence, frequency, biasTokens, biases, mask, maskRows):
        if self._h is None:
            raise RuntimeError("TokenSampler is destroyed")
        at = self._engine.device_index
        p = _lib.Logits()
        p.struct_size = C.sizeof(_lib.Logits)
        p.logits = device_of(logits, "logits", at, DTYPES, (None, None))
        rows = logits.shape[0]
        if logits.shape[1] < self.vocabSize:
            raise ValueError(f"logits: {logits.shape[1]} columns, the vocabulary has {self.vocabSize} tokens")
        p.dtype, p.n_rows, p.row_stride = DTYPES[str(logits.dtype)], rows, logits.stride(0)
        if history is not None:
            if lengths is None:
                raise ValueError("lengths: needed with a history")
            p.history = device_of(history, "history", at, IDS, (rows, None))
            p.history_stride, p.history_cap = history.stride(0), history.shape[1]
            for field, value, name, kinds in (("lengths", lengths, "lengths", IDS), ("prompt_lengths", promptLengths, "promptLengths", IDS),
                                              ("repetition", repetition, "repetition", FLOATS), ("presence", presence, "presence", FLOATS),
                                              ("frequency", frequency, "frequency", FLOATS)):
                if value is not None:
                    address, tensor = self._row(value, name, rows, kinds, logits)
                    setattr(p, field, address)
                    keep.append(tensor)
            if not history.shape[1]:
                p.history = p.lengths = p.prompt_lengths = p.repetition = p.presence = p.frequency = None
        elif any(x is not None for x in (lengths, promptLengths, repetition, presence, frequency)):
            raise ValueError("history: needed for lengths and penalties")
        if (biasTokens is None) != (biases is None):
            raise ValueError("biasTokens and biases: one without the other")
        if biasTokens is not None:
            p.n_bias = biasTokens.shape[-1] if len(biasTokens.shape) == 2 else 0
            if p.n_bias > 1024:
                raise ValueError("biasTokens: at most 1,024 a row")
            p.bias_tokens = device_of(biasTokens, "biasTokens", at, IDS, (rows, None))
            p.biases = device_of(biases, "biases", at, FLOATS, (rows, p.n_bias))
            p.bias_stride = biasTokens.stride(0)
            if biases.stride(0) != biasTokens.stride(0) and rows > 1 and p.n_bias:
                raise ValueError("biases: another distance between rows than biasTokens")
        if mask is not None:
            p.mask = device_of(mask, "mask", at, IDS, (None, None))
            p.n_mask_rows, p.mask_stride = mask.shape[0], mask.stride(0)
            if mask.shape[1] < (self.vocabSize + 31) // 32:
                raise ValueError(f"mask: {mask.shape[1]} words, the vocabulary needs {(self.vocabSize + 31) // 32}")
            if maskRows is not None:
                p.mask_rows = device_of(maskRows, "maskRows", at, IDS, (rows,))
            elif mask.shape[0] != rows:
                raise ValueError(f"mask: {mask.shape[0]} rows for {rows} rows of logits, and no maskRows")
        elif maskRows is not None:
            raise ValueError("maskRows: needs a mask")
        return p

    def _stream(self):
        import torch
        return torch.cuda.current_stream(self._engine.device_index).cuda_stream

    def adjustLogits(self, logits, out=None, history=None, lengths=None, promptLengths=None, repetition=None, presence=None, frequency=None,
                     biasTokens=None, biases=None, mask=None, maskRows=None):
        """Penalties for tokens of the history, biases and masks on logits [rows, at least vocabSize] (float32, float16 or bfloat16), in `out`
        (may be logits; of the same type; columns behind the vocabulary are left as they are) or a new tensor [rows, vocabSize].

        history [rows, room] holds each row's tokens so far, lengths says how many, promptLengths how many of them were given (they count for
        repetition, not for presence and frequency).  repetition, presence, frequency: one number a row, or one for all.
        biasTokens, biases [rows, n]: ids (-1: unused place) and what is added.  mask [rows, words]: bit v & 31 of word v >> 5 allows token v, as
        TokenGrammar.allowedTokens makes them; with maskRows, row maskRows[r] of it is row r's, and none allows anything."""
        keep = []
        p = self._logits(keep, logits, history, lengths, promptLengths, repetition, presence, frequency, biasTokens, biases, mask, maskRows)
        if out is None:
            out = logits.new_empty((logits.shape[0], self.vocabSize))
        else:
            device_of(out, "out", self._engine.device_index, (str(logits.dtype),), (logits.shape[0], None))
            if out.shape[1] < self.vocabSize:
                raise ValueError(f"out: {out.shape[1]} columns, the vocabulary has {self.vocabSize} tokens")
            if out.shape[0] > 1 and out.stride(0) < self.vocabSize:
                raise ValueError("out: rows overlap")
        _lib.check(_lib.lib().b200bpe_sampler_adjust(self._h, C.byref(p), out.data_ptr(), out.stride(0), self._stream()), "b200bpe_sampler_adjust")
        return out

    def sample(self, logits, uniform=None, temperature=None, topK=None, topP=None, minP=None, history=None, lengths=None, promptLengths=None,
               repetition=None, presence=None, frequency=None, biasTokens=None, biases=None, mask=None, maskRows=None):
        """→ (tokens int32 [rows], logprobs float32 [rows]): adjustLogits and the choice of a token in one kernel.

        Without uniform every row takes its largest adjusted logit.  With uniform [rows] in [0, 1): of the topK largest (0: all), of those the shortest
        run from the largest on that has topP of their weight exp(x / temperature), of those the ones with at least minP times the largest weight,
        the first in order of ids at which the running sum of weights is above uniform times their sum.  temperature below
        2^-16: the largest.  Each is one number a row, or one for all.  logprobs are under the weights of all allowed tokens (at temperature 1
        where the largest is taken).  A row without an allowed token gives -1 and -inf; a NaN is never chosen."""
        keep = []
        p = self._logits(keep, logits, history, lengths, promptLengths, repetition, presence, frequency, biasTokens, biases, mask, maskRows)
        rows = logits.shape[0]
        c = _lib.Choice()
        c.struct_size = C.sizeof(_lib.Choice)
        if uniform is None:
            if any(x is not None for x in (temperature, topK, topP, minP)):
                raise ValueError("uniform: needed to draw")
        else:
            c.uniform = device_of(uniform, "uniform", self._engine.device_index, FLOATS, (rows,))
            for field, value, name, kinds in (("temperature", temperature, "temperature", FLOATS), ("top_k", topK, "topK", IDS),
                                              ("top_p", topP, "topP", FLOATS), ("min_p", minP, "minP", FLOATS)):
                if value is not None:
                    address, tensor = self._row(value, name, rows, kinds, logits)
                    setattr(c, field, address)
                    keep.append(tensor)
        import torch
        tokens, logprobs = logits.new_empty(rows, dtype=torch.int32), logits.new_empty(rows, dtype=torch.float32)
        c.tokens_out, c.logprobs_out = tokens.data_ptr(), logprobs.data_ptr()
        _lib.check(_lib.lib().b200bpe_sampler_sample(self._h, C.byref(p), C.byref(c), self._stream()), "b200bpe_sampler_sample")
        return tokens, logprobs

    def destroy(self):
        if self._h is not None:
            _lib.lib().b200bpe_sampler_destroy(self._h)
            self._h = None
