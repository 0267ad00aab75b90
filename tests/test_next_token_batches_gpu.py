"""The divisions of work that only large batches take: slices of 8,192 tokens, 8 and 16 rows to a CTA of the masks, more rows than a grid has."""
import numpy as np
import pytest

from gpu_bpe_b200 import TokenGrammar, TokenSampler
from tests import next_token_model as model
from tests.test_grammar_gpu import _automaton, _vocabulary
from tests.test_sampler_gpu import _agree, _arguments, _extras, _logits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab, rows, pad, shift", [(16_385, 260, 0, 0), (16_385, 260, 3, 1), (8_192, 620, 8, 3), (8_191, 640, 1, 2)])
def test_adjusted_logits(engine, torch, kind, vocab, rows, pad, shift):
    """More than 592 slices of 4,096 tokens with a history, on 148 SMs: every row against the same ten rows at a time, some against the model."""
    rng = np.random.default_rng(vocab + pad)
    s = TokenSampler(engine, vocab)
    t, values = _logits(rng, rows, vocab, kind, torch, pad, shift)
    e = _extras(rng, rows, vocab, room=300)
    e["history"][:, 20:60] = rng.integers(0, vocab, (rows, 40))
    a = _arguments(torch, e)
    got = s.adjustLogits(t, out=torch.full_like(t, 77.0), **a)
    assert (got[:, vocab:] == 77).all()
    for r in range(0, rows, 10):
        few = {k: v[r:r + 10].contiguous() for k, v in a.items()}
        assert torch.equal(s.adjustLogits(t[r:r + 10], **few), got[r:r + 10, :vocab])
    some = rng.choice(rows, 12, replace=False)
    x, bound = model.adjusted(values[some].astype(np.float64), np.float64, **{k: v[some] for k, v in e.items()})
    _agree(x, bound, got[:, :vocab][torch.from_numpy(some).cuda()].float().cpu().numpy(), kind)
    s.destroy()


@pytest.mark.parametrize("entries, rows", [(700, 20_480), (700, 21_001), (700, 40_960), (700, 41_003), (5003, 4_200), (5003, 8_211), (33, 1_100_003)])
def test_masks(engine, torch, entries, rows):
    rng = np.random.default_rng(rows)
    vocab = _vocabulary(rng, entries)
    table, accepting = _automaton(rng, 40)
    g = TokenGrammar(engine, vocab, table, accepting, entries - 1)
    every = model.packed(np.stack([model.allowed(vocab, table, accepting, entries - 1, s) for s in range(40)] + [np.zeros(entries, bool)]))
    some = rng.integers(-1, 40, rows).astype(np.int32)
    want, words = torch.from_numpy(every[some]).cuda(), every.shape[1]
    d = torch.from_numpy(some).cuda()
    assert torch.equal(g.allowedTokens(d), want)
    wide = torch.full((rows, words + 1), 5, dtype=torch.int32, device="cuda")
    g.allowedTokens(d, out=wide)
    assert torch.equal(wide[:, :words], want) and (wide[:, words] == 5).all()
    g.destroy()
