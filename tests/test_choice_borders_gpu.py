"""Draws and top_p borders that lie behind nearly all of a row's weight: the token is the one that weights in 64 bits choose.

Sums of weights in 32 bits are off by some 2^-24 of the whole, which is more than the tokens behind a dominant one weigh, so a border there
cannot be told from such sums."""
import numpy as np
import pytest

from gpu_bpe_b200 import TokenSampler
from tests import next_token_model as model

pytestmark = pytest.mark.gpu
NEAR = 1e-12         # of the whole: nearer than that, sums in 64 bits do not tell either (a few hundred of their steps of 2^-53, and weights of 4e-14)


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def _row(rng, vocab, top, at, kind, torch, spread=1.0):
    """Logits of a row in which the token `at` has about `top` of the weight, and their values."""
    x = rng.normal(0, spread, vocab)
    x += np.log((1 / top - 1) / np.exp(np.delete(x, at)).sum())
    x[at] = 0
    t = torch.from_numpy(x).to(getattr(torch, kind))
    return t, t.float().numpy().astype(np.float64)


def _floats(first):
    """Every 32-bit number from `first`, at least a half, up to 1."""
    return (np.arange(int(first * 2 ** 24), 2 ** 24) / 2.0 ** 24).astype(np.float32)


def _draws(x, kept, u):
    """(token, gap) of each u among the tokens `kept`, ascending, of a row."""
    w = np.exp(x[kept] - x.max()).astype(np.longdouble)
    run = np.cumsum(w)
    target = u.astype(np.longdouble) * run[-1]
    i = np.minimum(np.searchsorted(run, target, side="right"), len(kept) - 1)
    gap = np.minimum(np.abs(run[i] - target), np.abs(run[i] - w[i] - target)) / run[-1]
    return kept[i], gap.astype(np.float64)


def _wrong(x, kept, u, tokens):
    want, gap = _draws(x, kept, u)
    return int(((tokens != want) & (gap >= NEAR)).sum())


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab, top, at", [(256, 0.9996, 0), (256, 0.9996, 77), (2048, 0.99, 0), (2048, 0.99, 1100), (2048, 0.9996, 1900), (20_000, 0.9996, 300)])
def test_draws_behind_a_dominant_token(engine, torch, kind, vocab, top, at):
    """Without limits, with a min_p that takes nothing away, with a top_k and a top_p of nearly all."""
    rng = np.random.default_rng(vocab + at)
    s = TokenSampler(engine, vocab)
    t, x = _row(rng, vocab, top, at, kind, torch)
    u = _floats(top if vocab < 2048 else 0.9985)
    order = np.argsort(-x, kind="stable")
    everything = np.arange(vocab)
    some = np.float32(0.99995)
    sums = np.cumsum(np.exp(x[order]).astype(np.longdouble))
    assert np.abs(sums - np.longdouble(some) * sums[-1]).min() > NEAR * sums[-1]
    by_p = np.sort(order[:1 + int(np.sum(sums[:-1] < np.longdouble(some) * sums[-1]))])
    by_k = np.sort(order[:vocab - 3])
    assert len(by_p) < vocab
    wrong = {}
    for shift in range(8 if kind == "bfloat16" else 4):
        flat = torch.zeros(vocab + shift, dtype=t.dtype, device="cuda")
        flat[shift:] = t.cuda()
        logits, uniform = flat[shift:].expand(len(u), vocab), torch.from_numpy(u).cuda()
        for name, kept, how in [("all", everything, {}), ("min_p", everything, {"minP": 1e-30}), ("top_k", by_k, {"topK": vocab - 3}), ("top_p", by_p, {"topP": float(some)})]:
            tokens = s.sample(logits, uniform, **how)[0].cpu().numpy()
            wrong[name, shift] = _wrong(x, kept, u, tokens)
    s.destroy()
    assert not any(wrong.values()), wrong


@pytest.mark.parametrize("vocab, rows", [(2_048, 60), (32_256, 40), (131_072, 25)])
@pytest.mark.parametrize("spread", [1.0, 2.0])
@pytest.mark.parametrize("p", [0.99, 0.995, 0.999, 0.9999])
def test_top_p_behind_a_dominant_token(engine, torch, vocab, rows, p, spread):
    """Logits descend with the ids and uniform is at its end, so that the token is the last one that top_p keeps."""
    rng = np.random.default_rng(vocab)
    s = TokenSampler(engine, vocab)
    x = np.stack([np.r_[0, np.sort(_row(rng, vocab, 0.94, 0, "float32", torch, spread)[1][1:])[::-1]] for _ in range(rows)]).astype(np.float32)
    p = np.float32(p)
    tokens = s.sample(torch.from_numpy(x).cuda(), torch.ones(rows, device="cuda"), topP=float(p))[0].cpu().numpy()
    s.destroy()
    wrong = []
    for r in range(rows):
        sums = np.cumsum(np.exp(x[r].astype(np.float64)).astype(np.longdouble))
        border = np.longdouble(p) * sums[-1]
        if tokens[r] != int(np.sum(sums[:-1] < border)) and np.abs(sums - border).min() >= NEAR * sums[-1]:
            wrong.append((r, int(tokens[r])))
    assert not wrong


@pytest.mark.parametrize("p", [0.999, 0.9999, 0.99999])
def test_top_p_of_few_tokens(engine, torch, p):
    """What top_p keeps is a short list of tokens, each the only one of some weight among its neighbours."""
    vocab, rows = 2048, 400
    rng = np.random.default_rng(7)
    s = TokenSampler(engine, vocab)
    x = np.full((rows, vocab), -40.0)
    x[:, ::8] = -np.sort(rng.uniform(3, 17, (rows, vocab // 8)), 1)
    x[:, 0] = 0
    t = torch.from_numpy(x).to(torch.bfloat16)
    x, p = t.double().numpy(), np.float32(p)
    tokens = s.sample(t.cuda(), torch.ones(rows, device="cuda"), topP=float(p))[0].cpu().numpy()
    s.destroy()
    wrong = []
    for r in range(rows):
        order = np.argsort(-x[r], kind="stable")
        sums = np.cumsum(np.exp(x[r, order]).astype(np.longdouble))
        border = np.longdouble(p) * sums[-1]
        want = int(order[:1 + int(np.sum(sums[:-1] < border))].max())
        if tokens[r] != want and np.abs(sums - border).min() >= NEAR * sums[-1]:
            wrong.append((r, int(tokens[r]), want))
    assert not wrong


def test_uniforms_next_to_nothing(engine, torch):
    """A uniform of almost 0 falls to the first token that has any weight in 64 bits, however little."""
    vocab = 3000
    s = TokenSampler(engine, vocab)
    x = np.zeros((5, vocab), np.float32)
    x[:, :700], x[:, 5] = -np.inf, -95        # e^-95 is below the smallest normal number in 32 bits
    u = np.float32([0, 1e-45, 1e-44, 1e-43, 1e-38])
    tokens, _ = s.sample(torch.from_numpy(x).cuda(), torch.from_numpy(u).cuda())
    want = [model.choice(x[r], u[r])[0] for r in range(5)]
    assert want == [5, 5, 700, 700, 700] and tokens.cpu().numpy().tolist() == want
    s.destroy()
