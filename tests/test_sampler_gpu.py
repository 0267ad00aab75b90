"""Adjusted logits and the choice of a token on the device against the plain model in 64 bits."""
import threading

import numpy as np
import pytest

from gpu_bpe_b200 import BPEEngine, TokenSampler
from tests import next_token_model as model

pytestmark = pytest.mark.gpu
VOCABS = [1, 2, 31, 33, 128, 129, 1000, 2049, 5000, 16385, 50021]
NEG = np.float32(np.finfo(np.float32).min)


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def _cuda(torch, a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _logits(rng, rows, vocab, kind, torch, pad=0, shift=0):
    """Logits with strong candidates on the device (rows `pad` elements longer than the vocabulary, `shift` elements into their memory), and their values."""
    x = rng.normal(0, 2.2, (rows, vocab))
    for r in range(rows):
        x[r, rng.integers(0, vocab, 12)] += 3 + 4 * np.abs(rng.normal(size=12))
    flat = torch.zeros(rows * (vocab + pad) + shift, dtype=getattr(torch, kind), device="cuda")
    t = flat[shift:].view(rows, vocab + pad)
    t.fill_(99.0)
    t[:, :vocab] = torch.from_numpy(x).to(getattr(torch, kind)).cuda()
    return t, t[:, :vocab].float().cpu().numpy()


def _extras(rng, rows, vocab, room=40, n_bias=6):
    """Histories with repeated, foreign and unused ids, lengths from none to more than there is room for; biases with ids twice; masks."""
    history = rng.integers(0, max(1, min(vocab, 60)), (rows, room)).astype(np.int32)
    history[:, ::7] = rng.integers(0, vocab, history[:, ::7].shape)
    history[:, 5::11], history[:, 6::13] = vocab, -1
    lengths = rng.integers(0, room + 1, rows).astype(np.int32)
    if rows > 1:
        lengths[0] = 0
    lengths[-1] = room + 5 if rows > 2 else room
    prompt = (rng.random(rows) * (lengths + 3)).astype(np.int32)
    rep = (0.7 + rng.random(rows)).astype(np.float32)
    rep[rng.random(rows) < 0.3] = 1
    pres, freq = rng.normal(size=rows).astype(np.float32), (rng.normal(size=rows) * (rng.random(rows) < 0.6)).astype(np.float32)
    tokens = rng.integers(-1, vocab + 1, (rows, n_bias)).astype(np.int32)
    tokens[:, 3] = tokens[:, 1]
    tokens[:, 5] = tokens[:, 1]
    biases = (rng.normal(size=(rows, n_bias)) * 5).astype(np.float32)
    mask = model.packed(rng.random((rows, vocab)) < rng.choice([0.03, 0.5, 0.98], (rows, 1)))
    return dict(history=history, lengths=lengths, prompt=prompt, repetition=rep, presence=pres, frequency=freq, bias_tokens=tokens, biases=biases, mask=mask)


NAMES = {"prompt": "promptLengths", "bias_tokens": "biasTokens", "mask_rows": "maskRows"}


def _arguments(torch, e):
    return {NAMES.get(k, k): _cuda(torch, v) for k, v in e.items()}


def _agree(x, bound, got, kind):
    """Adjusted logits in 64 bits against the device's: the steps' bound, and half a step of the result's type (for results below the normal
    ones, of the smallest of those)."""
    finite = np.isfinite(x)
    top = {"float32": 3.4028235e38, "float16": 65504.0, "bfloat16": 3.3895314e38}[kind]
    tiny = {"float32": 2.0 ** -126, "float16": 2.0 ** -14, "bfloat16": 2.0 ** -126}[kind]
    assert np.array_equal(np.isnan(x), np.isnan(got))
    fits = finite & (np.abs(x) < top)
    assert np.array_equal(got[~finite & ~np.isnan(x)], x[~finite & ~np.isnan(x)])
    half = model.HALF_STEP[kind] * np.maximum(np.abs(x) + bound, tiny)
    with np.errstate(invalid="ignore"):
        off = np.abs(got.astype(np.float64) - x)
    assert (off <= bound + half)[fits].all(), np.max((off - bound - half)[fits])


@pytest.mark.parametrize("kind", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("vocab", VOCABS)
def test_adjusted(engine, torch, kind, vocab):
    rng = np.random.default_rng(vocab)
    rows = 5
    s = TokenSampler(engine, vocab)
    e = _extras(rng, rows, vocab)
    for pad, shift, use in [(0, 0, e), (3, 1, e), (8, 0, {k: e[k] for k in ("mask",)}), (0, 5, {k: e[k] for k in ("bias_tokens", "biases")}),
                            (1, 0, {k: e[k] for k in ("history", "lengths", "frequency")}), (0, 0, {k: e[k] for k in ("history", "lengths", "repetition")}), (0, 3, {})]:
        t, values = _logits(rng, rows, vocab, kind, torch, pad, shift)
        x, bound = model.adjusted(values.astype(np.float64), np.float64, **use)
        out = torch.full_like(t, 77.0)
        a = _arguments(torch, use)
        got = s.adjustLogits(t, out=out, **a)
        assert got is out and (out[:, vocab:] == 77).all()
        _agree(x, bound, out[:, :vocab].float().cpu().numpy(), kind)
        fresh = s.adjustLogits(t, **a)
        assert fresh.shape == (rows, vocab) and torch.equal(fresh, out[:, :vocab])
        s.adjustLogits(t, out=t, **a)                        # in place
        assert torch.equal(t[:, :vocab], fresh) and (t[:, vocab:] == 99).all()
    s.destroy()


@pytest.mark.parametrize("kind", ["float32", "float16", "bfloat16"])
def test_adjusted_odd_values(engine, torch, kind):
    """Infinities, NaN and the type's lowest value, in masked and in allowed places; masks that leave nothing."""
    vocab, rows = 700, 4
    rng = np.random.default_rng(3)
    s = TokenSampler(engine, vocab)
    t, _ = _logits(rng, rows, vocab, kind, torch)
    low = torch.finfo(t.dtype).min
    for k, v in enumerate([float("nan"), float("inf"), float("-inf"), low, -low, 0.0, -0.0]):
        t[:, 10 + k] = v
        t[:, 110 + k] = v
    values = t.float().cpu().numpy()
    e = _extras(rng, rows, vocab)
    e["history"][:, :14] = np.r_[10:17, 110:117]
    e["lengths"][:] = 20
    e["biases"][0, 0], e["biases"][1, 0] = np.inf, -np.inf
    bits = rng.random((rows, vocab)) < 0.7
    bits[:, 10:17], bits[:, 110:117], bits[2] = True, False, False
    e["mask"] = model.packed(bits)
    x, bound = model.adjusted(values.astype(np.float64), np.float64, **e)
    x[np.abs(x) > {"float16": 65504.0}.get(kind, 3.4e38)] *= np.inf          # (too large for the type, by far)
    _agree(x, bound, s.adjustLogits(t, **_arguments(torch, e)).float().cpu().numpy(), kind)
    s.destroy()


def _compare(x, tokens, logprobs, vocab, u=None, **settings):
    for r in range(len(x)):
        pick = lambda n, d: d if settings.get(n) is None else settings[n][r]  # noqa: E731
        v, lp, gap = model.choice(x[r], None if u is None else u[r], pick("t", 1.0), int(pick("k", 0)), pick("p", 1.0), pick("m", 0.0))
        assert tokens[r] == v or gap < 1e-12, (r, tokens[r], v, gap)
        if v < 0:
            assert tokens[r] == -1 and logprobs[r] == -np.inf
        elif tokens[r] == v:
            assert abs(logprobs[r] - lp) <= model.logprob_bound(lp, vocab), (r, logprobs[r], lp)


def _settings(rng, rows, vocab):
    t = np.where(rng.random(rows) < 0.15, 0, 0.05 + 1.6 * rng.random(rows)).astype(np.float32)
    k = rng.choice([0, 0, 1, 2, 20, 50, vocab // 2, vocab, vocab + 7], rows).astype(np.int32)
    p = rng.choice([1.0, 1.0, 0.95, 0.9, 0.5, 0.05], rows).astype(np.float32)
    m = rng.choice([0.0, 0.0, 0.02, 0.3], rows).astype(np.float32)
    return rng.random(rows).astype(np.float32), dict(t=t, k=k, p=p, m=m)


CALL = {"t": "temperature", "k": "topK", "p": "topP", "m": "minP"}


def _sample(torch, s, t, u=None, settings={}, **more):
    tokens, logprobs = s.sample(t, **({} if u is None else {"uniform": _cuda(torch, u)}), **{CALL[n]: _cuda(torch, v) for n, v in settings.items()}, **more)
    return tokens.cpu().numpy(), logprobs.cpu().numpy()


@pytest.mark.parametrize("kind", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("vocab", VOCABS + [131072, 262145])
def test_choice(engine, torch, kind, vocab):
    rng = np.random.default_rng(vocab + 1)
    rows = 24 if vocab < 100_000 else 6
    s = TokenSampler(engine, vocab)
    t, values = _logits(rng, rows, vocab, kind, torch, *[(0, 0), (3, 1), (8, 3)][vocab % 3])
    u, settings = _settings(rng, rows, vocab)
    for use in [settings, {}, {"t": settings["t"]}, {"k": settings["k"]}, {"p": settings["p"]}, {"m": settings["m"]}]:
        _compare(values, *_sample(torch, s, t, u, use), vocab, u, **use)
    _compare(values, *_sample(torch, s, t), vocab)
    e = _extras(rng, rows, vocab)
    x, _ = model.adjusted(values, np.float32, **e)
    a = _arguments(torch, e)
    _compare(x, *_sample(torch, s, t, u, settings, **a), vocab, u, **settings)
    again = _sample(torch, s, t, u, settings, **a)
    assert all(np.array_equal(p, q) for p, q in zip(again, _sample(torch, s, t, u, settings, **a)))
    s.destroy()


@pytest.mark.parametrize("vocab", [3, 130, 4099, 40000])
def test_borders_and_ties(engine, torch, vocab):
    """Equal logits and a handful of values, where each border is a tie; the ends of every setting's range."""
    s = TokenSampler(engine, vocab)
    rng = np.random.default_rng(vocab)
    top = np.float32(1 - 2.0 ** -24)
    for values in (np.zeros(vocab), np.arange(vocab) % 3 * 1.0, np.where(np.arange(vocab) == vocab // 2, 5.0, -5.0), -np.arange(vocab) / 64):
        u = np.array([0, 0.5, top, 0.25, 0.75, 0.3, 0.999, 0.0, 0.1, top, top, 0.6], np.float32)
        rows = len(u)
        x = np.tile(values.astype(np.float32), (rows, 1))
        t = _cuda(torch, x)
        for k, p, m in [(0, 1.0, 0.0), (2, 1.0, 0.0), (vocab // 2, 1.0, 0.0), (vocab - 1, 0.5, 0.0), (0, 0.5, 0.0), (0, 0.25, 0.3), (0, 1.0, 1.0), (0, 0.0, 0.0),
                        (7, 0.75, 0.0), (0, 1e-30, 0.0), (0, float(top), 0.0), (5, 0.3, 1.0)]:
            st = dict(k=np.full(rows, k, np.int32), p=np.full(rows, p, np.float32), m=np.full(rows, m, np.float32))
            _compare(x, *_sample(torch, s, t, u, st), vocab, u, **st)
    s.destroy()


def test_settings_out_of_range(engine, torch):
    vocab, rows = 5000, 16
    rng = np.random.default_rng(9)
    s = TokenSampler(engine, vocab)
    t, values = _logits(rng, rows, vocab, "float32", torch)
    nan, inf = np.float32("nan"), np.float32("inf")
    u = np.array([nan, -1, 1, 2, inf, -inf, 0.5, 0.5, 0.5, 0.5, 0.5, 0.5, 0.5, 0.5, 0.5, 0.5], np.float32)
    st = dict(t=np.array([1, 1, 1, 1, 1, 1, nan, inf, -1, 1e-6, 3e38, 2.0 ** -16, 1, 1, 1, 1], np.float32),
              p=np.array([1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, nan, -3, inf, 2], np.float32),
              m=np.array([0] * 14 + [nan, 5], np.float32))
    tokens, logprobs = _sample(torch, s, t, u, st)
    st["p"] = np.nan_to_num(st["p"], nan=1.0)
    st["m"] = np.nan_to_num(st["m"], nan=0.0)
    _compare(values, tokens, logprobs, vocab, u, **st)
    s.destroy()


def test_plain_numbers_as_settings(engine, torch):
    vocab, rows = 900, 6
    rng = np.random.default_rng(2)
    s = TokenSampler(engine, vocab)
    t, values = _logits(rng, rows, vocab, "float32", torch)
    u = rng.random(rows).astype(np.float32)
    got = _sample(torch, s, t, u, {}, temperature=0.7, topK=40, topP=0.9, minP=0.01)
    full = lambda v, d=np.float32: np.full(rows, v, d)  # noqa: E731
    _compare(values, *got, vocab, u, t=full(0.7), k=full(40, np.int32), p=full(0.9), m=full(0.01))
    s.destroy()


def test_odd_values_in_a_choice(engine, torch):
    """NaN, infinities, the lowest values; rows of which a mask or the logits leave nothing."""
    vocab = 1300
    rng = np.random.default_rng(4)
    s = TokenSampler(engine, vocab)
    t, values = _logits(rng, 14, vocab, "float32", torch)
    values[0, :] = -np.inf
    values[1, :] = np.nan
    values[2, 5:900:7] = np.nan
    values[3, [7, 1200]] = np.inf
    values[4, :] = NEG
    values[5, :1299] = -np.inf
    values[6, 100:] = NEG
    values[7] = np.where(np.arange(vocab) % 2, -NEG, NEG)
    values[8, 3:] = np.nan
    values[8, :3] = -np.inf
    values[9, :] = np.where(rng.random(vocab) < 0.5, 0.0, -0.0)
    values[10, 0] = np.inf
    t = _cuda(torch, values)
    bits = rng.random((14, vocab)) < 0.5
    bits[11], bits[12] = False, False
    bits[12, 77] = True
    bits[3, 7], bits[10, 0] = True, False
    u = rng.random(14).astype(np.float32)
    for mask in (None, model.packed(bits)):
        x = values if mask is None else np.where(bits, values, -np.inf)
        more = {} if mask is None else {"mask": _cuda(torch, mask)}
        _compare(x, *_sample(torch, s, t, **more), vocab)
        for st in ({}, {"k": np.full(14, 30, np.int32)}, {"p": np.full(14, 0.9, np.float32)}, {"m": np.full(14, 0.1, np.float32)},
                   {"k": np.full(14, 700, np.int32), "p": np.full(14, 0.6, np.float32), "t": np.full(14, 2.5, np.float32)}):
            _compare(x, *_sample(torch, s, t, u, st, **more), vocab, u, **st)
    s.destroy()


@pytest.mark.parametrize("low", [-1e9, -2e9, -5e9, -65504.0, -3e4, -1e38])
def test_low_values_and_temperatures(engine, torch, low):
    """Tokens put far below the others, rows that lie far out as a whole, at temperatures that make x / temperature large."""
    vocab, rows = 6000, 12
    rng = np.random.default_rng(6)
    s = TokenSampler(engine, vocab)
    _, values = _logits(rng, rows, vocab, "float32", torch)
    values[:3][rng.random((3, vocab)) < 0.5] = low
    values[3:6, 40:5900] = low
    values[6] += 400
    values[7] += 3e4
    values[8] += 1e8
    values[9] -= 2e9
    values[10, :] = low
    values[11, :] = low
    values[11, 17] = low / 2
    t = _cuda(torch, values)
    u = rng.random(rows).astype(np.float32)
    _compare(values, *_sample(torch, s, t), vocab)
    for warm in (1.0, 0.9, 0.7, 0.6, 0.4, 0.3, 0.2, 1e-3, 3e-5, 2.0 ** -16):
        for st in ({}, {"k": np.full(rows, 50, np.int32)}, {"k": np.full(rows, 3000, np.int32)}, {"p": np.full(rows, 0.9, np.float32)}, {"m": np.full(rows, 0.1, np.float32)}):
            st = dict(st, t=np.full(rows, warm, np.float32))
            _compare(values, *_sample(torch, s, t, u, st), vocab, u, **st)
    s.destroy()


def test_masks_shared_by_rows(engine, torch):
    vocab, rows = 2100, 7
    rng = np.random.default_rng(5)
    s = TokenSampler(engine, vocab)
    t, values = _logits(rng, rows, vocab, "float16", torch)
    bits = rng.random((3, vocab)) < 0.1
    wide = np.full((3, (vocab + 31) // 32 + 4), -1, np.int32)
    wide[:, :(vocab + 31) // 32] = model.packed(bits)
    which = np.array([0, 2, 1, 1, 3, -1, 0], np.int32)
    x = np.stack([np.where(bits[k], values[r], -np.inf) if 0 <= k < 3 else np.full(vocab, -np.inf) for r, k in enumerate(which)])
    more = dict(mask=_cuda(torch, wide), maskRows=_cuda(torch, which))
    u = rng.random(rows).astype(np.float32)
    _compare(x, *_sample(torch, s, t, u, **more), vocab, u)
    assert np.array_equal(s.adjustLogits(t, **more).float().cpu().numpy(), x.astype(np.float32))
    s.destroy()


def test_long_lists(engine, torch):
    """1,024 biases a row, most of them twice or more; a long history of few tokens."""
    vocab, rows = 9000, 3
    rng = np.random.default_rng(6)
    s = TokenSampler(engine, vocab)
    t, values = _logits(rng, rows, vocab, "float32", torch)
    e = dict(history=rng.integers(0, 40, (rows, 30_000)).astype(np.int32), lengths=np.array([30_000, 29_999, 1], np.int32), prompt=np.array([100, 0, 1], np.int32),
             repetition=np.float32([1.3, 0.8, 1.1]), frequency=np.float32([1e-3, 0, 2]), presence=np.float32([0, 0.5, 1]),
             bias_tokens=rng.integers(0, 500, (rows, 1024)).astype(np.int32), biases=rng.normal(size=(rows, 1024)).astype(np.float32))
    x, bound = model.adjusted(values.astype(np.float64), np.float64, **e)
    _agree(x, bound, s.adjustLogits(t, **_arguments(torch, e)).cpu().numpy(), "float32")
    x, _ = model.adjusted(values, np.float32, **e)
    assert np.array_equal(s.adjustLogits(t, **_arguments(torch, e)).cpu().numpy(), x)       # biases of a token in the order of the list
    s.destroy()


def test_no_rows_and_no_history(engine, torch):
    s = TokenSampler(engine, 50)
    t = torch.zeros(0, 50, device="cuda")
    tokens, logprobs = s.sample(t, uniform=torch.zeros(0, device="cuda"))
    assert tokens.shape == logprobs.shape == (0,) and s.adjustLogits(t).shape == (0, 50)
    t = torch.randn(2, 50, device="cuda")
    empty = dict(history=torch.zeros(2, 0, dtype=torch.int32, device="cuda"), lengths=torch.zeros(2, dtype=torch.int32, device="cuda"), repetition=2.0)
    assert torch.equal(s.adjustLogits(t, **empty), t) and torch.equal(s.sample(t, **empty)[0], t.argmax(1).int())
    s.destroy()


def test_many_rows(engine, torch):
    vocab, rows = 300, 20_000
    s = TokenSampler(engine, vocab)
    t = torch.randn(rows, vocab, device="cuda")
    assert torch.equal(s.sample(t)[0], t.argmax(1).int())
    u = torch.rand(rows, device="cuda")
    tokens = s.sample(t, uniform=u)[0]
    for r in range(0, rows, 997):
        v, _, gap = model.choice(t[r].cpu().numpy(), float(u[r]))
        assert int(tokens[r]) == v or gap < 1e-12
    s.destroy()


def test_streams_threads_and_graphs(engine, torch):
    """One handle: calls on several streams from several threads, and two captured graphs that replay at the same time."""
    vocab, rows = 20_000, 9
    s = TokenSampler(engine, vocab)
    rng = np.random.default_rng(8)
    sets = []
    for k in range(3):
        t, values = _logits(rng, rows, vocab, "bfloat16", torch)
        u, st = _settings(rng, rows, vocab)
        e = _extras(rng, rows, vocab)
        a = dict(_arguments(torch, e), uniform=_cuda(torch, u), **{CALL[n]: _cuda(torch, v) for n, v in st.items()})
        sets.append((t, a, [x.cpu() for x in s.sample(t, **a)]))
    torch.cuda.synchronize()
    failed = []

    def work(k):
        try:
            t, a, want = sets[k]
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = s.sample(t, **a)
                    if not all(torch.equal(x.cpu(), y) for x, y in zip(got, want)):
                        failed.append(k)
        except BaseException as e:
            failed.append(e)
    threads = [threading.Thread(target=work, args=(k,)) for k in range(3)]
    for th in threads:
        th.start()
    for th in threads:
        th.join(120)
    assert not failed
    graphs = []
    for t, a, want in sets[:2]:
        side = torch.cuda.Stream()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = s.sample(t, **a)
        graphs.append((g, out, side, want))
    for _ in range(5):
        for g, _, side, _ in graphs:
            with torch.cuda.stream(side):
                g.replay()
    torch.cuda.synchronize()
    for _, out, _, want in graphs:
        assert all(torch.equal(x.cpu(), y) for x, y in zip(out, want))
    s.destroy()


def test_a_sampler_outlives_its_engine(torch):
    e = BPEEngine(0).init()
    s = TokenSampler(e, 100)
    t = torch.randn(3, 100, device="cuda")
    e.destroy()
    assert torch.equal(s.sample(t)[0], t.argmax(1).int())
    s.destroy()


@pytest.mark.parametrize("length", [1, 255, 256, 2047, 2048, 2049, 5000])
def test_lengths_of_a_history(engine, torch, length):
    """Either side of what a thread keeps at hand; most of it one token, the rest spread over the vocabulary."""
    vocab, rows = 40_000, 2
    rng = np.random.default_rng(length)
    s = TokenSampler(engine, vocab)
    t, values = _logits(rng, rows, vocab, "bfloat16", torch)
    history = np.where(rng.random((rows, length)) < 0.4, 17, rng.integers(0, vocab, (rows, length))).astype(np.int32)
    e = dict(history=history, lengths=np.full(rows, length, np.int32), prompt=np.array([0, length // 3], np.int32), repetition=np.float32([1.4, 1]),
             frequency=np.float32([0.01, 0.02]), presence=np.float32([0.3, 0]), mask=model.packed(rng.random((rows, vocab)) < 0.9))
    x, bound = model.adjusted(values.astype(np.float64), np.float64, **e)
    a = _arguments(torch, e)
    _agree(x, bound, s.adjustLogits(t, **a).float().cpu().numpy(), "bfloat16")
    x, _ = model.adjusted(values, np.float32, **e)
    u, st = _settings(rng, rows, vocab)
    _compare(x, *_sample(torch, s, t, u, st, **a), vocab, u, **st)
    a["history"], a["lengths"] = a["history"].view(torch.uint32), a["lengths"].view(torch.uint32)
    _compare(x, *_sample(torch, s, t, u, st, **a), vocab, u, **st)
    s.destroy()


def test_the_largest_vocabulary(engine, torch):
    vocab, rows = 327_680, 3
    rng = np.random.default_rng(10)
    s = TokenSampler(engine, vocab)
    t, values = _logits(rng, rows, vocab, "float16", torch)
    u = rng.random(rows).astype(np.float32)
    for st in ({}, {"k": np.array([3, 300, 100_000], np.int32)}, {"p": np.full(rows, 0.97, np.float32), "t": np.float32([0.3, 1, 1.5])}):
        _compare(values, *_sample(torch, s, t, u, st), vocab, u, **st)
    s.destroy()


def test_one_row_for_all(engine, torch):
    """Rows that lie on top of one another are only read."""
    vocab, rows = 7000, 9
    rng = np.random.default_rng(11)
    s = TokenSampler(engine, vocab)
    t, values = _logits(rng, 1, vocab, "float32", torch)
    u = ((np.arange(rows) + 0.5) / rows).astype(np.float32)
    x = np.repeat(values, rows, 0)
    _compare(x, *_sample(torch, s, t.expand(rows, vocab), u), vocab, u)
    assert torch.equal(s.adjustLogits(t.expand(rows, vocab)), t.expand(rows, vocab))
    s.destroy()


def test_draws_follow_the_weights(engine, torch):
    """Uniforms on a grid draw each token as often as its share of the grid, to one."""
    vocab, n = 3000, 20_000
    rng = np.random.default_rng(12)
    s = TokenSampler(engine, vocab)
    t, values = _logits(rng, 1, vocab, "float32", torch)
    u = (torch.arange(n, device="cuda") + 0.5) / n
    tokens = s.sample(t.expand(n, vocab), u, topK=torch.full((n,), 40, dtype=torch.int32, device="cuda"))[0].cpu().numpy()
    order = np.argsort(-values[0], kind="stable")[:40]
    w = np.exp(values[0].astype(np.float64) - values[0].max())
    share = np.zeros(vocab)
    share[order] = w[order] / w[order].sum()
    assert np.abs(np.bincount(tokens, minlength=vocab) - n * share).max() <= 1 and (np.diff(tokens) >= 0).all()
    s.destroy()
