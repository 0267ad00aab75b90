"""Masks and steps of a byte automaton over a vocabulary on the device against the plain model, and the whole way from logits to text."""
import numpy as np
import pytest

from gpu_bpe_b200 import TokenGrammar, TokenSampler, TrieTokenizer, _lib
from tests import next_token_model as model

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def _vocabulary(rng, n, alphabet=b"abc,"):
    entries = [b"", b"a", b"", b"abcabcabc" * 30]
    while len(entries) < n:
        entries.append(bytes(rng.choice(list(alphabet), int(rng.integers(1, 12)))))
    return entries[:n]


def _automaton(rng, states, alphabet=b"abc,", dead=0.4):
    table = np.full((states, 256), -1)
    for b in alphabet:
        table[:, b] = np.where(rng.random(states) < dead, rng.choice([-1, states, 2**31 - 1], states), rng.integers(0, states, states))
    return table, (rng.random(states) < 0.4).astype(int)


@pytest.mark.parametrize("entries", [1, 3, 31, 32, 33, 500, 5003])
@pytest.mark.parametrize("states", [1, 2, 300])
@pytest.mark.parametrize("dead", [0.0, 0.3, 1.0])
def test_masks_and_steps(engine, torch, entries, states, dead):
    rng = np.random.default_rng(entries * 7 + states)
    vocab = _vocabulary(rng, entries)
    table, accepting = _automaton(rng, states, dead=dead)
    end = None if entries == 3 else entries - 1
    g = TokenGrammar(engine, vocab, table, accepting, end)
    some = np.r_[rng.integers(0, states, 7), -1, states, 2**31 - 1].astype(np.int32)
    want = model.packed(np.stack([model.allowed(vocab, table, accepting, end, s) for s in some]))
    d = torch.from_numpy(some).cuda()
    assert np.array_equal(g.allowedTokens(d).cpu().numpy(), want)
    wide = torch.full((len(some), want.shape[1] + 3), 5, dtype=torch.int32, device="cuda")
    assert g.allowedTokens(d, out=wide) is wide
    assert np.array_equal(wide[:, :want.shape[1]].cpu().numpy(), want) and (wide[:, want.shape[1]:] == 5).all()
    tokens = rng.integers(-1, entries + 1, (60, len(some))).astype(np.int32)
    tokens[0] = end if end is not None else 0
    for row in tokens:
        expect = []
        for s, t in zip(some, row):
            if t == -1:
                expect.append(s)
            elif not 0 <= s < states or not 0 <= t < entries:
                expect.append(-1)
            elif t == end:
                expect.append(s if accepting[s] else -1)
            else:
                expect.append(model.walk(table, s, vocab[t]) if vocab[t] else -1)
        got = g.advance(d, torch.from_numpy(row).cuda())
        assert got.cpu().numpy().tolist() == expect
        if entries > 100:
            break
    g.destroy()


def test_many_bytes_and_states(engine, torch):
    """All 256 bytes as classes of their own, and more states than fit a CTA's memory."""
    rng = np.random.default_rng(1)
    vocab = [bytes([b]) for b in range(256)] + [rng.bytes(int(rng.integers(1, 9))) for _ in range(700)]
    for states in (5, 1000, 65535):
        table = rng.integers(-states // 8, states, (states, 256))
        accepting = rng.integers(0, 2, states)
        g = TokenGrammar(engine, vocab, table, accepting, 17)
        some = np.r_[rng.integers(0, states, 5), states - 1].astype(np.int32)
        want = model.packed(np.stack([model.allowed(vocab, table, accepting, 17, s) for s in some]))
        assert np.array_equal(g.allowedTokens(torch.from_numpy(some).cuda()).cpu().numpy(), want)
        g.destroy()


def test_many_rows(engine, torch):
    rng = np.random.default_rng(2)
    vocab = _vocabulary(rng, 700)
    table, accepting = _automaton(rng, 40)
    g = TokenGrammar(engine, vocab, table, accepting, 699)
    every = model.packed(np.stack([model.allowed(vocab, table, accepting, 699, s) for s in range(40)]))
    for rows in (1, 2, 39, 256, 9001):
        some = rng.integers(0, 40, rows).astype(np.int32)
        assert np.array_equal(g.allowedTokens(torch.from_numpy(some).cuda()).cpu().numpy(), every[some])
    assert g.allowedTokens(torch.zeros(0, dtype=torch.int32, device="cuda")).shape == (0, 22)
    g.destroy()


def test_history(engine, torch):
    rng = np.random.default_rng(3)
    vocab = _vocabulary(rng, 50)
    table, accepting = _automaton(rng, 9, dead=0.1)
    g = TokenGrammar(engine, vocab, table, accepting, 49)
    rows, room = 600, 12
    before = rng.integers(0, 50, (rows, room + 4)).astype(np.int32)
    lengths = rng.integers(0, room + 3, rows).astype(np.int32)
    tokens = rng.integers(-1, 50, rows).astype(np.int32)
    states = torch.from_numpy(rng.integers(0, 9, rows).astype(np.int32)).cuda()
    wide = torch.from_numpy(before).cuda()
    new, longer = g.advance(states, torch.from_numpy(tokens).cuda(), history=wide[:, :room], lengths=torch.from_numpy(lengths).cuda())
    want, counts = before.copy(), lengths.copy()
    for r in range(rows):
        if tokens[r] >= 0 and lengths[r] < room:
            want[r, lengths[r]] = tokens[r]
            counts[r] += 1
    assert np.array_equal(wide.cpu().numpy(), want) and np.array_equal(longer.cpu().numpy(), counts)
    assert torch.equal(new, g.advance(states, torch.from_numpy(tokens).cuda()))
    # in place
    again, n, s = torch.from_numpy(before).cuda(), torch.from_numpy(lengths).cuda(), states.clone()
    out = g.advance(s, torch.from_numpy(tokens).cuda(), history=again[:, :room], lengths=n, out=s, lengthsOut=n)
    assert out[0] is s and out[1] is n and torch.equal(s, new) and torch.equal(n, longer) and torch.equal(again, wide)
    empty = torch.zeros(rows, 0, dtype=torch.int32, device="cuda")
    assert torch.equal(g.advance(states, torch.from_numpy(tokens).cuda(), history=empty, lengths=longer)[1], longer)
    g.destroy()


def _words_and_numbers():
    """key=<letters>;n=<digits>. with at least one letter and digit."""
    table, accepting = np.full((9, 256), -1), np.zeros(9, int)
    for s, b in enumerate(b"k="):
        table[s, b] = s + 1
    for b in range(97, 123):
        table[2, b] = table[3, b] = 3
    table[3, ord(";")] = 4
    table[4, ord("n")] = 5
    table[5, ord("=")] = 6
    for b in range(48, 58):
        table[6, b] = table[7, b] = 7
    table[7, ord(".")] = 8
    accepting[8] = 1
    return table, accepting


@pytest.mark.parametrize("graph", [False, True])
def test_from_logits_to_text(engine, torch, graph):
    """A batch is generated under a grammar, each step through mask, choice and advance (as calls or as one captured graph); every step against the
    plain model, the texts against the automaton."""
    rng = np.random.default_rng(12)
    vocab = [bytes([b]) for b in range(256)] + [b"k=", b"ab", b"the", b"ing", b";n=", b"12", b"7.", b"k=z", b"e;", b"99", b"x" * 6] + [b""]
    end, rows, room = len(vocab) - 1, 6, 40
    tok = TrieTokenizer.fromVocab(engine, vocab)
    table, accepting = _words_and_numbers()
    g, s = tok.grammar(table, accepting, end), tok.sampler()
    assert isinstance(g, TokenGrammar) and isinstance(s, TokenSampler) and s.vocabSize == len(vocab)
    prompt = tok.encodeBytes(b"the k=")
    history = torch.zeros(rows, room, dtype=torch.int32, device="cuda")
    history[:, :len(prompt)] = torch.from_numpy(prompt.astype(np.int32)).cuda()
    begin = torch.full((rows,), len(prompt), dtype=torch.int32, device="cuda")
    lengths, states = begin.clone(), torch.zeros(rows, dtype=torch.int32, device="cuda")
    logits, uniform = torch.zeros(rows, len(vocab), dtype=torch.bfloat16, device="cuda"), torch.zeros(rows, device="cuda")
    mask = torch.zeros(rows, (len(vocab) + 31) // 32, dtype=torch.int32, device="cuda")
    settings = dict(temperature=torch.full((rows,), 0.9, device="cuda"), topK=torch.full((rows,), 9, dtype=torch.int32, device="cuda"),
                    topP=torch.full((rows,), 0.97, device="cuda"), repetition=torch.full((rows,), 1.2, device="cuda"),
                    frequency=torch.full((rows,), 0.3, device="cuda"))

    def step():
        g.allowedTokens(states, out=mask)
        tokens, logprobs = s.sample(logits, uniform, history=history, lengths=lengths, promptLengths=begin, mask=mask, **settings)
        g.advance(states, tokens, history=history, lengths=lengths, out=states, lengthsOut=lengths)
        return tokens, logprobs
    if graph:
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            out = step()
    done = np.zeros(rows, bool)
    for n in range(30):
        values = torch.from_numpy(rng.normal(0, 3, logits.shape)).to(torch.bfloat16)
        values[:, end] += 4
        u = rng.random(rows).astype(np.float32)
        logits.copy_(values)
        uniform.copy_(torch.from_numpy(u))
        now = [x.cpu().numpy() for x in (history, lengths, states)]
        if graph:
            captured.replay()
        else:
            out = step()
        tokens, logprobs = (x.cpu().numpy() for x in out)
        allowed = np.stack([model.allowed(vocab, table, accepting, end, k) for k in now[2]])
        x, _ = model.adjusted(values.float().numpy(), np.float32, now[0], now[1], np.full(rows, len(prompt)), np.full(rows, 1.2, np.float32), None,
                              np.full(rows, 0.3, np.float32), mask=model.packed(allowed))
        for r in range(rows):
            v, lp, gap = model.choice(x[r], u[r], np.float32(0.9), 9, np.float32(0.97))
            assert tokens[r] == v or gap < 1e-12
            assert abs(logprobs[r] - lp) <= model.logprob_bound(lp, len(vocab))
        done |= tokens == end
    assert done.any()
    final = [x.cpu().numpy() for x in (history, lengths, states)]
    for r in range(rows):
        ids = final[0][r, len(prompt):final[1][r]]
        text = tok.decode(ids[ids != end].astype(np.uint32))
        assert model.walk(table, 0, text) == final[2][r] >= 0
        if end in ids:
            assert accepting[final[2][r]] and text.endswith(b".")
    for h in (g, s, tok):
        h.destroy()


def test_c_entry_points(engine, torch):
    g = TokenGrammar(engine, [b"a", b"b"], np.full((1, 256), -1), [0])
    L, t = _lib.lib(), torch.zeros(8, dtype=torch.int32, device="cuda")
    bad = lambda status: _lib.STATUS[status] == "BAD_ARG"  # noqa: E731
    assert bad(L.b200bpe_grammar_mask(g._h, None, 1, t.data_ptr(), 1, None)) and bad(L.b200bpe_grammar_mask(g._h, t.data_ptr(), 1, None, 1, None))
    assert bad(L.b200bpe_grammar_mask(g._h, t.data_ptr(), 2, t.data_ptr(), 0, None)) and bad(L.b200bpe_grammar_mask(g._h, t.data_ptr(), 1 << 28, t.data_ptr(), 1, None))
    assert bad(L.b200bpe_grammar_advance(g._h, t.data_ptr(), t.data_ptr(), 1, t.data_ptr(), t.data_ptr(), 1, 1, None, None, None))
    assert bad(L.b200bpe_grammar_mask(g._h, t.data_ptr() + 2, 1, t.data_ptr(), 1, None)) and bad(L.b200bpe_grammar_mask(g._h, t.data_ptr(), 1, t.data_ptr() + 1, 1, None))
    assert bad(L.b200bpe_grammar_advance(g._h, t.data_ptr(), t.data_ptr() + 2, 1, t.data_ptr(), None, 0, 0, None, None, None))
    assert L.b200bpe_grammar_mask(g._h, None, 0, None, 0, None) == 0
    g.destroy()


def test_masks_of_all_states_ahead(engine, torch):
    """A grammar's masks made once, rows of a batch picked from them by state."""
    rng = np.random.default_rng(4)
    vocab = _vocabulary(rng, 900)
    table, accepting = _automaton(rng, 60)
    g, s = TokenGrammar(engine, vocab, table, accepting, 899), TokenSampler(engine, 900)
    every = g.allowedTokens(torch.arange(60, dtype=torch.int32, device="cuda"))
    states = torch.from_numpy(rng.integers(-1, 61, 40).astype(np.int32)).cuda()
    logits, u = torch.randn(40, 900, device="cuda"), torch.rand(40, device="cuda")
    direct, by_state = s.sample(logits, u, mask=g.allowedTokens(states)), s.sample(logits, u, mask=every, maskRows=states)
    assert torch.equal(direct[0], by_state[0]) and torch.equal(direct[1], by_state[1])
    ahead = g.advance(states, direct[0]).cpu().numpy()
    for k, t, to in zip(states.cpu().numpy(), direct[0].cpu().numpy(), ahead):
        ok = model.allowed(vocab, table, accepting, 899, k)
        assert (t == -1 and not ok.any() and to == k) or (ok[t] and to >= 0)
    g.destroy()
    s.destroy()
