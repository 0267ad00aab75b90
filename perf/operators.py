"""What turns a model's logits into the next token of a vocabulary, as cases that can be timed: the tokens that a grammar
allows (a byte automaton walked over the vocabulary's entries), penalties, biases and masks on logits, the choice of a
token, and the step of every request's automaton and history.

`own` false: plain torch operations.  `own` true: the calls that a user makes of gpu_bpe_b200 (TokenSampler, TokenGrammar).

Definitions, for a row of logits l and a token v:
  adjusted    x = l;  where v occurs in the row's history: x / repetition (x > 0) or x * repetition;
              x - frequency * (occurrences behind the prompt);  x - presence where there are any;  + bias;  -inf where the
              mask's bit is 0.  The choice works on x held in 32 bits.
  chosen      w = exp((x - max x) / temperature);  the top_k largest x (ties: lowest index);  of those the shortest run, from
              the largest on, with at least top_p of their weight;  of those the ones with w >= min_p;  then the first in
              index order at which the running sum of w passes uniform * sum.  Temperature 0: the largest x.
  logprob     of the chosen token under all w of the row (temperature 0: at temperature 1).
Vocabulary sizes are the repository's own (4,096, 32,256 and 64,256 entries) and generic ones; logits are normal with a few
dozen strong candidates a row, as a model's are.
"""
import functools
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LARGEST = 256 * 131072        # logits of the largest inputs
DEAD = -1                     # transition to nowhere
LONGEST = 24                  # bytes of the longest vocabulary entry


def listed():
    return [
        # one request, decoded greedily with a repetition penalty: latency only
        {"name": "sample_one", "op": "sample", "rows": 1, "vocab": 32256, "dtype": "bf16", "history": 200, "bias": 0, "mask": False, "mode": "greedy"},
        # a chat server's step: every request with its own settings, some under a grammar
        {"name": "sample_chat", "op": "sample", "rows": 32, "vocab": 64256, "dtype": "f16", "history": 700, "bias": 16, "mask": True, "mode": "mixed"},
        # a full batch with long histories
        {"name": "sample_batch", "op": "sample", "rows": 256, "vocab": 131072, "dtype": "bf16", "history": 2000, "bias": 0, "mask": False, "mode": "mixed"},
        # rollouts: the whole distribution at temperature 1, logits in 32 bits
        {"name": "sample_pure", "op": "sample", "rows": 128, "vocab": 262144, "dtype": "f32", "history": 0, "bias": 0, "mask": False, "mode": "pure"},
        # adjusted logits of one request, for a caller who chooses by himself
        {"name": "adjust_one", "op": "adjust", "rows": 1, "vocab": 32256, "dtype": "f32", "history": 333, "bias": 3, "mask": True, "pad": 0},
        # odd vocabulary, rows padded by the model
        {"name": "adjust_odd", "op": "adjust", "rows": 61, "vocab": 50021, "dtype": "bf16", "history": 517, "bias": 5, "mask": True, "pad": 27},
        # a full batch in 32 bits
        {"name": "adjust_batch", "op": "adjust", "rows": 256, "vocab": 131072, "dtype": "f32", "history": 1500, "bias": 8, "mask": True, "pad": 0},
        # the allowed tokens of one request's next step
        {"name": "mask_one", "op": "mask", "rows": 1, "vocab": 32256, "fields": 6},
        # of a batch, every request at its own place in the grammar
        {"name": "mask_batch", "op": "mask", "rows": 256, "vocab": 64256, "fields": 12},
        # of every state of a grammar, ahead of serving
        {"name": "mask_states", "op": "mask", "rows": 1500, "vocab": 32256, "fields": 80},
        # the step after the choice, for one request and for a large batch
        {"name": "advance_one", "op": "advance", "rows": 1, "vocab": 32256, "fields": 6},
        {"name": "advance_batch", "op": "advance", "rows": 2048, "vocab": 64256, "fields": 40},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["sample", "sample", "sample", "adjust", "adjust", "mask", "mask", "advance"])
    if op == "advance":
        return {"op": op, "rows": _log(rng, 1, 2048), "vocab": _log(rng, 300, 64256), "fields": rng.randint(1, 60)}
    if op == "mask":
        vocab = _log(rng, 300, 64256)
        return {"op": op, "rows": _log(rng, 1, min(1500, 1500 * 32256 // vocab)), "vocab": vocab, "fields": rng.randint(1, 80)}
    vocab = _log(rng, 300, 262144)
    rows = _log(rng, 1, min(512, LARGEST // vocab))
    c = {"op": op, "rows": rows, "vocab": vocab, "dtype": rng.choice(["f32", "f16", "bf16", "bf16"]), "history": rng.choice([0, _log(rng, 1, 4000)]),
         "bias": rng.choice([0, 0, rng.randint(1, 64)]), "mask": rng.random() < 0.5}
    if op == "adjust":
        return dict(c, pad=rng.choice([0, 0, rng.randint(1, 64)]))
    return dict(c, mode=rng.choice(["greedy", "mixed", "mixed", "nucleus", "pure"]))


# ── inputs ──

@functools.lru_cache(None)
def _vocabulary(size):
    """Entries as a trainer makes them: the bytes, then pairs of earlier entries, letters and spaces the most frequent.  The last id ends
    a text and has no bytes."""
    rng = random.Random(11)
    letters = b"etaoinshrdlcumwfgypbvk,. etaoinsr \"0123456789TASIBCMP:{}[]-_\n"
    entries, seen = [bytes([i]) for i in range(256)], set()
    base = [bytes([b]) for b in letters] + ["é".encode(), "ü".encode(), "я".encode(), "你".encode()]
    pool = list(base)
    while len(entries) < size - 1:
        e = pool[int(len(pool) * rng.random() ** 6)] + pool[int(len(pool) * rng.random() ** 8)]
        if len(e) <= LONGEST and e not in seen:
            seen.add(e)
            entries.append(e)
            pool.append(e)
    return entries + [b""]


def _grammar(seed, fields):
    """An object with `fields` keys in order, each a string, a number or a truth value, as a byte automaton: (transitions, accepting)."""
    rng = random.Random(seed)
    table = [[DEAD] * 256]

    def new():
        table.append([DEAD] * 256)
        return len(table) - 1

    def text(at, s):
        for b in s:
            if table[at][b] == DEAD:
                table[at][b] = new()
            at = table[at][b]
        return at

    at = text(0, b"{")
    for k in range(fields):
        at = text(at, ("\"%s\": " % "".join(rng.choice("abcdefghiklmnoprstuvw_") for _ in range(rng.randint(2, 9)))).encode())
        kind = rng.choice(["string", "string", "number", "bool"])
        if kind == "string":
            body, escape, last = text(at, b"\""), new(), new()
            more = [new(), new(), new()]
            for b in range(0x20, 0x80):
                table[body][b] = body
            table[body][0x5C], table[body][0x22] = escape, last
            for b in b"\"\\/bfnrt":
                table[escape][b] = body
            for lead, n in ((range(0xC2, 0xE0), 0), (range(0xE1, 0xEC), 1), (range(0xF1, 0xF4), 2)):
                for b in lead:
                    table[body][b] = more[n]
            for n in range(3):
                for b in range(0x80, 0xC0):
                    table[more[n]][b] = more[n - 1] if n else body
            at = last
        elif kind == "number":
            whole, point, part = new(), new(), new()
            for b in b"0123456789":
                table[at][b] = table[whole][b] = whole
                table[point][b] = table[part][b] = part
            table[whole][0x2E] = point
            joined = new()
            for s in (whole, part):
                table[s][0x20] = joined      # a space ends a number
            at = joined
        else:
            joined = new()
            for word in (b"true", b"false"):
                table[text(at, word[:-1])][word[-1]] = joined
            at = joined
        at = text(at, b", " if k + 1 < fields else b"}")
    accepting = [False] * len(table)
    accepting[at] = True
    return np.array(table, np.int32), np.array(accepting, np.uint8)


@functools.lru_cache(None)
def _engine():
    from gpu_bpe_b200 import BPEEngine
    return BPEEngine(0).init()


@functools.lru_cache(None)
def _sampler(vocab):
    from gpu_bpe_b200 import TokenSampler
    return TokenSampler(_engine(), vocab)


def _token_grammar(entries, table, accepting):
    from gpu_bpe_b200 import TokenGrammar
    return TokenGrammar(_engine(), entries, table, accepting, endToken=len(entries) - 1)


class _State:
    pass


def _logits(g, rows, vocab, pad, dtype):
    x = torch.randn(rows, vocab + pad, generator=g, device="cuda") * 2.2
    at = torch.randint(0, vocab, (rows, 24), generator=g, device="cuda")
    x.scatter_add_(1, at, torch.randn(rows, 24, generator=g, device="cuda").abs() * 4 + 3)
    return x.to(dtype)


def prepare(case, seed):
    s = _State()
    s.case, rows, vocab = case, case["rows"], case["vocab"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    uniform = lambda *size: torch.rand(*size, generator=g, device="cuda")  # noqa: E731
    integers = lambda lo, hi, *size: torch.randint(lo, hi, size, generator=g, device="cuda", dtype=torch.int32)  # noqa: E731
    if case["op"] in ("mask", "advance"):
        entries = _vocabulary(vocab)
        table, accepting = _grammar(seed, case["fields"])
        s.grammar = _token_grammar(entries, table, accepting) if own else None
        s.states = integers(0, table.shape[0], rows)
        if case["op"] == "advance":
            s.tokens = integers(0, vocab, rows)
            s.history, s.lengths = integers(0, vocab, rows, 64), integers(0, 64, rows)
        lengths = np.array([len(e) for e in entries])
        padded = np.zeros((vocab, LONGEST), np.uint8)
        padded[np.arange(LONGEST) < lengths[:, None]] = np.frombuffer(b"".join(entries), np.uint8)
        s.bytes, s.byte_counts = torch.from_numpy(padded).cuda().long(), torch.from_numpy(lengths).cuda()
        s.table, s.accepting = torch.from_numpy(table).cuda().long(), torch.from_numpy(accepting).cuda().bool()
        return s
    s.sampler = _sampler(vocab) if own else None
    s.logits = _logits(g, rows, vocab, case.get("pad", 0), DTYPES[case["dtype"]])
    s.adjust = a = {}
    if case["history"]:
        n = case["history"]
        a["history"] = (uniform(rows, n) ** 3 * vocab).int().clamp_(0, vocab - 1)
        a["history"][:, ::5] = s.logits[:, :vocab].float().topk(min(16, vocab)).indices.int()[:, :1]
        a["lengths"] = integers(n // 2, n + 1, rows)
        a["promptLengths"] = (a["lengths"] * uniform(rows)).int()
        a["repetition"] = 1 + 0.3 * uniform(rows) * (uniform(rows) < 0.7)
        a["presence"] = 0.5 * uniform(rows) * (uniform(rows) < 0.5)
        a["frequency"] = 0.2 * uniform(rows) * (uniform(rows) < 0.5)
    if case["bias"]:
        a["biasTokens"] = torch.argsort(uniform(rows, min(vocab, 4096)), dim=1)[:, :case["bias"]].int()
        a["biasTokens"][uniform(rows, a["biasTokens"].shape[1]) < 0.3] = -1
        a["biases"] = torch.randn(a["biasTokens"].shape, generator=g, device="cuda") * 4
    if case["mask"]:
        words = (vocab + 31) // 32
        bits = torch.randint(-2**31, 2**31, (rows, words), generator=g, device="cuda").int()
        tight = torch.randint(-2**31, 2**31, (3, rows, words), generator=g, device="cuda").int()
        some = uniform(rows, 1) < 0.5
        a["mask"] = torch.where(some, bits & tight[0] & tight[1] & tight[2], bits | tight[0])
        if vocab % 32:
            a["mask"][:, -1] &= (1 << vocab % 32) - 1
    if case["op"] == "adjust":
        s.out = torch.empty_like(s.logits)
        return s
    s.choice = c = {}
    c["uniform"] = uniform(rows)
    mode = case["mode"]
    c["temperature"] = torch.zeros(rows, device="cuda") if mode == "greedy" else 0.6 + 0.8 * uniform(rows)
    if mode == "pure":
        c["temperature"] = torch.ones(rows, device="cuda")
    if mode == "mixed":
        c["temperature"][uniform(rows) < 0.15] = 0
        c["topK"] = torch.tensor([0, 1, 20, 50, 400], dtype=torch.int32, device="cuda")[integers(0, 5, rows).long()]
        c["minP"] = torch.tensor([0, 0, 0.02, 0.1], device="cuda")[integers(0, 4, rows).long()]
    if mode in ("mixed", "nucleus"):
        c["topP"] = torch.tensor([1, 0.95, 0.9, 0.7], device="cuda")[integers(0 if mode == "mixed" else 1, 4, rows).long()]
    return s


# ── the plain forms ──

def _adjusted(logits, vocab, history=None, lengths=None, promptLengths=None, repetition=None, presence=None, frequency=None, biasTokens=None,
              biases=None, mask=None):
    rows = logits.shape[0]
    x = logits[:, :vocab].float()
    if history is not None:
        at = torch.arange(history.shape[1], device=x.device)[None]
        seen = torch.zeros(rows, vocab, dtype=torch.int32, device=x.device).scatter_add_(1, history.long(), (at < lengths[:, None]).int())
        out = torch.zeros_like(seen).scatter_add_(1, history.long(), ((at < lengths[:, None]) & (at >= promptLengths[:, None])).int())
        r = repetition[:, None]
        x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
        x = x - frequency[:, None] * out.float()
        x = x - presence[:, None] * (out > 0).float()
    if biasTokens is not None:
        used = biasTokens >= 0
        x = x.scatter_add(1, biasTokens.clamp(min=0).long(), torch.where(used, biases, torch.zeros_like(biases)))
    if mask is not None:
        v = torch.arange(vocab, device=x.device)
        x = torch.where((mask[:, v >> 5] >> (v & 31)[None].int()) & 1 != 0, x, -math.inf)
    return x


def _chosen(x, uniform, temperature, topK=None, topP=None, minP=None):
    rows, vocab = x.shape
    d = x.double()
    best = d.max(1, keepdim=True).values
    greedy = temperature == 0
    t = torch.where(greedy, torch.ones_like(temperature), temperature).double()[:, None]
    y = (d - best) / t
    w = y.exp()
    all_of_it = w.sum(1, keepdim=True)
    if topK is not None or topP is not None or minP is not None:
        order = x.sort(dim=1, descending=True, stable=True).indices
        ws = w.gather(1, order)
        if topK is not None:
            k = torch.where(topK > 0, topK, vocab)[:, None]
            ws = torch.where(torch.arange(vocab, device=x.device)[None] < k, ws, 0.0)
        if topP is not None:
            run = ws.cumsum(1)
            before = torch.cat([torch.zeros_like(run[:, :1]), run[:, :-1]], 1)
            ws = torch.where((before < topP.double()[:, None] * run[:, -1:]) | (topP >= 1)[:, None], ws, 0.0)
        if minP is not None:
            ws = torch.where(y.gather(1, order) >= minP.double()[:, None].log(), ws, 0.0)
        kept = torch.zeros_like(w).scatter_(1, order, ws)
    else:
        kept = w
    run = kept.cumsum(1)
    token = (run <= uniform.double()[:, None] * run[:, -1:]).sum(1)
    index = torch.arange(vocab, device=x.device)[None]
    first = torch.where(d == best, index, vocab).amin(1)
    token = torch.where(greedy, first, token)
    logprob = y.gather(1, token[:, None])[:, 0] - all_of_it[:, 0].log()
    return token.int(), logprob.float()


def _walk(table, states, text, counts):
    """The automaton's state behind `text` [.., LONGEST] of `counts` bytes, from `states`; DEAD once there is no transition."""
    for k in range(LONGEST):
        step = table[states.clamp(min=0), text[..., k]]
        states = torch.where((k < counts) & (states >= 0), step, states)
    return states


def _allowed(states, table, accepting, text, counts):
    rows, vocab = states.shape[0], text.shape[0]
    end = _walk(table, states.long()[:, None].expand(rows, vocab), text[None].expand(rows, vocab, LONGEST), counts[None])
    ok = (end >= 0) & (counts > 0)[None]
    ok[:, -1] = accepting[states.long()]
    words = (vocab + 31) // 32
    bits = torch.zeros(rows, words * 32, dtype=torch.int64, device=states.device)
    bits[:, :vocab] = ok.long()
    return (bits.view(rows, words, 32) << torch.arange(32, device=states.device)).sum(2).int()


def _advanced(states, tokens, table, accepting, text, counts, history, lengths):
    s, t = states.long(), tokens.long()
    end = _walk(table, s, text[t], counts[t])
    last = t == text.shape[0] - 1
    end = torch.where(last, torch.where(accepting[s], s, DEAD), end)
    return end.int(), history.scatter(1, lengths.long()[:, None], tokens[:, None]), lengths + 1


def run(state):
    s, op = state, state.case["op"]
    if own:
        if op == "mask":
            return {"mask": s.grammar.allowedTokens(s.states)}
        if op == "advance":
            states, lengths = s.grammar.advance(s.states, s.tokens, history=s.history, lengths=s.lengths)
            return {"states": states, "history": s.history, "lengths": lengths}
        if op == "adjust":
            return {"logits": s.sampler.adjustLogits(s.logits, out=s.out, **s.adjust)[:, :s.case["vocab"]]}
        tokens, logprobs = s.sampler.sample(s.logits, **s.choice, **s.adjust)
        return {"tokens": tokens, "logprobs": logprobs}
    if op == "mask":
        return {"mask": _allowed(s.states, s.table, s.accepting, s.bytes, s.byte_counts)}
    if op == "advance":
        states, history, lengths = _advanced(s.states, s.tokens, s.table, s.accepting, s.bytes, s.byte_counts, s.history, s.lengths)
        return {"states": states, "history": history, "lengths": lengths}
    x = _adjusted(s.logits, s.case["vocab"], **s.adjust)
    if op == "adjust":
        return {"logits": x.to(s.logits.dtype)}
    tokens, logprobs = _chosen(x, **s.choice)
    return {"tokens": tokens, "logprobs": logprobs}


def work(case):
    """Logits, the used part of the histories (three quarters of their room), biases and masks read once, results written once; about ten
    operations a logit for a choice and four for an adjustment.  Masks: the entries' bytes and the transitions (a byte each) read once.
    Steps: an entry's bytes and a transition for each of them."""
    rows, vocab = case["rows"], case["vocab"]
    if case["op"] in ("mask", "advance"):
        text = sum(map(len, _vocabulary(vocab)))
        if case["op"] == "advance":
            return {"bytes": rows * (4 * 6 + 5 * text / vocab), "flops": 0}
        return {"bytes": text + 256 * 17 * case["fields"] + 4 * rows + rows * vocab / 8, "flops": 0}
    size = 4 if case["dtype"] == "f32" else 2
    n = rows * vocab
    read = n * size + rows * (3 * case["history"] + 20 * (case["history"] > 0)) + 8 * rows * case["bias"] + (n / 8 if case["mask"] else 0)
    return {"bytes": read + (n * size if case["op"] == "adjust" else 24 * rows), "flops": n * (4 if case["op"] == "adjust" else 10)}


# ── in 64 bits ──

def _exact_row(l, a, r, precision):
    """Adjusted logits of row r, in `precision`."""
    vocab = l.size
    x = l.astype(precision)
    if "history" in a:
        n, p = int(a["lengths"][r]), int(a["promptLengths"][r])
        h = a["history"][r, :n]
        seen = np.bincount(h, minlength=vocab) > 0
        out = np.bincount(h[p:], minlength=vocab)
        rep, pres, freq = (precision(a[k][r]) for k in ("repetition", "presence", "frequency"))
        x[seen] = np.where(x[seen] > 0, x[seen] / rep, x[seen] * rep)
        x -= freq * out.astype(precision)
        x[out > 0] -= pres
    if "biasTokens" in a:
        for v, b in zip(a["biasTokens"][r], a["biases"][r]):
            if v >= 0:
                x[v] += precision(b)
    if "mask" in a:
        bits = np.unpackbits(np.ascontiguousarray(a["mask"][r]).view(np.uint8), bitorder="little")[:vocab]
        x[bits == 0] = -np.inf
    return x


def exact(case, seed):
    if case["op"] in ("mask", "advance"):
        return None
    s = prepare(case, seed)
    vocab = case["vocab"]
    logits = s.logits[:, :vocab].float().cpu().numpy()
    a = {k: v.cpu().numpy() for k, v in s.adjust.items()}
    if case["op"] == "adjust":
        return {"logits": np.stack([_exact_row(logits[r], a, r, np.float64) for r in range(case["rows"])])}
    c = {k: v.cpu().numpy() for k, v in s.choice.items()}
    logprobs = np.empty(case["rows"], np.float64)
    for r in range(case["rows"]):
        x = _exact_row(logits[r], a, r, np.float32).astype(np.float64)
        t = float(c["temperature"][r])
        y = (x - x.max()) / (t or 1.0)
        w = np.exp(y)
        if t == 0:
            v = int(x.argmax())
        else:
            order = np.argsort(-x, kind="stable")
            k = int(c["topK"][r]) if "topK" in c else 0
            if k:
                order = order[:k]
            p = float(c["topP"][r]) if "topP" in c else 1.0
            if p < 1:
                sums = np.cumsum(w[order])
                order = order[:1 + int(np.sum(sums[:-1] < p * sums[-1]))]
            m = float(c["minP"][r]) if "minP" in c else 0.0
            if m > 0:
                order = order[y[order] >= math.log(m)]
            kept = np.sort(order)
            sums = np.cumsum(w[kept])
            v = int(kept[min(kept.size - 1, np.searchsorted(sums, float(c["uniform"][r]) * sums[-1], side="right"))])
        logprobs[r] = y[v] - math.log(w.sum())
    return {"tokens": None, "logprobs": logprobs}
