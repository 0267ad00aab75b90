"""The next token in plain numpy: adjusted logits, the choice of a token, a byte automaton over a vocabulary (not collected)."""
import math

import numpy as np

HALF_STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def adjusted(logits, kind, history=None, lengths=None, prompt=None, repetition=None, presence=None, frequency=None, bias_tokens=None, biases=None,
             mask=None, mask_rows=None):
    """(x, bound) of every row: x in `kind`; bound, in 64 bits, what steps rounded to 32 bits may be off (each by half a step of its result, which
    later steps, sums all of them, pass on as it is)."""
    rows, vocab = logits.shape
    x = logits.astype(kind)
    bound = np.zeros((rows, vocab))
    with np.errstate(all="ignore"):
        for r in range(rows):
            if history is not None:
                cap = history.shape[1]
                n = min(int(lengths[r]) & 0xFFFFFFFF, cap)
                p = 0 if prompt is None else int(prompt[r])
                every = [int(t) for t in history[r, :n]]
                rep = kind(1 if repetition is None else repetition[r])
                fre = kind(0 if frequency is None else frequency[r])
                pre = kind(0 if presence is None else presence[r])
                for v in sorted({t for t in every if 0 <= t < vocab}):
                    c = sum(t == v for t in every[p:])
                    if rep != 1:
                        x[r, v] = x[r, v] / rep if x[r, v] > 0 else x[r, v] * rep
                        bound[r, v] += abs(x[r, v])
                    if c:
                        by = fre * kind(c)
                        bound[r, v] += abs(by)
                        x[r, v] = x[r, v] - by
                        bound[r, v] += abs(x[r, v])
                        x[r, v] = x[r, v] - pre
                        bound[r, v] += abs(x[r, v])
            if bias_tokens is not None:
                for v, b in zip(bias_tokens[r], biases[r]):
                    if 0 <= v < vocab:
                        x[r, v] = x[r, v] + kind(b)
                        bound[r, v] += abs(x[r, v])
            if mask is not None:
                k = r if mask_rows is None else int(mask_rows[r])
                if not 0 <= k < len(mask):
                    x[r] = -np.inf
                else:
                    bits = np.unpackbits(np.ascontiguousarray(mask[k]).view(np.uint8), bitorder="little")[:vocab]
                    x[r, bits == 0] = -np.inf
    return x, bound * 2.0 ** -24


def choice(x, u=None, t=1.0, k=0, p=1.0, m=0.0):
    """(token, logprob, gap) of one row, in 64 bits; gap: how near, as a share of the weights, another choice was."""
    x = np.where(np.isnan(x), -np.inf, x).astype(np.float64)
    if not (x > -np.inf).any():
        return -1, -math.inf, 1.0
    best = x.max()
    greedy = u is None or not t >= 2.0 ** -16
    t = 1.0 if greedy else min(float(t), 3.4e38)
    with np.errstate(all="ignore"):
        y = np.where(x == best, 0.0, (x - best) / t)
    w = np.exp(y)
    total = math.fsum(w)
    if greedy:
        v = int(np.argmax(x))
        return v, y[v] - math.log(total), 1.0
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    gap = 1.0
    if k:
        order = order[:k]
    if p < 1:
        before = np.concatenate([[0], np.cumsum(w[order])])
        enough = float(p) * before[-1]
        keep = max(1, int(np.sum(before[:-1] < enough)))
        if enough > 0:
            gap = min(gap, np.abs(before[1:-1] - enough).min(initial=1.0) / total)
        order = order[:keep]
    if m > 0:
        order = order[y[order] >= math.log(min(m, 1.0))]
    kept = np.sort(order)
    run = np.cumsum(w[kept])
    u = float(u)
    u = 0.0 if not u > 0 else min(u, 1.0)
    at = min(int(np.searchsorted(run, u * run[-1], side="right")), len(kept) - 1)
    gap = min(gap, np.abs(run - u * run[-1])[:-1].min(initial=1.0) / total)
    while w[kept[at]] == 0:
        at -= 1
    v = int(kept[at])
    return v, y[v] - math.log(total), gap


def logprob_bound(logprob, vocab):
    """What a logprob may be off: weights in 32 bits, from a difference, a product and a factor of 2^-24 each (in the exponent, so times |ln w|) and an
    exponential of 2^-22, summed exactly; the weighted mean of |ln w| is the entropy less ln of the sum, so at most ln of the vocabulary's size;
    then a rounding to 32 bits, and one of the result's parts."""
    return 2.0 ** -22 + 3 * 2.0 ** -24 * math.log(vocab + 1) + 2.0 ** -23 + 2.0 ** -23 * abs(logprob)


def walk(table, state, text):
    for b in text:
        if not 0 <= state < len(table):
            return -1
        state = int(table[state][b])
    return state if 0 <= state < len(table) else -1


def allowed(entries, table, accepting, end, state):
    if not 0 <= state < len(table):
        return np.zeros(len(entries), bool)
    return np.array([bool(accepting[state]) if t == end else len(e) > 0 and walk(table, state, e) >= 0 for t, e in enumerate(entries)])


def packed(bits):
    """Rows of truth values as rows of mask words."""
    bits = np.atleast_2d(np.asarray(bits, bool))
    padded = np.zeros((bits.shape[0], (bits.shape[1] + 31) // 32 * 32), bool)
    padded[:, :bits.shape[1]] = bits
    return np.packbits(padded, axis=1, bitorder="little").view(np.int32)


def literals(words):
    """An automaton of exactly these byte strings."""
    table, accepting = [[-1] * 256], [0]
    for w in words:
        at = 0
        for b in w:
            if table[at][b] < 0:
                table[at][b] = len(table)
                table.append([-1] * 256)
                accepting.append(0)
            at = table[at][b]
        accepting[at] = 1
    return np.array(table), np.array(accepting)
