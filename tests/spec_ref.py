"""Speculative decoding's operators in 64 bits, as the tests' reference: attention of a tree of
drafted tokens over a cache, and the verification of its tokens."""
from __future__ import annotations

import numpy as np


def make_tree(rng, n, width):
    """Parents of a random tree of n nodes with at most `width` children each (1: a chain)."""
    parent, room = [-1], [width]
    for i in range(1, n):
        p = i - 1 if width == 1 else int(rng.choice([j for j in range(i) if room[j]]))
        parent.append(p)
        room[p] -= 1
        room.append(width)
    return np.array(parent, np.int32)


def ancestors(parent):
    n = len(parent)
    a = np.zeros((n, n), bool)
    for i in range(n):
        if i:
            a[i] = a[parent[i]]
        a[i, i] = True
    return a


def mask_words(see):
    """Rows of truth values as 64-bit words, bit j % 64 of word j // 64 for column j."""
    n, m = see.shape
    words = (m + 63) // 64
    out = np.zeros((n, words), np.uint64)
    for j in range(m):
        out[:, j // 64] |= see[:, j].astype(np.uint64) << np.uint64(j % 64)
    return out


def target(logits, temperature, top_p):
    """The distribution that sample_logits draws from, in 64 bits."""
    x = np.asarray(logits, np.float64).copy()
    x[np.isnan(x)] = -np.inf
    if temperature <= 0:
        p = np.zeros(len(x))
        p[int(np.argmax(x))] = 1.0
        return p
    with np.errstate(invalid="ignore"):
        d = (x - x.max()) / float(np.float32(temperature))
    d[x == x.max()] = 0.0
    p = np.exp(d)
    p /= p.sum()
    if top_p < 1:
        order = np.argsort(-x, kind="stable")
        before = np.cumsum(p[order]) - p[order]
        keep = before < float(np.float32(top_p))
        keep[0] = True
        p[order[~keep]] = 0.0
        p /= p.sum()
    return p


def verify(logits, tokens, parent, draft, temperature, top_p, draws):
    """(path, next token, probs): the walk as the header describes it, one node after the other."""
    n, vocab = logits.shape
    draws = np.asarray(draws, np.float64)
    rows = [target(logits[i], temperature, top_p) for i in range(n)]
    up = [int(p) if i and 0 <= p < i else -1 for i, p in enumerate(parent)]
    probs = np.zeros(n)
    for i in range(1, n):
        if up[i] >= 0 and 0 <= tokens[i] < vocab:
            probs[i] = rows[up[i]][tokens[i]]
    path, at = [0], 0
    while True:
        r = rows[at].copy()
        q = None if draft is None else np.asarray(draft[at], np.float64)
        took = -1
        for c in range(at + 1, n):
            if up[c] != at:
                continue
            x = int(tokens[c])
            known = 0 <= x < vocab
            have = r[x] if known else 0.0
            ask = (1.0 if q is None else q[x]) if known else 0.0
            if have > 0 and draws[c] * ask < have:
                took = c
                break
            if q is not None:
                r = np.maximum(r - q, 0.0)
            elif known:
                r[x] = 0.0
            if r.sum() > 0:
                r = r / r.sum()
        if took < 0:
            break
        path.append(took)
        at = took
    w = r if r.sum() > 0 else rows[at]
    run = np.cumsum(w)
    token = min(int(np.searchsorted(run, draws[0] * run[-1], side="right")), int(np.flatnonzero(w > 0)[-1]))
    if temperature <= 0:
        token = int(np.argmax(rows[at]))
    probs[0] = rows[at][token]
    return path, token, probs
