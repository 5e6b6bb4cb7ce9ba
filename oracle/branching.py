"""Generation that branches over a paged cache, in float64 and python integers, token by token: drafted trees
and beams. The per-row arithmetic is oracle/paged.py's."""
from __future__ import annotations

import numpy as np

from .paged import prep

TREE_MAX = 1024


def line(parents, i):
    """Token i of a tree and its ancestors, nearest first."""
    out = [i]
    while 0 <= parents[out[-1]] < out[-1]:
        out.append(int(parents[out[-1]]))
    return out


def packed(keys, cu, n_tokens):
    """(sequence, index in its tree) of every packed row, None for rows of nobody."""
    who = [None] * n_tokens
    for b in range(len(keys)):
        for i in range(min(cu[b + 1] - cu[b], TREE_MAX)):
            who[cu[b] + i] = (b, i)
    return who


def there(table, b, t, page_size, n_pages):
    """Of rows t of sequence b those whose pages are there: their rows in the pool."""
    t = np.asarray(t, np.int64)
    page = table[b, t // page_size].astype(np.int64)
    ok = (page >= 0) & (page < n_pages)
    return (page * page_size + t % page_size)[ok]


def attended(parents, start, i, window):
    """Rows of its sequence that token i of a tree at row `start` attends, and its position."""
    up = line(parents, i)
    pos = start + len(up) - 1
    hist = range(max(0, pos + 1 - window) if window else 0, max(start, 0))
    tree = [start + j for j in (up[:window] if window else up) if start + j >= 0]
    return list(hist) + sorted(tree), pos


def attend_tree(q, keys, cu, parents, k_pages, v_pages, table, *, q_gain, cos, sin, window=0, scale=1.0, eps=1e-6):
    """As oracle.paged.attend: out, A = sum w |v|, S = the largest sum |q k| * scale, NaN for rows of nobody."""
    n, nH, hd = q.shape
    n_pages, ps, kvH, _ = k_pages.shape
    kr, vr = (np.asarray(x).reshape(-1, kvH, hd) for x in (k_pages, v_pages))
    out, A, S = np.full((n, nH, hd), np.nan), np.zeros((n, nH, hd)), np.zeros((n, nH, 1))
    G = nH // kvH
    for tok, who in enumerate(packed(keys, cu, n)):
        if who is None:
            continue
        b, i = who
        out[tok] = 0.0
        start = keys[b] - (cu[b + 1] - cu[b])
        if start + i < 0:
            continue
        t, pos = attended(parents[cu[b]:cu[b + 1]], start, i, window)
        rows = there(table, b, t, ps, n_pages)
        if not len(rows):
            continue
        x = prep(q[tok], q_gain, None if cos is None else cos[max(pos, 0)], None if sin is None else sin[max(pos, 0)], eps) * scale
        for kh in range(kvH):
            k, v = kr[rows, kh].astype(np.float64), vr[rows, kh].astype(np.float64)
            h = slice(kh * G, (kh + 1) * G)
            s = x[h] @ k.T
            w = np.exp(s - s.max(-1, keepdims=True))
            w /= w.sum(-1, keepdims=True)
            out[tok, h] = w @ v
            A[tok, h] = w @ np.abs(v)
            S[tok, h] = (np.abs(x[h]) @ np.abs(k).T).max(-1, keepdims=True)
    return out, A, S
