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


def accept(keys, cu, parents, drafts, targets, max_path):
    """path, n_path, next, kept of every sequence."""
    path, count, nxt, kept = [], [], [], []
    for b in range(len(keys)):
        n = min(cu[b + 1] - cu[b], TREE_MAX)
        p, d, t = (x[cu[b]:cu[b] + n] for x in (parents, drafts, targets))
        got = [0] if n else []
        while got and len(got) < max_path:
            child = [c for c in range(got[-1] + 1, n) if p[c] == got[-1] and d[c] == t[got[-1]]]
            if not child:
                break
            got.append(child[0])
        path.append(got + [-1] * (max_path - len(got)))
        count.append(len(got))
        nxt.append(int(t[got[-1]]) if got else -1)
        kept.append(int(keys[b] - (cu[b + 1] - cu[b]) + len(got)))
    return path, count, nxt, kept


def keep(pools, keys, cu, path, n_path, table, page_size, n_pages):
    """The pools [rows][...] with each sequence's path moved up."""
    before = [p.copy() for p in pools]
    for b in range(len(keys)):
        n = min(cu[b + 1] - cu[b], TREE_MAX)
        start = keys[b] - (cu[b + 1] - cu[b])
        last = -1
        for d in range(min(n_path[b], len(path[b]), n)):
            i = path[b][d]
            if not last < i < n:
                break
            last = i
            if start + d < 0:
                continue
            src, dst = (there(table, b, [start + x], page_size, n_pages) for x in (i, d))
            if len(src) and len(dst):
                for p, q in zip(pools, before):
                    p[dst[0]] = q[src[0]]
    return pools


def fork(pools, table, keys, parent, free, room, page_size, n_pages):
    """New table, lengths, free list and the pools [pages][rows][...]."""
    cols, n = table.shape[1], len(parent)
    ok = lambda p: 0 <= p < n_pages  # noqa: E731
    live = [0 <= p < len(keys) for p in parent]
    new = np.full((n, cols), -1, np.int64)
    length = [min(max(int(keys[p]), 0), cols * page_size) if a else 0 for p, a in zip(parent, live)]
    full, owner, todo = set(), {}, []
    for j in range(n):
        for c in range(length[j] // page_size if live[j] else 0):
            if ok(table[parent[j], c]):
                new[j, c] = table[parent[j], c]
                full.add(int(new[j, c]))
    for j in range(n):
        for c in range(length[j] // page_size, min(-(-(length[j] + room) // page_size), cols) if live[j] else 0):
            p = int(table[parent[j], c])
            if ok(p) and p not in full and owner.setdefault(p, j) == j:
                new[j, c] = p
            elif ok(p) or c * page_size >= length[j]:
                todo.append((j, c, p))
    held = full | set(owner)
    free = list(free) + sorted({int(p) for p in table.reshape(-1) if ok(p)} - held)
    pools = [p.copy() for p in pools]
    for j, c, p in todo:
        if not free:
            continue
        new[j, c] = free.pop()
        fill = length[j] - c * page_size
        if fill > 0:
            for x in pools:
                x[new[j, c], :fill] = x[p, :fill]
    return new, length, free, pools


def select(logits, scores, cap, n_out, done=None, pad=0):
    """score, parent, token of each group's n_out best, in 64 bits."""
    B, W = scores.shape
    score, parent, token = (np.full((B, n_out), x) for x in (-np.inf, -1, -1))
    for b in range(B):
        cand = []
        for w in range(W):
            at = float(scores[b, w])
            if done is not None and done[b, w]:
                cand.append((-at, w, 0, pad))
                continue
            x = np.asarray(logits[b * W + w], np.float64)
            t = np.flatnonzero(x > -np.inf)  # (not NaN either)
            x = cap * np.tanh(x[t] / cap) if cap else x[t]
            if not len(t):
                continue
            m = x.max()
            with np.errstate(invalid="ignore"):
                lp = np.where(x == m, 0.0, x - m)
            lp = lp - np.log(np.exp(lp).sum())
            order = np.lexsort((t, -np.asarray(logits[b * W + w], np.float64)[t]))[:n_out]
            cand += [(-(at + lp[i]), w, k, int(t[i])) for k, i in enumerate(order)]
        cand = sorted(c for c in cand if c[0] < np.inf)[:n_out]
        for k, c in enumerate(cand):
            score[b, k], parent[b, k], token[b, k] = -c[0], b * W + c[1], c[3]
    return score, parent, token
