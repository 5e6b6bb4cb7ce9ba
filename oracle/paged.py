"""Attention over a paged K/V cache in float64: the definition, token by token, with the terms
of its error bounds. The per-row arithmetic (norms, RoPE) is gemma4_150/reference.py:38-55's."""
from __future__ import annotations

import numpy as np


def rms(x, eps):
    return x / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps)


def rotate(x, c, s):
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return np.concatenate([a * c - b * s, b * c + a * s], -1)


def prep(x, gain, c, s, eps=1e-6):
    """rms(x) * gain (gain None: x as it is), rotated by one table row (None: not)."""
    x = np.asarray(x, np.float64)
    if gain is not None:
        x = rms(x, eps) * np.asarray(gain, np.float64)
    return x if c is None else rotate(x, np.asarray(c, np.float64), np.asarray(s, np.float64))


def keys_of(table, b, p, page_size, n_pages, window):
    """Attended positions of a token at p of sequence b, and their rows in the pool."""
    if p < 0:
        return np.zeros(0, np.int64), np.zeros(0, np.int64)
    t = np.arange(max(0, p + 1 - window) if window else 0, p + 1)
    page = table[b, t // page_size].astype(np.int64)
    there = (page >= 0) & (page < n_pages)
    return t[there], (page * page_size + t % page_size)[there]


def attend(q, tokens, k_pages, v_pages, table, *, q_gain, cos, sin, window=0, scale=1.0, eps=1e-6):
    """q [n][nH][hd] raw; tokens[i] = (sequence, position) or None (a row of nobody: NaN).

    Returns out, A = sum_t w_t |v_t| per output, and S = the largest sum_i |q_i k_i| * scale of
    the token's heads: a relative error e of every q (or k) element moves a score by at most e S."""
    n, nH, hd = q.shape
    n_pages, ps, kvH, _ = k_pages.shape
    kr, vr = (np.asarray(x).reshape(-1, kvH, hd) for x in (k_pages, v_pages))
    out = np.full((n, nH, hd), np.nan)
    A, S = np.zeros((n, nH, hd)), np.zeros((n, nH, 1))
    G = nH // kvH
    for i, tok in enumerate(tokens):
        if tok is None:
            continue
        out[i] = 0.0
        b, p = tok
        _, rows = keys_of(table, b, p, ps, n_pages, window)
        if not len(rows):
            continue
        x = prep(q[i], q_gain, None if cos is None else cos[p], None if sin is None else sin[p], eps) * scale
        for kh in range(kvH):
            k, v = kr[rows, kh].astype(np.float64), vr[rows, kh].astype(np.float64)
            h = slice(kh * G, (kh + 1) * G)
            s = x[h] @ k.T
            w = np.exp(s - s.max(-1, keepdims=True))
            w /= w.sum(-1, keepdims=True)
            out[i, h] = w @ v
            A[i, h] = w @ np.abs(v)
            S[i, h] = (np.abs(x[h]) @ np.abs(k).T).max(-1, keepdims=True)
    return out, A, S
