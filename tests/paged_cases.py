"""Ragged batches on a paged cache for the tests: shuffled pages, poisoned rows, error bounds."""
import numpy as np
import torch

import oracle.paged as OP
import slang_amd as sa

NH, MAX_POS = 8, 2048


def f16(x):
    return np.asarray(x, np.float32).astype(np.float16)


class Batch:
    """Sequences of keys[b] keys, the last new[b] of them this call's tokens. The pool's rows that
    no sequence attends hold NaN; `missing` pages (sequence, index) have no entry."""

    def __init__(self, keys, new, *, hd=256, kvh=2, page=16, kv=np.float16, seed=0, window=0, pad=0, missing=(), theta=1e4,
                 spare=3, extra_cols=1, nh=NH, written=True):
        r = np.random.default_rng(seed)
        self.keys, self.new, self.hd, self.kvh, self.page, self.window, self.nh = list(keys), list(new), hd, kvh, page, window, nh
        n = len(keys)
        self.cols = -(-max(1, max(keys)) // page) + extra_cols
        self.table = np.full((n, self.cols), -1, np.int32)
        count = [-(-k // page) for k in keys]
        self.n_pages = sum(count) + spare
        ids = r.permutation(self.n_pages)[:sum(count)].astype(np.int32)
        at = 0
        for b in range(n):
            self.table[b, :count[b]] = ids[at:at + count[b]]
            at += count[b]
        for j, (b, i) in enumerate(missing):
            self.table[b, i] = (-1, self.n_pages, -2 ** 31, 2 ** 31 - 1)[j % 4]
        shape = (self.n_pages, page, kvh, hd)
        self.k_pages, self.v_pages = np.full(shape, np.nan, kv), np.full(shape, np.nan, kv)
        kr, vr = self.k_pages.reshape(-1, kvh, hd), self.v_pages.reshape(-1, kvh, hd)
        for b in range(n):
            m = keys[b] - (0 if written else new[b])
            first = max(0, keys[b] - new[b] + 1 - window) if window else 0
            t, rows = OP.keys_of(self.table, b, m - 1, page, self.n_pages, 0)
            rows = rows[t >= first]
            kr[rows] = 0.4 * r.standard_normal((len(rows), kvh, hd))
            vr[rows] = r.standard_normal((len(rows), kvh, hd))
        self.cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.T = int(self.cu[-1]) + pad
        self.gain = (0.4 * (1 + 0.1 * r.standard_normal(hd))).astype(np.float32)
        self.k_gain = (0.4 * (1 + 0.1 * r.standard_normal(hd))).astype(np.float32)
        c, s = sa.rope_tables(np.arange(MAX_POS), hd, theta, device="cpu")
        self.cos, self.sin = c.numpy(), s.numpy()
        self.q = r.standard_normal((max(1, self.T), nh, hd)).astype(np.float32)
        self.k_new = r.standard_normal((max(1, self.T), kvh, hd)).astype(np.float32)
        self.v_new = r.standard_normal((max(1, self.T), kvh, hd)).astype(np.float32)

    def tokens(self):
        """(sequence, position) of every packed row, None for rows of nobody."""
        rows = [(b, self.keys[b] - self.new[b] + i) for b in range(len(self.keys)) for i in range(self.new[b])]
        return rows + [None] * (max(1, self.T) - len(rows))

    def dev(self, **over):
        """The device operands every entry point takes."""
        t = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
        d = dict(k_pages=t(self.k_pages), v_pages=t(self.v_pages), table=t(self.table),
                 key_len=t(np.array(self.keys, np.int32)), cu=t(self.cu), q=t(self.q), gain=t(self.gain),
                 k_gain=t(self.k_gain), cos=t(self.cos), sin=t(self.sin), k_new=t(self.k_new), v_new=t(self.v_new))
        d.update(over)
        return d

    def cfg(self, **kw):
        return sa.AttnConfig(self.nh, self.kvh, self.hd, self.window, **kw)

    def oracle(self, q=None, tokens=None, k_pages=None, v_pages=None, scale=1.0, gain=True, rope=True):
        return OP.attend(self.q if q is None else q, self.tokens() if tokens is None else tokens,
                         self.k_pages if k_pages is None else k_pages, self.v_pages if v_pages is None else v_pages,
                         self.table, q_gain=self.gain if gain else None, cos=self.cos if rope else None,
                         sin=self.sin if rope else None, window=self.window, scale=scale)


def bound(out, A, S, *, q16, kv32, out16, k16=False):
    """Largest |kernel - exact| of an output. Half a step of f16 is u = 2^-11, of f32 2^-24.

    P and V enter f16 products: P rounded (u A), V rounded on f32 caches (u A); partial outputs of
    a split held in f16 (u A, and 2^-25 below the normal range; P's own subnormals likewise, per
    key, at most 2^-25 sum |v| / l, inside the same term for the hundreds of keys used here). A
    score is off by d <= e S: e = u for q in f16, u more for K rounded to f16, and 2^-19 S for the
    f32 arithmetic (the norm, the rotation, hd products, exp2). Weights then move by exp(+-2 d).
    The output type rounds by u or 2^-24 of the value."""
    u = 2.0 ** -11
    e = (u if q16 else 2.0 ** -21) + (u if k16 else 0.0) + 2.0 ** -19
    d = e * S + 2.0 ** -20
    fac = np.expm1(2 * d) + 3 * u
    return fac * A + (u if out16 else 2.0 ** -24) * np.abs(out) + 2.0 ** -17


def check(got, want, tol, what=""):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, f"{what}: {got.shape} vs {want.shape}"
    assert np.isfinite(got).all(), f"{what}: non-finite outputs at {np.argwhere(~np.isfinite(got))[:4].tolist()}"
    d = np.abs(got - want)
    assert (d <= tol).all(), f"{what}: off by {(d / tol).max():.2f} x the bound at {np.unravel_index((d / tol).argmax(), d.shape)}"
