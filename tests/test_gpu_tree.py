"""paged_tree against its float64 definition: types, head layouts, trees from one token to several blocks of
columns, histories from nothing to several pieces, windows, missing pages, poisoned rows, what stays untouched."""
import numpy as np
import pytest
import torch

import oracle.branching as OB
import oracle.paged as OP
import slang_amd as sa
from paged_cases import Batch, bound, check

pytestmark = pytest.mark.gpu


def bits(x):
    return x.detach().cpu().contiguous().view(torch.uint8).numpy()


def trees(new, seed, kind="mixed"):
    """Packed parents of trees of new[b] tokens."""
    r, out = np.random.default_rng(seed), []
    for n in new:
        i = np.arange(n)
        p = {"mixed": np.floor(i * r.random(n) ** 0.6), "chain": i - 1, "star": np.where(i > 0, 0, -1), "roots": -np.ones(n)}[kind].astype(np.int32)
        if kind == "mixed" and n:
            p[0] = -1
            p[r.random(n) < 0.1] = -7
        out.append(p)
    return np.concatenate(out).astype(np.int32) if out else np.zeros(0, np.int32)


class Trees(Batch):
    """A batch whose packed rows are trees."""

    def __init__(self, keys, new, *, kind="mixed", **kw):
        super().__init__(keys, new, **kw)
        par = trees(new, kw.get("seed", 0) + 1, kind)
        self.parents = np.concatenate([par, np.full(max(1, self.T) - len(par), 3, np.int32)])

    def dev(self, **over):
        return super().dev(**dict(dict(parents=torch.from_numpy(self.parents).cuda()), **over))

    def oracle(self, **kw):
        kw = dict(dict(q_gain=self.gain, cos=self.cos, sin=self.sin, window=self.window), **kw)
        return OB.attend_tree(self.q, self.keys, self.cu, self.parents, self.k_pages, self.v_pages, self.table, **kw)

    def live(self):
        return np.array([w is not None for w in OB.packed(self.keys, self.cu, max(1, self.T))])


def tree(b, d, append=False, **kw):
    new = dict(k_new=d["k_new"], v_new=d["v_new"], k_gain=d["k_gain"]) if append else {}
    kw = dict(dict(q_gain=d["gain"], rope_cos=d["cos"], rope_sin=d["sin"], workspace=sa.Workspace()), **new, **kw)
    return sa.paged_tree(d["q"], d["k_pages"], d["v_pages"], d["table"], d["key_len"], d["cu"], d["parents"], kw.pop("cfg", b.cfg()), **kw)


def run(b, kv32=False, dts=(torch.float16, torch.float32), what="", tol=1.0, **kw):
    out, A, S = b.oracle()
    live = b.live()
    for dt in dts:
        d = b.dev()
        o = torch.full((max(1, b.T), b.nh, b.hd), 7.25, dtype=dt, device="cuda")
        got = tree(b, d, out=o, **kw).cpu().numpy()
        check(got[live], out[live], bound(out, A, S, q16=True, kv32=kv32, out16=dt is torch.float16, k16=kv32)[live], f"{what} {dt}")
        assert (got[~live] == 7.25).all()
        assert np.array_equal(bits(d["k_pages"]).reshape(-1), b.k_pages.reshape(-1).view(np.uint8))
        assert np.array_equal(bits(d["v_pages"]).reshape(-1), b.v_pages.reshape(-1).view(np.uint8))
    return got


@pytest.mark.parametrize("hd,kvh,kv", [(256, 2, np.float16), (256, 1, np.float32), (512, 1, np.float16), (512, 2, np.float32)])
@pytest.mark.parametrize("window", [0, 100, 16, 2])
def test_tree(hd, kvh, kv, window):
    new = [1, 0, 33, 65, 16, 2, 40, 12]
    hist = [0, 0, 100, 3, 240, 511, 0, 64]
    b = Trees([a + h for a, h in zip(new, hist)], new, hd=hd, kvh=kvh, kv=kv, window=window, pad=5, seed=window)
    run(b, kv32=kv is np.float32)


@pytest.mark.parametrize("kvh", [1, 2, 4, 8])
@pytest.mark.parametrize("hd", [256, 512])
@pytest.mark.parametrize("page", [16, 128])
def test_groups_and_pages(hd, kvh, page):
    b = Trees([70, 129, 17], [70, 40, 17], hd=hd, kvh=kvh, page=page, seed=kvh)
    run(b, dts=(torch.float16,))


@pytest.mark.parametrize("kind", ["chain", "star", "roots"])
@pytest.mark.parametrize("window", [0, 30])
def test_shapes_of_trees(kind, window):
    b = Trees([130, 200, 64], [70, 129, 64], kind=kind, window=window)
    run(b, dts=(torch.float16,))


@pytest.mark.parametrize("kvh", [1, 4])
@pytest.mark.parametrize("keys", [[40, 130], [1500, 700]])
def test_queries_keep_their_bits(kvh, keys):
    """At head_dim 256 q is a pair of f16 operands: the error of its rounding is not there."""
    b = Trees(keys, [20, 33], kvh=kvh, seed=7)
    out, A, S = b.oracle()
    check(tree(b, b.dev()).cpu().numpy(), out, bound(out, A, S, q16=False, kv32=False, out16=True))


@pytest.mark.parametrize("hd,kvh", [(256, 2), (512, 1)])
@pytest.mark.parametrize("window", [0, 300])
def test_long_histories(hd, kvh, window):
    """Histories long enough to be cut into pieces, beside short ones."""
    b = Trees([1500, 20, 900, 1201], [40, 20, 130, 1], hd=hd, kvh=kvh, window=window, page=32)
    run(b, dts=(torch.float16,))


@pytest.mark.parametrize("n", [1, 15, 16, 17, 63, 64, 65, 128])
def test_one_sequence(n):
    """Each length of one tree, at every place of its first row within a word of bits."""
    for hist in (0, 1, 63, 64, 700 + n):
        run(Trees([hist + n], [n], kvh=2, seed=n), dts=(torch.float16,), what=f"history {hist}")


@pytest.mark.parametrize("hd", [256, 512])
def test_many_sequences(hd):
    """More blocks than compute units; more sequences than a list's chunk."""
    r = np.random.default_rng(3)
    new = r.integers(0, 7, 300)
    keys = new + r.integers(0, 60, 300) * (new > 0)
    run(Trees(list(keys), list(new), hd=hd, kvh=1), dts=(torch.float16,))


@pytest.mark.parametrize("hd", [256, 512])
def test_missing_pages(hd):
    b = Trees([100, 48, 150, 40], [60, 48, 20, 10], hd=hd, kvh=1, missing=[(0, 0), (0, 3), (1, 0), (1, 1), (1, 2), (2, 4), (2, 5), (2, 9), (3, 2)])
    got = run(b, dts=(torch.float16,))
    assert (got[60:108] == 0).all()


@pytest.mark.parametrize("hd,kvh", [(256, 1), (256, 8), (512, 3)])
@pytest.mark.parametrize("rows", ["f16", "f32"])
@pytest.mark.parametrize("kv", [np.float16, np.float32])
def test_rows_are_kv_writes(hd, kvh, rows, kv):
    """With k_new and v_new: every row that kv_write would store for the token at its position, to the bit, at the row of
    its index; nothing else; and they are attended."""
    nh = 8 if kvh != 3 else 6
    new = [40, 0, 5, 1, 33, 1]
    b = Trees([40, 0, 17, 1, 130, 16], new, hd=hd, kvh=kvh, kv=kv, pad=3, missing=[(0, 1), (4, 8)], seed=hd + kvh, nh=nh)
    b.k_pages[np.isnan(b.k_pages)] = 0.5
    b.v_pages[np.isnan(b.v_pages)] = 0.5
    d = b.dev()
    t = torch.float16 if rows == "f16" else torch.float32
    k, v = d["k_new"].to(t), d["v_new"].to(t)
    want_k, want_v = b.k_pages.copy(), b.v_pages.copy()
    dense = [torch.zeros(b.T, kvh, hd, dtype=d["k_pages"].dtype, device="cuda") for _ in range(2)]
    who = OB.packed(b.keys, b.cu, b.T)
    pos = [0 if w is None else b.keys[w[0]] - new[w[0]] + len(OB.line(b.parents[b.cu[w[0]]:b.cu[w[0] + 1]], w[1])) - 1 for w in who]
    at = torch.tensor(pos, device="cuda")
    sa.kv_write(k, v, *dense, 0, sa.AttnConfig(kvh, kvh, hd), k_gain=d["k_gain"], rope_cos=d["cos"][at].contiguous(),
                rope_sin=d["sin"][at].contiguous(), k_in_q=0.03, v_in_q=0.05)
    rk, rv = (x.cpu().numpy() for x in dense)
    for tok, w in enumerate(who):
        if w is None:
            continue
        row = OB.there(b.table, w[0], [b.keys[w[0]] - new[w[0]] + w[1]], b.page, b.n_pages)
        if len(row):
            want_k.reshape(-1, kvh, hd)[row[0]] = rk[tok]
            want_v.reshape(-1, kvh, hd)[row[0]] = rv[tok]
    got = tree(b, dict(d, k_new=k, v_new=v), append=True, k_in_q=0.03, v_in_q=0.05)
    assert np.array_equal(bits(d["k_pages"]).reshape(-1), want_k.reshape(-1).view(np.uint8))
    assert np.array_equal(bits(d["v_pages"]).reshape(-1), want_v.reshape(-1).view(np.uint8))
    b.k_pages, b.v_pages = want_k, want_v
    out, A, S = b.oracle()
    live, kv32 = b.live(), kv is np.float32
    check(got.cpu().numpy()[live], out[live], bound(out, A, S, q16=True, kv32=kv32, out16=True, k16=kv32)[live])


@pytest.mark.parametrize("hd", [256, 512])
@pytest.mark.parametrize("window", [0, 50])
def test_a_chain_is_a_prompt(hd, window):
    """A tree without branches is a prompt's piece: paged_prefill's outputs, up to the order of sums."""
    b = Trees([150, 700], [90, 30], hd=hd, kvh=1, window=window, kind="chain")
    d = b.dev()
    got = tree(b, d).cpu().numpy()
    ref = sa.paged_prefill(d["q"], d["k_pages"], d["v_pages"], d["table"], d["key_len"], d["cu"], b.cfg(), workspace=sa.Workspace(),
                           q_gain=d["gain"], rope_cos=d["cos"], rope_sin=d["sin"]).cpu().numpy()
    out, A, S = b.oracle()
    tol = bound(out, A, S, q16=True, kv32=False, out16=True)
    check(got, out, tol)
    check(got, ref, 2 * tol)


@pytest.mark.parametrize("hd", [256, 512])
def test_masked_keys_may_be_anything(hd):
    """The K row of a draft does not reach its siblings' branches, whatever it holds; with V of the type's lowest value."""
    b = Trees([150], [60], hd=hd, kvh=1, kind="mixed", seed=5)
    out, A, S = b.oracle()
    victim = 7
    others = [i for i in range(60) if victim not in OB.line(b.parents, i)]
    at = b.table[0, 97 // 16], 97 % 16
    k, v = b.k_pages.copy(), b.v_pages.copy()
    v[at] = -65504.0
    for junk in (np.inf, -np.inf, np.nan, 65504.0):
        k[at] = junk
        got = tree(b, b.dev(k_pages=torch.from_numpy(k).cuda(), v_pages=torch.from_numpy(v).cuda())).cpu().numpy()
        check(got[others], out[others], bound(out, A, S, q16=True, kv32=False, out16=True)[others], f"{junk}")


@pytest.mark.parametrize("hd,kvh", [(256, 2), (512, 1)])
@pytest.mark.parametrize("keys", [100, 1500])
@pytest.mark.parametrize("what", ["q", "k"])
def test_shows_what_is_not_finite(hd, kvh, keys, what):
    """A query head, or an attended K row, that is not finite makes its outputs NaN and no other, however the keys are cut."""
    b = Trees([keys], [20], hd=hd, kvh=kvh, seed=2)
    out, A, S = b.oracle()
    tol = bound(out, A, S, q16=True, kv32=False, out16=True)
    bad = np.zeros(out.shape, bool)
    G = 8 // kvh
    if what == "q":
        b.q[3, 3, 7] = np.nan
        bad[3, 3] = True
    else:
        b.k_pages.reshape(-1, kvh, hd)[OB.there(b.table, 0, [60], b.page, b.n_pages)[0], 0, 5] = np.nan
        bad[:, :G] = True
    got = tree(b, b.dev()).cpu().numpy()
    assert np.isnan(got[bad]).all()
    check(got[~bad], out[~bad], tol[~bad])


def test_more_rows_than_keys():
    """Tokens whose row would be below zero attend nothing, and are nobody's ancestors; offsets out of range are cut."""
    b = Trees([30, 20], [30, 20])
    b.keys = [12, 20]
    out, A, S = b.oracle()
    tol = bound(out, A, S, q16=True, kv32=False, out16=True)
    short = torch.tensor([12, 20], dtype=torch.int32, device="cuda")
    got = tree(b, b.dev(key_len=short)).cpu().numpy()
    check(got, out, tol)
    assert (got[:18] == 0).all()
    got = tree(b, b.dev(key_len=short, cu=torch.tensor([0, 30, 1000], dtype=torch.int32, device="cuda"))).cpu().numpy()
    check(got, out, tol)


def test_trees_of_more_tokens_than_there_may_be():
    """The rows behind a tree's first 1024 are rows of nobody: not stored, their outputs stay."""
    n = 1100
    b = Trees([n + 10], [n], kvh=8, kind="star", extra_cols=2)
    d = b.dev()
    o = torch.full((n, 8, 256), 7.25, dtype=torch.float16, device="cuda")
    before = bits(d["k_pages"]).copy()
    got = tree(b, d, append=True, out=o).cpu().numpy()
    assert (got[1024:] == 7.25).all()
    stored = (bits(d["k_pages"]) != before).reshape(b.n_pages, 16, -1).any(-1)
    want = np.zeros_like(stored)
    t = np.arange(10, 1034)
    want[b.table[0, t // 16], t % 16] = True
    assert np.array_equal(stored, want)
    b.k_pages, b.v_pages = d["k_pages"].cpu().numpy(), d["v_pages"].cpu().numpy()
    out, A, S = b.oracle()
    check(got[:1024], out[:1024], bound(out, A, S, q16=True, kv32=False, out16=True)[:1024])


@pytest.mark.parametrize("n", [300, 1024])
def test_deep_trees(n):
    """Chains of hundreds of tokens, a window shorter than the tree."""
    for window in (0, 40):
        b = Trees([n + 33], [n], kvh=8, kind="chain", window=window)
        run(b, dts=(torch.float16,), what=f"window {window}")


@pytest.mark.parametrize("hd", [256, 512])
@pytest.mark.parametrize("n_seq", [3, 300])
def test_offsets_that_do_not_ascend(hd, n_seq):
    """Whatever the offsets, the cache stays, rows behind the packed ones stay, and a later call is right."""
    b = Trees([700, 640], [640, 20], hd=hd, kvh=1, pad=9)
    d = b.dev()
    cu = [0] + [(660, 0)[i % 2] for i in range(n_seq)]
    o = torch.full((b.T + 4, 8, hd), 7.25, dtype=torch.float16, device="cuda")
    w = sa.Workspace()
    tree(b, dict(d, table=d["table"][:1].repeat(n_seq, 1), key_len=d["key_len"][:1].repeat(n_seq),
                 cu=torch.tensor(cu, dtype=torch.int32, device="cuda")), out=o[:b.T], workspace=w)
    assert np.array_equal(bits(d["k_pages"]).reshape(-1), b.k_pages.reshape(-1).view(np.uint8))
    assert (o[660:] == 7.25).all()
    out, A, S = b.oracle()
    check(tree(b, d, workspace=w).cpu().numpy()[:660], out[:660], bound(out, A, S, q16=True, kv32=False, out16=True)[:660])


def test_options():
    """No norm, no RoPE, another scale, srq'd output; numpy steps."""
    b = Trees([200, 31], [9, 5], kvh=4)
    out, A, S = b.oracle(q_gain=None, cos=None, sin=None, scale=0.0625)
    got = tree(b, b.dev(), q_gain=None, rope_cos=None, rope_sin=None, cfg=b.cfg(scale=0.0625), out_dtype=torch.float32)
    tol = bound(out, A, S, q16=True, kv32=False, out16=False)
    check(got.cpu().numpy(), out, tol)
    got = tree(b, b.dev(), q_gain=None, rope_cos=None, rope_sin=None, cfg=b.cfg(scale=0.0625, out_q=0.02), k_in_q=np.float32(0))
    k = got.float().cpu().numpy() / 0.02
    assert np.abs(k - np.round(k)).max() <= 128 * 2.0 ** -11 + 1e-3  # on the grid, up to the f16 rounding
    check(got.cpu().numpy(), np.clip(out, -2.56, 2.54), tol + 0.0101 + 2.56 * 2.0 ** -11)


def test_plain_rows():
    """No gain, no RoPE, no v norm: the stored rows are the given ones."""
    b = Trees([9, 33], [9, 2], kv=np.float32)
    d = b.dev()
    tree(b, dict(d, k_gain=None), append=True, q_gain=None, rope_cos=None, rope_sin=None, v_norm=False)
    for tok, (s, i) in enumerate(OB.packed(b.keys, b.cu, b.T)):
        row = OB.there(b.table, s, [b.keys[s] - b.new[s] + i], b.page, b.n_pages)[0]
        assert np.array_equal(d["k_pages"].cpu().numpy().reshape(-1, 2, 256)[row], b.k_new[tok])
        assert np.array_equal(d["v_pages"].cpu().numpy().reshape(-1, 2, 256)[row], b.v_new[tok])


def test_longer_than_the_bound():
    b = Trees([64, 40], [5, 7])
    out, A, S = b.oracle()
    d = b.dev(key_len=torch.tensor([10 ** 9, 40], dtype=torch.int32, device="cuda"))
    check(tree(b, d, max_key_len=64).cpu().numpy(), out, bound(out, A, S, q16=True, kv32=False, out16=True))


@pytest.mark.parametrize("kv", [np.float16, np.float32])
def test_captured(kv):
    """A captured call over a reserved workspace, replayed on new queries, lengths, trees and tables."""
    b = [Trees([200, 37, 900], [20, 5, 33], kv=kv, seed=s, extra_cols=e) for s, e in ((1, 1), (2, 1))]
    b.append(Trees([100, 50, 900], [3, 50, 5], kv=kv, seed=3, extra_cols=1))
    b[2].cu, b[2].T = b[2].cu, 58
    for x in b:  # one set of buffers
        x.q, x.k_new, x.v_new = (np.resize(y, (58, *y.shape[1:])) for y in (x.q, x.k_new, x.v_new))
        x.parents = np.resize(x.parents, 58)
    d = b[0].dev()
    pool = max(x.n_pages for x in b)
    for n in ("k_pages", "v_pages"):
        d[n] = torch.zeros(pool, *d[n].shape[1:], dtype=d[n].dtype, device="cuda")
    ws = sa.Workspace().reserve(sa.paged_tree_ws_bytes(58, 3, 57 * 16, b[0].cfg(), page_size=16, kv_f32=kv is np.float32))
    out = torch.zeros(58, 8, 256, dtype=torch.float16, device="cuda")

    def load(x):
        for n, v in (("q", x.q), ("k_new", x.k_new), ("v_new", x.v_new), ("cu", x.cu), ("parents", x.parents),
                     ("key_len", np.array(x.keys, np.int32)), ("table", x.table), ("gain", x.gain), ("k_gain", x.k_gain)):
            d[n].copy_(torch.from_numpy(np.ascontiguousarray(v)))
        for n in ("k_pages", "v_pages"):
            d[n][:x.n_pages].copy_(torch.from_numpy(getattr(x, n)))

    def call():
        tree(b[0], d, append=True, workspace=ws, out=out, max_key_len=57 * 16)

    load(b[0])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for x in (b[0], b[1], b[2], b[1]):
        load(x)
        call()
        want, pages = out.clone(), d["k_pages"].clone()
        torch.cuda.synchronize()
        load(x)
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(d["k_pages"].view(torch.uint8), pages.view(torch.uint8))


def test_refusals():
    b = Trees([40, 50], [4, 5])
    d = b.dev()
    for over in (dict(parents=d["parents"][:-1]), dict(parents=d["parents"].long()), dict(parents=d["parents"].cpu()),
                 dict(parents=d["parents"].view(3, 3)), dict(cu=d["cu"][:-1]), dict(q=d["q"].half())):
        with pytest.raises(ValueError):
            tree(b, dict(d, **over))
    for over in (dict(k_new=d["k_new"][:-1]), dict(v_new=d["v_new"].half()), dict(v_new=None), dict(k_gain=d["k_gain"][:4]),
                 dict(k_new=d["k_new"].double(), v_new=d["v_new"].double())):
        with pytest.raises(ValueError):
            tree(b, dict(d, **over), append=True)
    small = sa.Workspace().reserve(4096)
    with pytest.raises(RuntimeError):
        tree(b, d, workspace=small)
    assert tree(b, dict(d, q=d["q"][:0], parents=d["parents"][:0])).shape == (0, 8, 256)


@pytest.mark.parametrize("hd,kvh,n_seq", [(256, 2, 200), (512, 1, 400)])
@pytest.mark.parametrize("new", [3, 24])
def test_units_of_many_tiles(hd, kvh, n_seq, new):
    """More blocks than can be cut, each over more tiles than a wave holds pages of (64), with waves that have no token: all
    sequences read one history through tables of their own."""
    keys = 5000
    b = Trees([keys], [new], hd=hd, kvh=kvh, page=16)
    d = b.dev()
    q = torch.randn(n_seq * new, 8, hd, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    i32 = lambda x: torch.as_tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    got = sa.paged_tree(q, d["k_pages"], d["v_pages"], d["table"].repeat(n_seq, 1), i32([keys] * n_seq), i32(np.arange(n_seq + 1) * new),
                        d["parents"].repeat(n_seq), b.cfg(scale=0.3), workspace=sa.Workspace(), q_gain=d["gain"]).cpu().numpy()
    for s in (0, 1, n_seq // 2, n_seq - 1):
        b.q = q[s * new:(s + 1) * new].cpu().numpy()
        out, A, S = b.oracle(cos=None, sin=None, scale=0.3)
        check(got[s * new:(s + 1) * new], out, bound(out, A, S, q16=True, kv32=False, out16=True), f"sequence {s}")


@pytest.mark.parametrize("hd", [256, 512])
def test_one_long_history_among_many_sequences(hd):
    """More sequences than a chunk of the list, one of them worth cutting."""
    new = [5] + [1, 2] * 150
    keys = [1900] + [20, 9] * 150
    keys[290] = 1700
    run(Trees(keys, new, hd=hd, kvh=1), dts=(torch.float16,))


@pytest.mark.parametrize("hd,kvh", [(256, 2), (512, 1)])
@pytest.mark.parametrize("window", [0, 40, 5])
@pytest.mark.parametrize("kv", [np.float16, np.float32])
def test_appended_rows_behind_a_window(hd, kvh, window, kv):
    """Rows stored by the call itself, histories of every alignment, pages in front of the window not there."""
    new, hist = [12, 1, 40, 7, 0], [100, 63, 17, 300, 0]
    keys = [a + h for a, h in zip(new, hist)]
    b = Trees(keys, new, hd=hd, kvh=kvh, kv=kv, window=window, written=False, seed=window)
    if window:
        for s, h in enumerate(hist):
            b.table[s, :max(0, h + 1 - window) // b.page] = -1
    d = b.dev()
    got = tree(b, d, append=True).cpu().numpy()
    b.k_pages, b.v_pages = d["k_pages"].cpu().numpy(), d["v_pages"].cpu().numpy()
    out, A, S = b.oracle()
    kv32 = kv is np.float32
    check(got, out, bound(out, A, S, q16=True, kv32=kv32, out16=True, k16=kv32))
