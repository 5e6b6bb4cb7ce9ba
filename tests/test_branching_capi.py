"""CPU checks of the entry points of generation that branches: refusals before anything runs, workspace sizes,
the definitions themselves, and the arithmetic of trees' rows and tiles for the host compiler."""
import ctypes

import numpy as np
import pytest
import torch

import oracle.branching as OB
import slang_amd as sa
from slang_amd import _lib
from slang_amd._lib import G4APaged
from test_paged_capi import E, FAKE, U, W, cfg, paged
from test_paged_rows import holds

OUT, FAR = 0x4000000, 1 << 44


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def tree(lib, c=None, pg=None, n=8, cu=FAKE, par=FAKE, q=FAKE, qg=None, cos=None, sin=None, kn=None, vn=None, ks=0.0, vs=0.0, kg=None,
         out=OUT, ws=FAKE, nb=1 << 40):
    return lib.g4a_paged_tree(ctypes.byref(c or cfg()), None if pg == 0 else ctypes.byref(pg or paged()), n, cu, par, q, qg, cos, sin,
                              kn, vn, ks, vs, kg, out, ws, nb, None)


def accept(lib, n=8, seqs=2, max_path=4, **kw):
    a = dict(cu=FAKE, par=FAKE, drafts=FAKE, targets=FAKE, lens=FAKE, path=FAKE, count=FAKE, nxt=FAKE, kept=FAKE)
    a.update(kw)
    return lib.g4a_tree_accept(n, seqs, a["cu"], a["par"], a["drafts"], a["targets"], a["lens"], max_path, a["path"], a["count"],
                               a["nxt"], a["kept"], None)


def pools(*rows):
    return (ctypes.c_int64 * (2 * len(rows)))(*[x for r in rows for x in r])


ONE = ((FAR, 512),)


def keep(lib, ps=ONE, n_pools=None, pg=None, n=8, cu=FAKE, path=FAKE, max_path=4, count=FAKE):
    arr = pools(*ps) if ps is not None else None
    return lib.g4a_paged_keep(arr, len(ps or ()) if n_pools is None else n_pools, None if pg == 0 else ctypes.byref(pg or paged()), n, cu,
                              path, max_path, count, None)


def fork(lib, ps=ONE, n_pools=None, pg=None, n_new=4, par=FAKE, room=1, free=0x20000, n_free=0x30000, table=0x40000, lens=0x50000,
         new_free=0x60000, new_n=0x70000, ws=FAKE, nb=1 << 40):
    arr = pools(*ps) if ps is not None else None
    pg = paged(page_table=0x10000, key_len=0x18000) if pg is None else pg
    return lib.g4a_paged_fork(arr, len(ps or ()) if n_pools is None else n_pools, None if pg == 0 else ctypes.byref(pg), n_new, par, room,
                              free, n_free, table, lens, new_free, new_n, ws, nb, None)


def select(lib, groups=2, width=4, vocab=1000, f16=0, logits=FAKE, stride=1000, scores=FAKE, done=None, pad=0, cap=0.0, n_out=4, s=FAKE,
           p=FAKE, t=FAKE, ws=FAKE, nb=1 << 40):
    return lib.g4a_beam_select(groups, width, vocab, f16, logits, stride, scores, done, pad, cap, n_out, s, p, t, ws, nb, None)


def test_tree_refusals(lib):
    assert tree(lib, pg=0) == E and tree(lib, pg=paged(k_pages=None)) == E and tree(lib, pg=paged(page_size=24)) == U
    assert tree(lib, pg=paged(n_seq=40000)) == E and tree(lib, c=cfg(head_dim=128)) == U
    assert tree(lib, c=cfg(n_q_heads=24, n_kv_heads=2)) == E and b"1, 2, 4 or 8" in lib.g4a_last_error()
    assert tree(lib, n=0) == E and tree(lib, n=1 << 30) == E and tree(lib, cu=None) == E
    assert tree(lib, par=None) == E and tree(lib, par=FAKE + 2) == E
    assert tree(lib, q=None) == E and tree(lib, q=FAKE + 4) == E and tree(lib, out=OUT + 8) == E and tree(lib, out=FAKE + 4096) == E
    assert tree(lib, cos=FAKE) == E and tree(lib, cos=FAKE + 4, sin=FAKE) == E and tree(lib, qg=FAKE + 4) == E
    assert tree(lib, kn=FAKE) == E and tree(lib, vn=FAKE) == E and tree(lib, kn=FAKE + 8, vn=FAKE) == E
    assert tree(lib, kg=FAKE + 4) == E and tree(lib, ks=-1.0) == E and tree(lib, vs=float("nan")) == E
    assert tree(lib, c=cfg(flags=_lib.Q_HILO)) == U
    assert tree(lib, ws=None) == W and tree(lib, ws=FAKE + 16) == W and tree(lib, nb=16) == W
    size = lambda n=8, c=None, **k: lib.g4a_paged_tree_ws_bytes(ctypes.byref(c or cfg()), ctypes.byref(paged(**k)), n)  # noqa: E731
    assert size() > 0 and size(n=0) == 0 and size(n_pages=0) == 0 and size(c=cfg(n_q_heads=24)) == 0


@pytest.mark.parametrize("kvh,hd,window", [(1, 256, 512), (2, 256, 0), (8, 256, 0), (2, 512, 0), (1, 512, 4096)])
@pytest.mark.parametrize("kv_f32", [False, True])
def test_a_workspace_holds_every_smaller_call(kvh, hd, window, kv_f32):
    c, kw = sa.AttnConfig(8, kvh, hd, window), dict(page_size=16, kv_f32=kv_f32)
    seqs, keys = [1, 2, 7, 33, 64, 200, 1000, 4000], [1, 16, 129, 320, 600, 4096, 30000, 131072]
    tokens = [1, 5, 33, 63, 64, 65, 1000, 1024, 1025, 10000, 100000]
    got = np.array([[[sa.paged_tree_ws_bytes(t, n, k, c, **kw) for k in keys] for n in seqs] for t in tokens])
    assert all((np.diff(got, axis=i) >= 0).all() for i in range(3))
    b = np.array([[[sa.beam_select_ws_bytes(g, 4, v, k) for k in (1, 4, 64)] for v in (1, 500, 32000, 65536, 100000, 131071, 131072, 262144)]
                  for g in (1, 2, 16, 20, 21, 32, 40, 128, 1000)])
    assert all((np.diff(b, axis=i) >= 0).all() for i in range(3))
    assert all(sa.paged_fork_ws_bytes(a, n) <= sa.paged_fork_ws_bytes(b, n) for a, b in ((1, 2), (31, 33), (1000, 100000)) for n in (1, 9))


def test_accept_refusals(lib):
    assert accept(lib, n=0) == E and accept(lib, seqs=0) == E and accept(lib, max_path=0) == E
    for name in ("cu", "par", "drafts", "targets", "lens", "path", "count", "nxt", "kept"):
        assert accept(lib, **{name: None}) == E and accept(lib, **{name: FAKE + 2}) == E, name


def test_keep_refusals(lib):
    assert keep(lib, pg=0) == E and keep(lib, pg=paged(page_table=None)) == E and keep(lib, pg=paged(page_size=17)) == U
    assert keep(lib, pg=paged(k_pages=None, v_pages=None), n=0) == E  # the pages are the pools'
    assert keep(lib, n=0) == E and keep(lib, cu=None) == E and keep(lib, path=None) == E and keep(lib, count=FAKE + 1) == E
    assert keep(lib, max_path=0) == E
    for bad in ((0, 512), (FAR + 8, 512), (FAR, 0), (FAR, -16), (FAR, 24), (FAR, 1 << 21)):
        assert keep(lib, ps=(bad,)) == E, bad
    assert keep(lib, ps=None, n_pools=1) == E and keep(lib, n_pools=-1) == E
    assert keep(lib, ps=[(FAR + (i << 30), 512) for i in range(65)]) == E
    size = 100 * 16 * 512  # of a pool
    assert keep(lib, ps=((FAR, 512), (FAR + size - 16, 512))) == E and b"share memory" in lib.g4a_last_error()
    assert keep(lib, ps=((FAR + size, 512), (FAR, 512)), n=0) == E and b"share" not in lib.g4a_last_error()
    assert keep(lib, ps=()) == 0  # nothing to move


def test_fork_refusals(lib):
    assert fork(lib, pg=0) == E and fork(lib, n_new=0) == E and fork(lib, room=-1) == E and fork(lib, room=(1 << 30) + 1) == E
    for name in ("par", "free", "n_free", "table", "lens", "new_free", "new_n"):
        assert fork(lib, **{name: None}) == E and fork(lib, **{name: 0x90002}) == E, name
    for over in (dict(table=0x10010), dict(table=0x18000), dict(lens=FAKE), dict(new_free=0x20000), dict(new_n=0x30000),
                 dict(new_free=0x20000 - 396), dict(lens=0x40000 + 4 * 39), dict(new_n=0x50000 + 12)):
        assert fork(lib, **over) == E and b"overlap" in lib.g4a_last_error(), over
    assert fork(lib, ws=None) == W and fork(lib, ws=FAKE + 16) == W and fork(lib, nb=64) == W
    assert fork(lib, ps=((FAR, 512), (FAR, 512))) == E
    assert lib.g4a_paged_fork_ws_bytes(ctypes.byref(paged()), 0) == 0 and lib.g4a_paged_fork_ws_bytes(ctypes.byref(paged()), 5) > 0


def test_select_refusals(lib):
    for bad in (dict(groups=0), dict(width=0), dict(vocab=0), dict(n_out=0), dict(width=65), dict(n_out=65), dict(groups=40000),
                dict(vocab=(1 << 30) + 1, stride=1 << 31), dict(logits=None), dict(logits=FAKE + 8), dict(scores=None), dict(s=None),
                dict(p=None), dict(t=FAKE + 2), dict(stride=999), dict(cap=-1.0), dict(cap=float("nan")), dict(cap=float("inf")),
                dict(done=FAKE, pad=-1), dict(done=FAKE, pad=1000)):
        assert select(lib, **bad) == E, bad
    assert select(lib, ws=None) == W and select(lib, ws=FAKE + 16) == W and select(lib, nb=64) == W
    assert lib.g4a_beam_select_ws_bytes(1, 65, 10, 4) == 0 and lib.g4a_beam_select_ws_bytes(1, 4, 10, 4) > 0
    assert sa.beam_select_ws_bytes(16, 8, 262144) > 0
    with pytest.raises(_lib.G4AError):
        sa.beam_select_ws_bytes(1, 8, 0)


def test_host_refusals_without_a_gpu():
    """The host layer refuses CPU tensors before it loads anything."""
    c = sa.AttnConfig(8, 2, 256)
    q, pages = torch.zeros(2, 8, 256), torch.zeros(4, 16, 2, 256, dtype=torch.float16)
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    for call in (lambda: sa.paged_tree(q, pages, pages, i(2, 2), i(2), i(3), i(2), c, workspace=None),
                 lambda: sa.paged_tree(q[:, :4], pages, pages, i(2, 2), i(2), i(3), i(2), c, workspace=None),
                 lambda: sa.tree_accept(i(4), i(4), i(4), i(2), i(1)),
                 lambda: sa.paged_keep([pages], i(2, 2), i(2), i(3), i(2, 2), i(2)),
                 lambda: sa.paged_fork([pages], i(2, 2), i(2), i(2), i(4), i(1), workspace=None),
                 lambda: sa.beam_select(torch.zeros(4, 10), torch.zeros(2, 2), workspace=None),
                 lambda: sa.CachePools([pages])):
        with pytest.raises(ValueError):
            call()


def test_definitions():
    """Small ones by hand."""
    par = np.array([-1, 0, 0, 1, 7, 2, 5])
    assert OB.line(par, 3) == [3, 1, 0] and OB.line(par, 4) == [4] and OB.line(par, 6) == [6, 5, 2, 0]
    assert OB.attended(par, 10, 6, 0) == (list(range(10)) + [10, 12, 15, 16], 13)
    assert OB.attended(par, 10, 6, 3) == ([12, 15, 16], 13)  # two ancestors, no history
    assert OB.attended(par, 10, 6, 5) == ([9, 10, 12, 15, 16], 13)
    assert OB.attended(par, -2, 3, 0) == ([1], 0)  # the ancestors' rows are not there
    assert OB.accept([20], [0, 4], np.array([-1, 0, 0, 2]), np.array([1, 5, 6, 7]), np.array([6, 0, 7, 9]), 3) == ([[0, 2, 3]], [3], [9], [19])
    new, length, free, _ = OB.fork([], np.array([[0, 1, -1], [2, 3, 4]]), [20, 33], [0, 0], [5], 1, 16, 6)
    assert new.tolist() == [[0, 1, -1], [0, 4, -1]] and length == [20, 20] and free == [5, 2, 3]
    s, p, t = OB.select(np.array([[-np.log(2), -np.log(4), -np.log(4)], [np.log(0.125), np.log(0.875), -np.inf]]), np.log([[0.5, 0.5]]), 0.0, 4)
    assert np.allclose(np.exp(s), [[0.4375, 0.25, 0.125, 0.125]]) and p.tolist() == [[1, 0, 0, 0]] and t.tolist() == [[1, 0, 1, 2]]


def test_tiles_of_trees(tmp_path):
    """Every key that a token attends lies in its block's tiles, each tile within a word of the token's bits, and the
    bits within the words; nothing overflows up to 2^30 keys."""
    holds(tmp_path, """
constexpr int kMost = 1 << 30;
constexpr bool fits(int start, int S, int bq, int kt, int window) {
    for (int qb = 0; qb * bq < S; ++qb) {
        const int64_t lo = tree_first(start, window) & ~(kt - 1), end = (int64_t)start + (qb + 1) * (int64_t)bq;
        const int64_t hi = end < (int64_t)start + S ? end : (int64_t)start + S;
        const int n = tree_tiles(start, S, qb, bq, kt, window);
        if (n < 0 || (hi > lo ? n != (hi - lo + kt - 1) / kt : n != 0)) return false;
        if (n > 0) {  // the last tile's word, for keys of the tree
            const int64_t kb = lo + (int64_t)(n - 1) * kt, word = (kb - (start & ~63)) >> 6;
            if (kb + kt > start && (word < 0 || word >= tree_words(S) || (kb & (kt - 1)))) return false;
            if (((hi - 1 - (start & ~63)) >> 6) >= tree_words(S)) return false;
        }
    }
    return true;
}
constexpr bool all() {
    for (int start : {-1000, -63, -1, 0, 1, 31, 32, 63, 64, 65, 700, 4096, kMost - 1500})
        for (int S : {1, 2, 16, 63, 64, 65, 100, 700, 1024})
            for (int bq : {16, 32, 64, 128})
                for (int kt : {32, 64})
                    for (int window : {0, 1, 16, 30, 512, kMost})
                        if (!fits(start, S, bq, kt, window)) return false;
    return true;
}
static_assert(all(), "a key outside the tiles or the bits");
static_assert(cut_tree(SeqRows{5, 1500, 2000}).hi == 1029 && cut_tree(SeqRows{5, 1500, 2000}).keys == 1529, "");
static_assert(cut_tree(SeqRows{5, 1029, 2000}).hi == 1029 && cut_tree(SeqRows{5, 6, 7}).keys == 7, "");
""")


def test_structs():
    assert ctypes.sizeof(G4APaged) == 64  # g4a_pool is an address and a count: two 64-bit words
