"""Walking drafts, keeping accepted rows, forking beams' pages and selecting beams against their definitions in 64
bits and python integers, alone and as a server runs them."""
import numpy as np
import pytest
import torch

import oracle.branching as OB
import slang_amd as sa
from test_gpu_tree import Trees, tree, trees

pytestmark = pytest.mark.gpu


def dev(x, dtype=np.int32):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(x, dtype))).cuda()


# ---------------------------------------------------------------- tree_accept
def drafted(new, seed, kind="mixed", agree=0.7):
    """Parents, drafts and targets; drafts that the model agrees with as often as `agree`, siblings with equal tokens among them."""
    r = np.random.default_rng(seed)
    par = trees(new, seed, kind)
    lo = np.repeat(np.cumsum([0] + list(new))[:-1], new)
    targets = r.integers(0, 7, len(par))
    drafts = np.where(r.random(len(par)) < agree, targets[lo + np.clip(par, 0, None)] if len(par) else par, r.integers(0, 7, len(par)))
    return par, drafts.astype(np.int32), targets.astype(np.int32)


def accept(keys, new, par, drafts, targets, max_path=None, pad=0, **kw):
    cu = np.concatenate([[0], np.cumsum(new)])
    z = lambda x: dev(np.concatenate([x, np.full(pad, 3)]))  # noqa: E731
    return cu, sa.tree_accept(z(drafts), z(targets), z(par), dev(cu), dev(keys), max_path=max_path, **kw)


@pytest.mark.parametrize("new", [[1], [0], [12], [64, 65, 0, 1, 63], [253, 1, 256, 257, 0, 700], [3] * 130])
@pytest.mark.parametrize("kind,agree", [("mixed", 0.7), ("chain", 0.95), ("star", 0.5), ("mixed", 1.0), ("mixed", 0.0)])
def test_accept(new, kind, agree):
    par, drafts, targets = drafted(new, len(new), kind, agree)
    keys = [n + 10 for n in new]
    for max_path in (None, 1, 3, 1024):
        if sum(new) == 0 and max_path is None:
            continue
        cu, got = accept(keys, new, par, drafts, targets, max_path, pad=2)
        want = OB.accept(keys, cu, par, drafts, targets, got[0].shape[1])
        for g, w in zip(got, want):
            assert np.array_equal(g.cpu().numpy(), np.array(w).reshape(g.shape))


def test_accept_long_chain():
    """1024 tokens that the model all agrees with; more than that in the tree."""
    new = [1024, 1500]
    par, drafts, targets = drafted(new, 1, "chain", 1.0)
    cu, got = accept([2000, 2000], new, par, drafts, targets)
    assert got[1].tolist() == [1024, 1024] and got[0][1].tolist() == list(range(1024))
    assert got[3].tolist() == [2000, 2000 - 1500 + 1024]


def test_accept_prefers_the_first_of_equal_children():
    par, drafts, targets = np.array([-1, 0, 0, 1, 2], np.int32), np.array([9, 5, 5, 6, 6], np.int32), np.array([5, 6, 6, 1, 2], np.int32)
    _, got = accept([5], [5], par, drafts, targets, 5)
    assert got[0].tolist() == [[0, 1, 3, -1, -1]] and got[2].tolist() == [1]


def test_accept_empty_and_refused():
    z = torch.zeros(0, dtype=torch.int32, device="cuda")
    got = sa.tree_accept(z, z, z, dev([0, 0, 0]), dev([4, 0]))
    assert [x.tolist() for x in got] == [[[-1], [-1]], [0, 0], [-1, -1], [4, 0]]
    par, drafts, targets = (dev(x) for x in drafted([5], 1))
    cu, keys = dev([0, 5]), dev([9])
    bad = ((drafts, targets[:-1], par, cu, keys), (drafts.long(), targets, par, cu, keys), (drafts, targets, par, cu[:1], keys),
           (drafts, targets, par.cpu(), cu, keys), (drafts.view(1, 5), targets, par, cu, keys))
    for args in bad:
        with pytest.raises(ValueError):
            sa.tree_accept(*args)
    for kw in (dict(max_path=0), dict(out=got), dict(max_path=3, out=[x[:1] for x in got])):
        with pytest.raises(ValueError):
            sa.tree_accept(drafts, targets, par, cu, keys, **kw)


def test_accept_offsets_that_do_not_ascend():
    par, drafts, targets = (dev(x) for x in drafted([40], 1))
    for cu in ([0, 40, 0, 40], [-5, 100, 3, 2 ** 31 - 1], [40, 40, 0, 0]):
        got = sa.tree_accept(drafts, targets, par, dev(cu), dev([50] * 3))
        assert all(0 <= x <= 40 for x in got[1].tolist())


# ---------------------------------------------------------------- paged_keep
def pools_of(b, layers, seed, widths=((1, 256, torch.float16),)):
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for i in range(layers):
        kvh, hd, t = widths[i % len(widths)]
        out += [torch.randn(b.n_pages, b.page, kvh, hd, device="cuda", generator=g).to(t) for _ in range(2)]
    return out


def rows_of(x):
    return x.cpu().numpy().reshape(-1, *x.shape[2:])


WIDTHS = ((1, 256, torch.float16), (2, 512, torch.float32), (3, 256, torch.float16), (16, 512, torch.float32))


@pytest.mark.parametrize("layers", [1, 4])
@pytest.mark.parametrize("new", [[1], [12], [20, 0, 7, 64, 1], [130, 3]])
@pytest.mark.parametrize("page", [16, 64])
def test_keep(layers, new, page):
    keys = [n + 5 + 3 * i if n else 0 for i, n in enumerate(new)]
    b = Trees(keys, new, page=page, kvh=1, pad=2, missing=[(0, 0)] if len(new) > 1 else ())
    for seed, kind in ((1, "mixed"), (2, "chain"), (3, "star")):
        par, drafts, targets = drafted(new, seed, kind, 0.9)
        cu, (path, count, _, _) = accept(keys, new, par, drafts, targets)
        pools = pools_of(b, layers, seed, WIDTHS)
        want = OB.keep([rows_of(p).copy() for p in pools], keys, cu, path.tolist(), count.tolist(), b.table, page, b.n_pages)
        sa.paged_keep(pools, dev(b.table), dev(keys), dev(cu), path, count)
        for p, w in zip(pools, want):
            assert np.array_equal(rows_of(p), w)


@pytest.mark.parametrize("path,count", [([0, 2, 4, 6, 9], 5), ([5, 6, 7, 8, 9], 5), ([0, 3, 3, 4, 5], 5), ([0, 2, 1, 4, 5], 5),
                                        ([0, 2, 99, 5, 6], 5), ([-3, 2, 4, 5, 6], 5), ([1, 2, 3, 4, 5], 99), ([1, 2, 3, 4, 5], -1),
                                        ([9, 2 ** 31 - 1, -2 ** 31, 0, 0], 5)])
def test_keep_of_any_path(path, count):
    """A path ends at the first entry that does not ascend or is no token; its length is cut to what there is."""
    b = Trees([30], [10], kvh=1)
    pools = pools_of(b, 1, 7)
    want = OB.keep([rows_of(p).copy() for p in pools], [30], [0, 10], [path], [count], b.table, 16, b.n_pages)
    sa.paged_keep(pools, dev(b.table), dev([30]), dev([0, 10]), dev([path]), dev([count]))
    for p, w in zip(pools, want):
        assert np.array_equal(rows_of(p), w)


def test_keep_moves_a_long_path():
    """More rows than a workgroup holds at a time, over page borders, over rows that are read later."""
    n = 500
    b = Trees([n + 9], [n], kvh=1)
    path = np.sort(np.random.default_rng(1).permutation(n)[:400])
    for widths in WIDTHS:
        pools = pools_of(b, 1, 7, (widths,))
        want = OB.keep([rows_of(p).copy() for p in pools], [n + 9], [0, n], [path], [400], b.table, 16, b.n_pages)
        sa.paged_keep(pools, dev(b.table), dev([n + 9]), dev([0, n]), dev([path]), dev([400]))
        for p, w in zip(pools, want):
            assert np.array_equal(rows_of(p), w)


def test_keep_refused_and_empty():
    b = Trees([30, 20], [10, 5], kvh=1)
    pools, path, count = pools_of(b, 2, 7), dev(np.zeros((2, 3))), dev([1, 1])
    t, k, cu = dev(b.table), dev([30, 20]), dev([0, 10, 15])
    sa.paged_keep([], t, k, cu, path, count)
    sa.paged_keep(pools, t, k, cu, path[:, :0].contiguous(), count)
    for args in ((pools, t, k, cu, path[:1], count), (pools, t, k, cu, path, count[:1]), (pools, t, k, cu[:2], path, count),
                 (pools + [pools[0][:-1]], t, k, cu, path, count), (pools + [pools[0].cpu()], t, k, cu, path, count),
                 (pools * 40, t, k, cu, path, count), ([pools[0][0]], t, k, cu, path, count), (pools, t, k[:1], cu, path, count),
                 (pools + [pools[0].transpose(2, 3)], t, k, cu, path, count)):
        with pytest.raises((ValueError, sa._lib.G4AError)):
            sa.paged_keep(*args)
    with pytest.raises(sa._lib.G4AError, match="share memory"):
        sa.paged_keep(pools + pools[:1], t, k, cu, path, count)
    with pytest.raises(sa._lib.G4AError, match="multiple of 16"):
        sa.paged_keep([torch.zeros(b.n_pages, 16, 3, device="cuda")], t, k, cu, path, count)


# ---------------------------------------------------------------- paged_fork
def fork(pools, table, keys, parent, free, room, n_pages, page, **kw):
    free_t = np.full(n_pages, -1)
    free_t[:len(free)] = free
    kw = dict(dict(workspace=sa.Workspace(), room=room), **kw)
    if not pools:
        kw.update(n_pages=n_pages, page_size=page)
    return sa.paged_fork(pools, dev(table), dev(keys), dev(parent), dev(free_t), dev([len(free)]), **kw)


def beams(groups, W, prompts, grown, page, seed, spare=None, room=1):
    """Tables of groups of beams that share their prompts' full pages, each with pages of its own behind them."""
    r = np.random.default_rng(seed)
    n = groups * W
    keys = np.array([prompts[j // W] + grown[j // W] for j in range(n)])
    cols = max(1, int(keys.max() + room + page - 1) // page) + 1
    table, used = np.full((n, cols), -1, np.int64), 0
    for j in range(n):
        first, last = prompts[j // W] // page, -(-int(keys[j]) // page)
        if j % W == 0:
            table[j, :first] = np.arange(used, used + first)
            used += first
        table[j, :first] = table[j - j % W, :first]
        table[j, first:last] = np.arange(used, used + last - first)
        used += last - first
    n_pages = used + (n * (2 + room // page) if spare is None else spare)
    perm = r.permutation(n_pages)
    return np.where(table >= 0, perm[np.maximum(table, 0)], -1), keys, list(perm[used:]), n_pages


def check_fork(pools, table, keys, parent, free, room, n_pages, page, **kw):
    want = OB.fork([p.cpu().numpy() for p in pools], table, keys, parent, free, room, page, n_pages)
    got = fork(pools, table, keys, parent, free, room, n_pages, page, **kw)
    assert np.array_equal(got[0].cpu().numpy(), want[0])
    assert got[1].tolist() == want[1]
    assert got[3].tolist() == [len(want[2])]
    assert got[2].tolist() == [int(x) for x in want[2]] + [-1] * (n_pages - len(want[2]))
    for p, w in zip(pools, want[3]):
        assert np.array_equal(p.cpu().numpy(), w)
    return got


class Pages:
    def __init__(self, n_pages, page):
        self.n_pages, self.page = n_pages, page


@pytest.mark.parametrize("groups,W", [(1, 1), (1, 4), (5, 3), (40, 8), (130, 16)])
@pytest.mark.parametrize("room", [0, 1, 40])
@pytest.mark.parametrize("page", [16, 64])
def test_fork(groups, W, room, page):
    r = np.random.default_rng(groups + room)
    prompts, grown = r.integers(0, 100, groups), r.integers(0, 50, groups)
    grown[0] = (-prompts[0]) % page  # a group whose pages are just full
    table, keys, free, n_pages = beams(groups, W, prompts, grown, page, groups, room=room)
    parent = np.arange(groups * W) // W * W + r.integers(0, W, groups * W)
    pools = pools_of(Pages(n_pages, page), 2 if groups < 40 else 1, 3, ((1, 256, torch.float16), (1, 64, torch.float32)))
    check_fork(pools, table, keys, parent, free, room, n_pages, page)


def test_fork_of_a_prompt():
    """One prompt becomes sixteen beams; ones that follow nobody are idle; rows that do not branch stay as they are."""
    table, keys, free, n_pages = beams(3, 1, [37, 100, 5], [0, 0, 0], 16, 1, spare=60)
    pools = pools_of(Pages(n_pages, 16), 1, 3)
    got = check_fork(pools, table, keys, [0] * 16 + [1, -1, 2, 3, 2 ** 31 - 1, -2 ** 31], free, 1, n_pages, 16)
    assert got[1].tolist() == [37] * 16 + [100, 0, 5, 0, 0, 0]
    assert got[0][16].tolist()[:7] == table[1][:7].tolist()


def test_fork_shares_no_page_that_is_written():
    """A page that one row fills and another only partly has (sequences of one prefix) is not written to by the latter."""
    table = np.array([[0, 1, 2, -1], [0, 1, -1, -1], [3, 4, 5, -1]])
    keys, free = [40, 20, 33], [6, 7, 8, 9]
    for parent in ([0, 1, 2], [1, 1, 1], [2, 0, 1], [1, 0, 0]):
        pools = pools_of(Pages(10, 16), 1, 3)
        check_fork(pools, table, keys, parent, free, 1, 10, 16)


def test_fork_missing_pages():
    """Pages that are not there stay so (behind a window; a filled one that was lost); entries that name no page are none."""
    table = np.array([[-1, -1, 3, 4, -1], [2 ** 31 - 1, 10, 5, -1, -1], [-5, 6, -1, -1, -1]])
    for parent in ([0, 1, 2], [0, 0, 0, 1, 1, 2, 2]):
        pools = pools_of(Pages(10, 16), 1, 3)
        check_fork(pools, table, [60, 40, 40], parent, [0, 1, 2, 7, 8, 9], 1, 10, 16)


@pytest.mark.parametrize("free", [[], [7], [7, 8, 9]])
def test_fork_without_enough_pages(free):
    """The last columns that need a page have none; the ones that are freed by this very step count."""
    table = np.array([[0, 1, -1], [2, 3, -1], [4, 5, -1]])
    for parent in ([0, 0, 0, 0, 0], [0, 0, 0], [1, 2, 1]):
        pools = pools_of(Pages(10, 16), 1, 3)
        check_fork(pools, table, [20, 25, 30], parent, free, 30, 10, 16)


def test_fork_of_lists_that_are_none():
    """A count outside the list is cut to it; entries that name no page give none."""
    table, keys = np.array([[0, 1, -1], [2, 3, -1]]), [20, 25]
    for free, count in (([5, 6], -3), ([99, -7, 2 ** 31 - 1] + [-1] * 7, 10 ** 9)):
        free_t = np.full(10, -1)
        free_t[:len(free)] = free
        got = sa.paged_fork(pools_of(Pages(10, 16), 1, 3), dev(table), dev(keys), dev([0, 0, 0]), dev(free_t), dev([count]),
                            workspace=sa.Workspace())
        assert got[0][0].tolist() == [0, 1, -1] and 0 <= got[3].item() <= 10
        assert all(-1 <= p < 10 for p in got[0].flatten().tolist())


def test_fork_tables_alone():
    table, keys, free, n_pages = beams(4, 4, [20, 30, 40, 50], [3, 14, 15, 9], 16, 2)
    check_fork([], table, keys, np.arange(16) // 4 * 4 + np.arange(16)[::-1] % 4, free, 1, n_pages, 16)


def test_fork_many_pages_and_long_tables():
    """More pages than one step of a workgroup's list; tables of thousands of columns, rows further apart than that."""
    page, n = 16, 6
    table, keys, free, n_pages = beams(2, 3, [40000, 33000], [100, 5], page, 2, spare=60000)
    wide = np.full((n, table.shape[1] + 37), 12345)
    wide[:, :table.shape[1]] = table
    parent = [1, 1, 0, 5, 5, 5]
    want = OB.fork([], table, keys, parent, free, 1, page, n_pages)
    free_t = np.full(n_pages, -1)
    free_t[:len(free)] = free
    got = sa.paged_fork([], dev(wide)[:, :table.shape[1]], dev(keys), dev(parent), dev(free_t), dev([len(free)]), workspace=sa.Workspace(),
                        n_pages=n_pages, page_size=page)
    assert np.array_equal(got[0].cpu().numpy(), want[0]) and got[3].item() == len(want[2])
    assert got[2].tolist()[:len(want[2])] == [int(x) for x in want[2]]


def test_fork_refused():
    table, keys, free, n_pages = beams(1, 2, [20], [3], 16, 2)
    pools = pools_of(Pages(n_pages, 16), 1, 3)
    fr = np.full(n_pages, -1)
    fr[:len(free)] = free
    a = dict(pools=pools, page_table=dev(table), key_len=dev(keys), parent=dev([0, 0]), free_pages=dev(fr), n_free=dev([len(free)]),
             workspace=sa.Workspace())
    out = sa.paged_fork(**a)
    assert torch.equal(sa.paged_fork(**dict(a, parent=a["parent"].view(1, 2)))[0], out[0])
    for over in (dict(parent=a["parent"].long()), dict(parent=a["parent"].cpu()), dict(free_pages=a["free_pages"][:-1]),
                 dict(n_free=dev([1, 2])), dict(room=-1), dict(room=2 ** 31), dict(out=[x[:1] for x in out]), dict(pools=[]),
                 dict(n_pages=3), dict(page_size=64), dict(parent=a["parent"][:0]), dict(key_len=a["key_len"][:1])):
        with pytest.raises(ValueError):
            sa.paged_fork(**dict(a, **over))
    with pytest.raises(sa._lib.G4AError, match="overlap"):
        sa.paged_fork(**dict(a, out=(out[0], out[1], a["free_pages"], out[3])))
    with pytest.raises(RuntimeError):
        sa.paged_fork(**dict(a, workspace=sa.Workspace().reserve(256)))


# ---------------------------------------------------------------- beam_select
def select(logits, scores, **kw):
    d = lambda x: None if x is None else torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
    kw = dict(dict(workspace=sa.Workspace()), **kw)
    if kw.get("done") is not None:
        kw["done"] = d(kw["done"])
    return [x.cpu().numpy() for x in sa.beam_select(d(logits), d(scores), **kw)]


def check_select(logits, scores, what="", n_out=None, cap=0.0, done=None, pad=0, got=None):
    """Tokens and parents as in 64 bits. A score is off by the f32 sum of its row's exponentials (each within 2^-21: the
    argument's f32 rounding at |x'| below 88, exp2 and cap's quotient; sums of 32 + 6 terms) and by one rounding to f32."""
    n_out = n_out or scores.shape[1]
    want = OB.select(logits, scores, cap, n_out, done, pad)
    if got is None:
        got = select(logits, scores, n_out=n_out, cap=cap, done=done, pad=pad)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2]), what
    fin = np.isfinite(want[0])
    assert np.array_equal(np.isfinite(got[0]), fin)
    assert (np.abs(got[0][fin] - want[0][fin]) <= (2.0 ** -16 if cap else 2.0 ** -18) + 2.0 ** -23 * np.abs(want[0][fin])).all(), what


def rows(n, V, seed, dtype=np.float32, spread=3.0):
    return (spread * np.random.default_rng(seed).standard_normal((n, V))).astype(dtype)


@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 511, 512, 513, 1000, 4097, 50001])
@pytest.mark.parametrize("W", [1, 3, 8])
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_select(V, W, dtype):
    for seed, (n_out, cap) in enumerate(((W, 0.0), (2 * W, 30.0), (1, 5.0))):
        s = -np.random.default_rng(seed).random((3, W)).astype(np.float32) * 4
        check_select(rows(3 * W, V, seed + V, dtype), s, f"n_out {n_out}", n_out=n_out, cap=cap)


@pytest.mark.parametrize("W,n_out", [(64, 64), (64, 1), (1, 64), (33, 50), (5, 64)])
def test_select_widest(W, n_out):
    check_select(rows(2 * W, 3001, 1), -np.random.default_rng(2).random((2, W)).astype(np.float32), n_out=n_out)


def test_select_large():
    """Long rows: the parts of 2048 tokens; one far from the others' scores."""
    V, W = 262144, 8
    x = rows(5 * W, V, 3)
    x[7, V - 1] = 40.0
    x[11, 0] = 60.0
    for cap in (0.0, 30.0):
        check_select(x, -np.random.default_rng(2).random((5, W)).astype(np.float32), n_out=16, cap=cap)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_select_ties(dtype):
    """Equal logits: lowest token first, however many; equal beams: lowest beam first; -0 is 0."""
    for V, W, n_out in ((5000, 4, 8), (262144, 16, 64), (100, 2, 64)):
        check_select(np.zeros((W, V), dtype), np.zeros((1, W), np.float32), "all equal", n_out=n_out)
        x = np.zeros((W, V), dtype)
        x[:, ::2] = -0.0
        check_select(x, np.zeros((1, W), np.float32), "signed zeros", n_out=n_out)
        x = np.tile(rows(1, V, 5, dtype), (W, 1)).round(1 if dtype is np.float32 else 0).astype(dtype)
        check_select(x, np.zeros((1, W), np.float32), "equal beams", n_out=n_out)
    ramp = np.arange(4096, dtype=dtype)[None] / 64
    check_select(ramp, np.zeros((1, 1), np.float32), "ascending", n_out=64)
    check_select(ramp[:, ::-1].copy(), np.zeros((1, 1), np.float32), "descending", n_out=64)


def test_select_first_step_and_done():
    """Beams of score -inf have no candidates; finished ones have one; what nothing fills."""
    W, V = 4, 700
    s = np.full((2, W), -np.inf, np.float32)
    s[:, 0] = 0
    check_select(rows(2 * W, V, 1), s, "first", n_out=2 * W)
    s = np.array([[-1, -2, -3, -4], [-0.5, -np.inf, -3, -9]], np.float32)
    for done in ([[1, 0, 0, 1], [0, 1, 1, 1]], [[1] * 4, [1] * 4]):
        check_select(rows(2 * W, V, 2), s, "done", n_out=2 * W, done=np.array(done, bool), pad=3)
    check_select(rows(2 * W, 1, 2), s, "one token", n_out=2 * W)
    check_select(rows(2 * W, V, 2), np.full((2, W), -np.inf, np.float32), "nothing", n_out=3)


@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_select_what_is_not_finite(cap):
    """-inf and NaN logits are no tokens, +inf takes the weight; scores that are NaN count for nothing."""
    x = rows(6, 900, 4)
    x[0, :] = -np.inf
    x[1, 5:] = -np.inf
    x[2, ::3] = np.nan
    x[3, [7, 400, 800]] = np.inf
    x[4, :] = np.nan
    check_select(x, np.zeros((1, 6), np.float32), n_out=12, cap=cap)
    s = np.array([[0, np.nan, -1, 0.5, 0, np.inf]], np.float32)
    got = select(x, s, n_out=12, cap=cap)
    assert got[0][0, 0] == np.inf and got[1][0, 0] == 5 and not np.isnan(got[0]).any() and not (got[1] == 1).any()


def test_select_lowest_values():
    """Rows masked with the type's lowest value, and rows of nothing else."""
    for dtype in (np.float32, np.float16):
        x = rows(2, 500, 4, dtype)
        x[0, 10:] = np.finfo(dtype).min
        x[1] = np.finfo(dtype).min
        check_select(x, np.zeros((1, 2), np.float32), n_out=20)
        check_select(x, np.zeros((1, 2), np.float32), n_out=20, cap=30.0)


def test_select_strided_rows():
    """Rows that lie apart and begin anywhere: a padded vocabulary, of which the pad is never read as a token."""
    for dtype in (np.float32, np.float16):
        for V, stride in ((1001, 1003), (500, 513), (4090, 4096)):
            x = np.full((6, stride), np.inf, dtype)
            x[:, :V] = rows(6, V, V, dtype)
            t = torch.from_numpy(x).cuda()[:, :V]
            got = [y.cpu().numpy() for y in sa.beam_select(t, torch.zeros(2, 3, device="cuda"), workspace=sa.Workspace())]
            check_select(x[:, :V], np.zeros((2, 3), np.float32), got=got)


def test_select_refused():
    w, x, s = sa.Workspace(), torch.zeros(6, 100, device="cuda"), torch.zeros(2, 3, device="cuda")
    for args, kw in (((x[:5], s), {}), ((x.double(), s), {}), ((x, s.view(6)), {}), ((x.t(), s), {}), ((x, s.half()), {}), ((x.cpu(), s), {}),
                     ((x, s), dict(done=torch.zeros(6, dtype=torch.bool, device="cuda"))), ((x, s), dict(done=s)),
                     ((x, s), dict(out=(s, s, s)))):
        with pytest.raises(ValueError):
            sa.beam_select(*args, workspace=w, **kw)
    for kw in (dict(n_out=65), dict(n_out=0), dict(cap=-1.0), dict(cap=float("inf")), dict(cap=float("nan")),
               dict(done=s > 0, pad=100), dict(done=s > 0, pad=-1)):
        with pytest.raises(sa._lib.G4AError):
            sa.beam_select(x, s, workspace=w, **kw)
    with pytest.raises(sa._lib.G4AError):
        sa.beam_select(torch.zeros(65, 4, device="cuda"), torch.zeros(1, 65, device="cuda"), workspace=w)
    with pytest.raises(RuntimeError):
        sa.beam_select(x, s, workspace=sa.Workspace().reserve(256))
    assert sa.beam_select(x[:0], s[:0], workspace=w)[0].shape == (0, 3)
