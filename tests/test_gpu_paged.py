"""The paged cache's operators against their float64 definition: types, head layouts, lengths from
nothing to several splits, windows, missing pages, poisoned rows, and what must stay untouched."""
import numpy as np
import pytest
import torch

import oracle.paged as OP
import slang_amd as sa
from paged_cases import Batch, bound, check

pytestmark = pytest.mark.gpu


def ws():
    return sa.Workspace()


def write(b, d, rows=None, **kw):
    k, v = rows if rows is not None else (d["k_new"], d["v_new"])
    sa.paged_write(k, v, d["k_pages"], d["v_pages"], d["table"], d["key_len"], d["cu"], b.cfg(), k_gain=d["k_gain"],
                   rope_cos=d["cos"], rope_sin=d["sin"], **kw)


def decode(b, d, append=False, **kw):
    new = dict(k_new=d["k_new"], v_new=d["v_new"], k_gain=d["k_gain"]) if append else {}
    kw = dict(dict(q_gain=d["gain"], rope_cos=d["cos"], rope_sin=d["sin"], workspace=ws()), **new, **kw)
    return sa.paged_decode(d["q"], d["k_pages"], d["v_pages"], d["table"], d["key_len"], kw.pop("cfg", b.cfg()), **kw)


def prefill(b, d, **kw):
    kw = dict(dict(q_gain=d["gain"], rope_cos=d["cos"], rope_sin=d["sin"], workspace=ws()), **kw)
    return sa.paged_prefill(d["q"], d["k_pages"], d["v_pages"], d["table"], d["key_len"], d["cu"],
                            kw.pop("cfg", b.cfg()), **kw)


def bits(x):
    return x.detach().cpu().contiguous().view(torch.uint8).numpy()


# ---------------------------------------------------------------- paged_write
@pytest.mark.parametrize("hd,kvh", [(256, 1), (256, 2), (512, 1), (256, 8), (512, 3)])
@pytest.mark.parametrize("rows", ["f16", "f32"])
@pytest.mark.parametrize("kv", [np.float16, np.float32])
def test_write_rows_are_kv_writes(hd, kvh, rows, kv):
    """Every row that kv_write would store for the token, to the bit, at its page; nothing else."""
    b = Batch([40, 0, 17, 1, 130, 16], [40, 0, 5, 1, 33, 1], hd=hd, kvh=kvh, kv=kv, pad=3, missing=[(0, 1), (4, 8)], seed=hd + kvh)
    d = b.dev()
    t = torch.float16 if rows == "f16" else torch.float32
    k, v = d["k_new"].to(t), d["v_new"].to(t)
    want_k, want_v = b.k_pages.copy(), b.v_pages.copy()
    cfg = sa.AttnConfig(kvh, kvh, hd)
    dense = [torch.zeros(b.T, kvh, hd, dtype=d["k_pages"].dtype, device="cuda") for _ in range(2)]
    pos = torch.tensor([0 if x is None else x[1] for x in b.tokens()], device="cuda")
    sa.kv_write(k, v, *dense, 0, sa.AttnConfig(kvh, kvh, hd), k_gain=d["k_gain"], rope_cos=d["cos"][pos].contiguous(),
                rope_sin=d["sin"][pos].contiguous(), k_in_q=0.03, v_in_q=0.05)
    rk, rv = (x.cpu().numpy() for x in dense)
    for i, tok in enumerate(b.tokens()):
        if tok is None:
            continue
        _, row = OP.keys_of(b.table, tok[0], tok[1], b.page, b.n_pages, 1)
        if len(row):
            want_k.reshape(-1, kvh, hd)[row[0]] = rk[i]
            want_v.reshape(-1, kvh, hd)[row[0]] = rv[i]
    sa.paged_write(k, v, d["k_pages"], d["v_pages"], d["table"], d["key_len"], d["cu"], cfg, k_gain=d["k_gain"],
                   rope_cos=d["cos"], rope_sin=d["sin"], k_in_q=0.03, v_in_q=0.05)
    assert np.array_equal(d["k_pages"].cpu().numpy().view(np.uint8), want_k.view(np.uint8))
    assert np.array_equal(d["v_pages"].cpu().numpy().view(np.uint8), want_v.view(np.uint8))


def test_write_plain_rows():
    """No gain, no RoPE, no v norm: the rows as they are, against float64."""
    b = Batch([9, 33], [9, 2], kv=np.float32)
    d = b.dev()
    sa.paged_write(d["k_new"], d["v_new"], d["k_pages"], d["v_pages"], d["table"], d["key_len"], d["cu"], b.cfg(), v_norm=False)
    for i, (s, p) in enumerate(b.tokens()):
        _, row = OP.keys_of(b.table, s, p, b.page, b.n_pages, 1)
        assert np.array_equal(d["k_pages"].cpu().numpy().reshape(-1, 2, 256)[row[0]], b.k_new[i])
        assert np.array_equal(d["v_pages"].cpu().numpy().reshape(-1, 2, 256)[row[0]], b.v_new[i])


def test_write_against_float64():
    b = Batch([70, 20], [70, 3], hd=512, kvh=1, kv=np.float32)
    d = b.dev()
    write(b, d)
    k, v = (d[n].cpu().numpy().reshape(-1, 1, 512) for n in ("k_pages", "v_pages"))
    for i, (s, p) in enumerate(b.tokens()):
        _, row = OP.keys_of(b.table, s, p, b.page, b.n_pages, 1)
        wk = OP.prep(b.k_new[i], b.k_gain, b.cos[p], b.sin[p])
        wv = OP.rms(b.v_new[i].astype(np.float64), 1e-6)
        # f32: the sum of squares (10 roundings deep), root, quotient, gain, rotation: under 24 half steps
        assert np.abs(k[row[0]] - wk).max() <= 24 * 2.0 ** -24 * np.abs(wk).max() * 1.5
        assert np.abs(v[row[0]] - wv).max() <= 24 * 2.0 ** -24 * np.abs(wv).max()


# ---------------------------------------------------------------- paged_decode
LENS = [0, 1, 2, 15, 16, 17, 64, 65, 300, 511, 512, 513, 700]


@pytest.mark.parametrize("append", [False, True])
@pytest.mark.parametrize("window", [0, 100, 16, 512])
@pytest.mark.parametrize("hd,kvh,kv", [(256, 2, np.float16), (256, 1, np.float32), (512, 1, np.float16), (512, 2, np.float32)])
def test_decode(hd, kvh, kv, window, append):
    b = Batch(LENS, [min(1, k) for k in LENS], hd=hd, kvh=kvh, kv=kv, window=window, written=not append, seed=window + hd)
    b.new = [1] * len(LENS)  # every sequence has a query; an idle one no key
    b.q, b.k_new, b.v_new = (np.random.default_rng(i).standard_normal((len(LENS), h, hd)).astype(np.float32)
                             for i, h in ((1, 8), (2, kvh), (3, kvh)))
    d = b.dev()
    tokens = [(i, k - 1) for i, k in enumerate(LENS)]
    if append:  # the same rows through paged_write
        ref = b.dev()
        cu = torch.tensor(np.cumsum([0] + [min(1, k) for k in LENS]).astype(np.int32), device="cuda")
        live = [i for i, k in enumerate(LENS) if k]
        sa.paged_write(ref["k_new"][live].contiguous(), ref["v_new"][live].contiguous(), ref["k_pages"], ref["v_pages"],
                       ref["table"], ref["key_len"], cu, b.cfg(), k_gain=ref["k_gain"], rope_cos=ref["cos"],
                       rope_sin=ref["sin"])
        b.k_pages, b.v_pages = ref["k_pages"].cpu().numpy(), ref["v_pages"].cpu().numpy()
    out, A, S = b.oracle(tokens=tokens)
    for dt in (torch.float16, torch.float32):
        got = decode(b, d, append, out_dtype=dt)
        check(got.cpu().numpy(), out, bound(out, A, S, q16=False, kv32=kv is np.float32, out16=dt is torch.float16), f"{dt}")
        if append:
            assert np.array_equal(bits(d["k_pages"]), b.k_pages.reshape(-1).view(np.uint8).reshape(bits(d["k_pages"]).shape))
            assert np.array_equal(bits(d["v_pages"]), b.v_pages.reshape(-1).view(np.uint8).reshape(bits(d["v_pages"]).shape))


@pytest.mark.parametrize("kvh", [1, 2, 4, 8])
@pytest.mark.parametrize("hd", [256, 512])
@pytest.mark.parametrize("page", [16, 64, 1024])
def test_decode_groups_and_pages(hd, kvh, page):
    keys = [5, 260, 1100]
    b = Batch(keys, [1] * 3, hd=hd, kvh=kvh, page=page, seed=kvh)
    out, A, S = b.oracle()
    got = decode(b, b.dev())
    check(got.cpu().numpy(), out, bound(out, A, S, q16=False, kv32=False, out16=True))


@pytest.mark.parametrize("keys", [1, 16, 17, 250, 1500])
@pytest.mark.parametrize("window", [0, 130])
def test_decode_one_sequence(keys, window):
    b = Batch([keys], [1], kvh=2, window=window, written=True)
    out, A, S = b.oracle()
    for bnd in (keys, MAX):  # a tight host bound, and a loose one
        got = decode(b, b.dev(table=torch.from_numpy(np.pad(b.table, ((0, 0), (0, 200)), constant_values=-1)).cuda()), max_key_len=bnd)
        check(got.cpu().numpy(), out, bound(out, A, S, q16=False, kv32=False, out16=True), f"max_key_len {bnd}")


MAX = 2048


@pytest.mark.parametrize("hd", [256, 512])
def test_decode_missing_pages(hd):
    """Pages that are not there hold no key: single ones, all of a sequence, the last one of an append."""
    keys = [100, 48, 33, 200, 16]
    missing = [(0, 0), (0, 3), (1, 0), (1, 1), (1, 2), (2, 2), (3, 5), (3, 6), (3, 7), (3, 12)]
    b = Batch(keys, [1] * 5, hd=hd, kvh=1, missing=missing)
    out, A, S = b.oracle()
    assert (out[1] == 0).all()
    got = decode(b, b.dev())
    check(got.cpu().numpy(), out, bound(out, A, S, q16=False, kv32=False, out16=True))
    d = b.dev()
    before = bits(d["k_pages"])
    got = decode(b, d, append=True)  # sequences 2 and 3 append to a page that is not there: dropped
    changed = (bits(d["k_pages"]) != before).reshape(b.n_pages, 16, -1).any(-1)
    want = np.zeros_like(changed)
    for s in (0, 4):
        p = keys[s] - 1
        want[b.table[s, p // 16], p % 16] = True
    assert np.array_equal(changed, want)
    check(got[[2, 3]].cpu().numpy(), out[[2, 3]], bound(out, A, S, q16=False, kv32=False, out16=True)[[2, 3]])


def test_decode_infinite_and_lowest_rows_outside():
    """Rows beyond the length, in front of the window and on foreign pages may hold anything."""
    b = Batch([37, 90], [1, 1], window=20)
    out, A, S = b.oracle()
    for junk in (np.inf, -np.inf, -65504.0, np.nan):
        k, v = b.k_pages.copy(), b.v_pages.copy()
        k[np.isnan(b.k_pages)] = junk
        v[np.isnan(b.v_pages)] = junk
        t = lambda x: torch.from_numpy(x).cuda()  # noqa: E731
        got = decode(b, b.dev(k_pages=t(k), v_pages=t(v)))
        check(got.cpu().numpy(), out, bound(out, A, S, q16=False, kv32=False, out16=True), f"{junk}")


def test_decode_options():
    """No norm, no RoPE, another scale, srq'd output."""
    b = Batch([200, 31], [1, 1], kvh=4)
    out, A, S = b.oracle(gain=False, rope=False, scale=0.0625)
    got = decode(b, b.dev(), q_gain=None, rope_cos=None, rope_sin=None, cfg=b.cfg(scale=0.0625), out_dtype=torch.float32)
    tol = bound(out, A, S, q16=False, kv32=False, out16=False)
    check(got.cpu().numpy(), out, tol)
    got = decode(b, b.dev(), q_gain=None, rope_cos=None, rope_sin=None, cfg=b.cfg(scale=0.0625, out_q=0.02))
    k = got.float().cpu().numpy() / 0.02
    assert np.abs(k - np.round(k)).max() <= 128 * 2.0 ** -11 + 1e-3  # on the grid, up to the f16 rounding
    check(got.cpu().numpy(), np.clip(out, -2.56, 2.54), tol + 0.0101 + 2.56 * 2.0 ** -11)


def test_decode_longer_than_the_bound():
    """A key_len beyond max_key_len is taken as max_key_len; a negative one as idle."""
    b = Batch([64, 40, 50], [1, 1, 1])
    d = b.dev(key_len=torch.tensor([10 ** 9, 40, -5], dtype=torch.int32, device="cuda"))
    out, A, S = b.oracle(tokens=[(0, 63), (1, 39), (2, -1)])
    got = decode(b, d, max_key_len=64)
    check(got.cpu().numpy(), out, bound(out, A, S, q16=False, kv32=False, out16=True))


# ---------------------------------------------------------------- paged_prefill
def run_prefill(b, kv32=False, dts=(torch.float16, torch.float32), what="", **kw):
    out, A, S = b.oracle()
    live = np.array([t is not None for t in b.tokens()])
    for dt in dts:
        d = b.dev()
        o = torch.full((max(1, b.T), b.nh, b.hd), 7.25, dtype=dt, device="cuda")
        got = prefill(b, d, out=o, **kw).cpu().numpy()
        check(got[live], out[live], bound(out, A, S, q16=True, kv32=kv32, out16=dt is torch.float16, k16=kv32)[live], f"{what} {dt}")
        assert (got[~live] == 7.25).all()
        assert np.array_equal(bits(d["k_pages"]).reshape(-1), b.k_pages.reshape(-1).view(np.uint8))
    return got


@pytest.mark.parametrize("window", [0, 100, 16])
@pytest.mark.parametrize("hd,kvh,kv", [(256, 2, np.float16), (256, 1, np.float32), (512, 1, np.float16), (512, 2, np.float32)])
def test_prefill(hd, kvh, kv, window):
    new = [1, 0, 33, 150, 16, 2, 64]
    hist = [0, 0, 100, 3, 240, 511, 0]
    b = Batch([a + h for a, h in zip(new, hist)], new, hd=hd, kvh=kvh, kv=kv, window=window, pad=5, seed=window)
    run_prefill(b, kv32=kv is np.float32)


@pytest.mark.parametrize("kvh", [1, 2, 4, 8])
@pytest.mark.parametrize("hd", [256, 512])
@pytest.mark.parametrize("page", [16, 128])
def test_prefill_groups_and_pages(hd, kvh, page):
    b = Batch([70, 129, 17], [70, 40, 17], hd=hd, kvh=kvh, page=page, seed=kvh)
    run_prefill(b, dts=(torch.float16,))


@pytest.mark.parametrize("hd,kvh", [(256, 2), (512, 1)])
@pytest.mark.parametrize("window", [0, 300])
def test_prefill_long_rows(hd, kvh, window):
    """Long histories beside short prompts: rows long enough to be cut into pieces."""
    b = Batch([1500, 20, 900, 1201], [40, 20, 130, 1], hd=hd, kvh=kvh, window=window, page=32)
    run_prefill(b, dts=(torch.float16,))


@pytest.mark.parametrize("hd", [256, 512])
def test_prefill_missing_pages(hd):
    b = Batch([100, 48, 150], [60, 48, 20], hd=hd, kvh=1, missing=[(0, 0), (0, 3), (1, 0), (1, 1), (1, 2), (2, 4), (2, 5), (2, 9)])
    got = run_prefill(b, dts=(torch.float16,))
    assert (got[60:108] == 0).all()


@pytest.mark.parametrize("hd", [256, 512])
@pytest.mark.parametrize("window", [0, 50])
def test_prefill_masked_keys_may_be_anything(hd, window):
    """K rows that a token does not attend (later tokens' ones, ones its window has left) do not reach it,
    whatever they hold; with V rows of the type's lowest value beside them."""
    b = Batch([150], [150], hd=hd, kvh=1, window=window)
    out, A, S = b.oracle()
    k, v = b.k_pages.copy(), b.v_pages.copy()
    at = b.table[0, 100 // 16], 100 % 16
    v[at] = -65504.0
    tokens = [i for i in range(150) if i < 100 or (window and i >= 100 + window)]
    for junk in (np.inf, -np.inf, np.nan, 65504.0):
        k[at] = junk
        got = prefill(b, b.dev(k_pages=torch.from_numpy(k).cuda(), v_pages=torch.from_numpy(v).cuda())).cpu().numpy()
        check(got[tokens], out[tokens], bound(out, A, S, q16=True, kv32=False, out16=True)[tokens], f"{junk}")


def test_prefill_more_rows_than_keys():
    """Tokens at positions below zero attend nothing; offsets out of range are cut."""
    b = Batch([30, 20], [30, 20])
    b.keys = [12, 20]
    toks = [(0, 12 - 30 + i) for i in range(30)] + [(1, i) for i in range(20)]
    out, A, S = b.oracle(tokens=toks)
    got = prefill(b, b.dev(key_len=torch.tensor([12, 20], dtype=torch.int32, device="cuda")))
    check(got.cpu().numpy(), out, bound(out, A, S, q16=True, kv32=False, out16=True))
    d = b.dev(cu=torch.tensor([0, 30, 1000], dtype=torch.int32, device="cuda"))
    got2 = prefill(b, dict(d, key_len=torch.tensor([12, 20], dtype=torch.int32, device="cuda")))
    check(got2.cpu().numpy(), out, bound(out, A, S, q16=True, kv32=False, out16=True))


@pytest.mark.parametrize("hd", [256, 512])
@pytest.mark.parametrize("n_seq", [3, 300])
def test_prefill_offsets_that_do_not_ascend(hd, n_seq):
    """Whatever the offsets, the cache stays, rows behind the packed ones stay, and a later call is right."""
    b = Batch([700, 640], [640, 20], hd=hd, kvh=1, pad=9)
    d = b.dev()
    cu = [0] + [(660, 0)[i % 2] for i in range(n_seq)]
    o = torch.full((b.T + 4, 8, hd), 7.25, dtype=torch.float16, device="cuda")
    w = ws()
    prefill(b, dict(d, table=d["table"][:1].repeat(n_seq, 1), key_len=d["key_len"][:1].repeat(n_seq),
                    cu=torch.tensor(cu, dtype=torch.int32, device="cuda")), out=o[:b.T], workspace=w)
    assert np.array_equal(bits(d["k_pages"]).reshape(-1), b.k_pages.reshape(-1).view(np.uint8))
    assert (o[660:] == 7.25).all()
    out, A, S = b.oracle()
    check(prefill(b, d, workspace=w).cpu().numpy()[:660], out[:660], bound(out, A, S, q16=True, kv32=False, out16=True)[:660])


def test_prefill_options():
    b = Batch([60, 33], [60, 9], kvh=4)
    out, A, S = b.oracle(gain=False, rope=False, scale=0.0625)
    got = prefill(b, b.dev(), q_gain=None, rope_cos=None, rope_sin=None, cfg=b.cfg(scale=0.0625), out_dtype=torch.float32)
    check(got.cpu().numpy(), out, bound(out, A, S, q16=True, kv32=False, out16=False))


@pytest.mark.parametrize("hd", [256, 512])
def test_prefill_no_tokens_at_all(hd):
    """Every sequence idle: nothing is written."""
    b = Batch([0, 0, 40], [0, 0, 0], hd=hd, pad=4)
    run_prefill(b, dts=(torch.float16,))


# ---------------------------------------------------------------- as they are used
@pytest.mark.parametrize("hd,kvh,window,kv", [(256, 1, 64, np.float16), (512, 1, 0, np.float16), (256, 2, 0, np.float32)])
def test_prompts_then_tokens(hd, kvh, window, kv):
    """Prompts written and attended in two calls each, then tokens generated, against float64 on the
    rows the cache holds; pages behind the window are given back on the way."""
    r = np.random.default_rng(3)
    prompt, steps, page = [70, 1, 129, 16], 5, 16
    n = len(prompt)
    full = Batch([p + steps for p in prompt], [0] * n, hd=hd, kvh=kvh, window=window, kv=kv, page=page)
    full.k_pages[:] = np.nan
    full.v_pages[:] = np.nan
    d = full.dev()
    w = ws()
    done = [0] * n
    for part in (0.6, 1.0):  # each prompt in two pieces
        new = [int(round(p * part)) - x for p, x in zip(prompt, done)]
        done = [x + y for x, y in zip(done, new)]
        T = sum(new)
        x = [torch.from_numpy(r.standard_normal((T, h, hd)).astype(np.float32)).cuda() for h in (8, kvh, kvh)]
        d["key_len"].copy_(torch.tensor(done, dtype=torch.int32))
        cu = torch.tensor(np.cumsum([0] + new).astype(np.int32), device="cuda")
        dd = dict(d, q=x[0], k_new=x[1], v_new=x[2], cu=cu)
        write(full, dd)
        got = prefill(full, dd, workspace=w)
        toks = [(b, done[b] - new[b] + i) for b in range(n) for i in range(new[b])]
        out, A, S = full.oracle(q=x[0].cpu().numpy(), tokens=toks, k_pages=d["k_pages"].cpu().numpy(), v_pages=d["v_pages"].cpu().numpy())
        check(got.cpu().numpy(), out, bound(out, A, S, q16=True, kv32=kv is np.float32, out16=True, k16=kv is np.float32), f"part {part}")
    for step in range(steps):
        done = [x + 1 for x in done]
        d["key_len"].add_(1)
        if window:
            for b in range(n):
                full.table[b, :max(0, done[b] - window) // page] = -1
            d["table"].copy_(torch.from_numpy(full.table))
        x = [torch.from_numpy(r.standard_normal((n, h, hd)).astype(np.float32)).cuda() for h in (8, kvh, kvh)]
        got = decode(full, dict(d, q=x[0], k_new=x[1], v_new=x[2]), append=True, workspace=w)
        out, A, S = full.oracle(q=x[0].cpu().numpy(), tokens=[(b, done[b] - 1) for b in range(n)],
                                k_pages=d["k_pages"].cpu().numpy(), v_pages=d["v_pages"].cpu().numpy())
        check(got.cpu().numpy(), out, bound(out, A, S, q16=False, kv32=kv is np.float32, out16=True), f"step {step}")


def test_shared_prefix_pages():
    """Two sequences over the same first pages."""
    b = Batch([80, 90], [1, 1])
    b.table[1, :4] = b.table[0, :4]
    out, A, S = b.oracle()
    check(decode(b, b.dev()).cpu().numpy(), out, bound(out, A, S, q16=False, kv32=False, out16=True))


def test_pool_past_4_gib():
    """Pages whose byte offsets pass 32 bits, first and last ones used."""
    page, hd = 64, 256
    n_pages = (5 << 30) // (page * 2 * hd * 2)
    b = Batch([200, 130], [100, 1], page=page)
    kp = torch.zeros(n_pages, page, 2, hd, dtype=torch.float16, device="cuda")
    vp = torch.zeros_like(kp)
    small = b.dev()
    ids = torch.arange(n_pages - b.n_pages, n_pages, device="cuda")
    kp[ids] = small["k_pages"]
    vp[ids] = small["v_pages"]
    tab = torch.where(small["table"] >= 0, small["table"] + (n_pages - b.n_pages), small["table"]).to(torch.int32)
    d = dict(small, k_pages=kp, v_pages=vp, table=tab)
    out, A, S = b.oracle()
    got = prefill(b, d)
    check(got.cpu().numpy(), out, bound(out, A, S, q16=True, kv32=False, out16=True))
    dt = dict(d, q=d["q"][[99, 100]].contiguous())
    got = decode(b, dt)
    check(got.cpu().numpy(), out[[99, 100]], bound(out, A, S, q16=False, kv32=False, out16=True)[[99, 100]])
    write(b, d)
    ref = b.dev()
    write(b, ref)
    assert torch.equal(kp[ids].view(torch.int16), ref["k_pages"].view(torch.int16))
    assert not kp[:n_pages - b.n_pages].any()


def test_table_rows_apart():
    """page_table as the first columns of a wider table."""
    b = Batch([80, 50], [1, 1])
    wide = torch.full((2, 40), -1, dtype=torch.int32, device="cuda")
    wide[:, :b.cols] = torch.from_numpy(b.table).cuda()
    out, A, S = b.oracle()
    d = b.dev(table=wide[:, :b.cols])
    check(decode(b, d).cpu().numpy(), out, bound(out, A, S, q16=False, kv32=False, out16=True))
    check(prefill(b, d).cpu().numpy(), out, bound(out, A, S, q16=True, kv32=False, out16=True))


def test_numbers_and_tables_of_other_kinds():
    """Steps as numpy numbers; a single column taken out of a transposed table."""
    b = Batch([80, 50], [1, 1], page=128, extra_cols=0)
    d, ref = b.dev(), b.dev()
    column = torch.stack([ref["table"][:, 0], ref["table"][:, 0]]).t()[:, :1]
    assert column.shape == (2, 1) and column.stride(1) != 1
    steps = dict(k_in_q=np.float32(0.03), v_in_q=np.float32(0.05))
    plain = {n: float(v) for n, v in steps.items()}
    write(b, dict(d, table=column), **steps)
    write(b, ref, **plain)
    assert np.array_equal(bits(d["k_pages"]), bits(ref["k_pages"])) and np.array_equal(bits(d["v_pages"]), bits(ref["v_pages"]))
    assert torch.equal(decode(b, dict(d, table=column), True, **steps), decode(b, ref, True, **plain))
    assert torch.equal(prefill(b, dict(d, table=column)), prefill(b, ref))


@pytest.mark.parametrize("hd,kvh", [(256, 2), (512, 1)])
def test_captured_steps(hd, kvh):
    """Write, prefill and decode captured once and replayed on new lengths, tables and rows, with
    eager calls and synchronisations between; each replay equals the eager call to the bit."""
    b = Batch([150, 60, 1300], [50, 60, 33], hd=hd, kvh=kvh)
    d = b.dev()
    sizes = dict(page_size=16)
    w = sa.Workspace().reserve(max(sa.paged_decode_ws_bytes(3, MAX, b.cfg(), **sizes),
                                   sa.paged_prefill_ws_bytes(b.T, 3, MAX, b.cfg(), **sizes)))
    tab = torch.full((3, MAX // 16), -1, dtype=torch.int32, device="cuda")
    tab[:, :b.cols] = d["table"]
    d["table"] = tab
    qd = d["q"][:3].contiguous()
    out = torch.zeros(b.T, 8, hd, dtype=torch.float16, device="cuda")
    outd = torch.zeros(3, 8, hd, dtype=torch.float16, device="cuda")

    def steps():
        write(b, d, max_key_len=MAX)
        prefill(b, d, workspace=w, out=out, max_key_len=MAX)
        decode(b, dict(d, q=qd), workspace=w, out=outd, max_key_len=MAX)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        steps()
        stream.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            steps()
    for i, (keys, cu) in enumerate([([150, 60, 1300], b.cu), ([100, 10, 1111], [0, 20, 30, 143]), ([50, 0, 33], [0, 50, 50, 83])]):
        torch.cuda.synchronize()
        d["key_len"].copy_(torch.tensor(keys, dtype=torch.int32))
        d["cu"].copy_(torch.tensor(np.asarray(cu, np.int32)))
        d["q"].normal_()
        qd.copy_(d["q"][:3])
        out.zero_()
        outd.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            g.replay()
            stream.synchronize()
            got = out.clone(), outd.clone()
            out.zero_()
            outd.zero_()
            steps()
            stream.synchronize()
        assert torch.equal(got[0], out) and torch.equal(got[1], outd), f"replay {i}"
        assert torch.isfinite(out).all() and out[:int(cu[-1])].abs().sum() > 0


def test_two_streams():
    """Calls on two streams at once, each with its own workspace."""
    bs = [Batch([300, 900], [1, 1], seed=s) for s in (1, 2)]
    ds = [b.dev() for b in bs]
    streams, w = [torch.cuda.Stream() for _ in bs], [ws() for _ in bs]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                outs[i].append(decode(bs[i], ds[i], workspace=w[i]))
                outs[i].append(prefill(bs[i], ds[i], workspace=w[i]))
    torch.cuda.synchronize()
    for b, o in zip(bs, outs):
        out, A, S = b.oracle()
        for x in o:
            check(x.cpu().numpy(), out, bound(out, A, S, q16=True, kv32=False, out16=True))


def test_two_graphs_share_a_workspace():
    """A prefill and a decode captured over one workspace, replayed in turn."""
    b = Batch([1300, 60], [40, 60])
    d = b.dev()
    w = sa.Workspace().reserve(max(sa.paged_decode_ws_bytes(2, MAX, b.cfg(), page_size=16),
                                   sa.paged_prefill_ws_bytes(b.T, 2, MAX, b.cfg(), page_size=16)))
    qd = d["q"][:2].contiguous()
    outs = [torch.zeros(b.T, 8, 256, dtype=torch.float16, device="cuda"), torch.zeros(2, 8, 256, dtype=torch.float16, device="cuda")]
    calls = [lambda: prefill(b, d, workspace=w, out=outs[0]), lambda: decode(b, dict(d, q=qd), workspace=w, out=outs[1])]
    graphs, stream = [torch.cuda.CUDAGraph() for _ in calls], torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for g, call in zip(graphs, calls):
            call()
            stream.synchronize()
            with torch.cuda.graph(g, stream=stream):
                call()
        want = []
        for call, o in zip(calls, outs):
            call()
            want.append(o.clone())
        for i in range(6):
            for o in outs:
                o.zero_()
            for g in graphs[::1 if i % 2 else -1]:
                g.replay()
            stream.synchronize()
            assert all(torch.equal(o, x) for o, x in zip(outs, want)), f"replay {i}"


# ---------------------------------------------------------------- many sequences, long ones
def sparse_oracle(b, rows, **kw):
    """The oracle at some of the packed rows, and those rows."""
    toks = [t if i in rows else None for i, t in enumerate(b.tokens())]
    out, A, S = b.oracle(tokens=toks, **kw)
    return [x[list(rows)] for x in (out, A, S)]


@pytest.mark.parametrize("hd,keys", [(256, 40000), (512, 24000)])
def test_prefill_history_of_many_tiles(hd, keys):
    """A piece of a block walks more than 64 key tiles. (scale 0.25: weights within 2^13 of each other, so
    that no weight is subnormal and the bound's terms hold for any number of keys.)"""
    b = Batch([keys, 70], [37, 70], hd=hd, kvh=1, page=64, missing=[(0, 5), (0, keys // 64 - 30)])
    rows = (0, 1, 17, 36, 37, 106)
    out, A, S = sparse_oracle(b, rows, rope=False, scale=0.25)
    got = prefill(b, b.dev(), rope_cos=None, rope_sin=None, cfg=b.cfg(scale=0.25)).cpu().numpy()[list(rows)]
    check(got, out, bound(out, A, S, q16=True, kv32=False, out16=True))


@pytest.mark.parametrize("hd", [256, 512])
def test_prefill_blocks_of_many_tiles(hd):
    """So many tokens that no block is cut: the longest walk more than 64 tiles whole."""
    kt = 64 if hd == 256 else 32
    n, new = 30, 4000
    b = Batch([70 * kt], [1], hd=hd, kvh=1, page=64)
    q = torch.randn(n * new, 8, hd, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    key_len = torch.tensor([70 * kt - i for i in range(n)], dtype=torch.int32, device="cuda")
    new_i = [min(new, int(k)) for k in key_len]
    cu = np.concatenate([[0], np.cumsum(new_i)]).astype(np.int32)
    d = b.dev()
    out = prefill(b, dict(d, q=q, table=d["table"].repeat(n, 1), key_len=key_len, cu=torch.from_numpy(cu).cuda()),
                  rope_cos=None, rope_sin=None, cfg=b.cfg(scale=0.25))
    rows = [int(cu[s + 1]) - back for s in (0, 13, n - 1) for back in (1, 2, 700, new_i[s])]
    toks = [(0, int(key_len[s]) - back) for s in (0, 13, n - 1) for back in (1, 2, 700, new_i[s])]
    want, A, S = b.oracle(q=q[rows].cpu().numpy(), tokens=toks, rope=False, scale=0.25)
    check(out[rows].cpu().numpy(), want, bound(want, A, S, q16=True, kv32=False, out16=True))


@pytest.mark.parametrize("hd,window", [(512, 0), (512, 14000), (256, 0)])
def test_decode_splits_of_many_blocks(hd, window):
    """Enough keys for splits of more than 4096: a wave reloads its table entries."""
    keys, n = (16000, 64) if hd == 512 else (20000, 128)
    b = Batch([keys], [1], hd=hd, kvh=1, page=16, window=0, missing=[(0, 300), (0, keys // 16 - 9)])
    b.window = window
    q = torch.randn(n, 8, hd, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    key_len = torch.tensor([keys - 17 * i for i in range(n)], dtype=torch.int32, device="cuda")
    d = b.dev()
    got = decode(b, dict(d, q=q, table=d["table"].repeat(n, 1), key_len=key_len), rope_cos=None, rope_sin=None, cfg=b.cfg(scale=0.25))
    rows = [0, 1, 33, n - 1]
    want, A, S = b.oracle(q=q[rows].cpu().numpy(), tokens=[(0, int(key_len[i]) - 1) for i in rows], rope=False, scale=0.25)
    check(got[rows].cpu().numpy(), want, bound(want, A, S, q16=False, kv32=False, out16=True))


@pytest.mark.parametrize("n_seq", [65, 150])
@pytest.mark.parametrize("hd,kvh", [(256, 2), (512, 1)])
def test_decode_many_sequences(hd, kvh, n_seq):
    """More sequences than lanes, of every length; every fifth idle."""
    r = np.random.default_rng(n_seq)
    keys = [0 if i % 5 == 4 else int(x) for i, x in enumerate(r.integers(1, 700, n_seq))]
    b = Batch(keys, [1] * n_seq, hd=hd, kvh=kvh)
    out, A, S = b.oracle()
    check(decode(b, b.dev()).cpu().numpy(), out, bound(out, A, S, q16=False, kv32=False, out16=True))


@pytest.mark.parametrize("hd,kvh,kv", [(256, 2, np.float16), (512, 1, np.float16), (256, 1, np.float32)])
@pytest.mark.parametrize("n_seq", [65, 300])
def test_prefill_many_sequences(hd, kvh, kv, n_seq):
    """More sequences than lanes and than the plan takes at a time, short ones beside two long ones; rows
    written by the call before."""
    r = np.random.default_rng(n_seq)
    keys = [int(x) for x in r.integers(0, 40, n_seq)]
    new = [int(r.integers(0, 6)) if k > 6 else k for k in keys]
    for i, (k, m) in {3: (1500, 70), n_seq - 1: (1100, 3)}.items():
        keys[i], new[i] = k, m
    b = Batch(keys, new, hd=hd, kvh=kvh, kv=kv, pad=2)
    ref = b.dev()
    write(b, ref)
    d = b.dev()
    rows = torch.zeros(2, b.T, kvh, hd, dtype=d["k_pages"].dtype, device="cuda")
    pos = torch.tensor([0 if x is None else x[1] for x in b.tokens()], device="cuda")
    sa.kv_write(d["k_new"], d["v_new"], rows[0], rows[1], 0, sa.AttnConfig(kvh, kvh, hd), k_gain=d["k_gain"],
                rope_cos=d["cos"][pos].contiguous(), rope_sin=d["sin"][pos].contiguous())
    for i, x in enumerate(b.tokens()):
        if x is not None:
            row = OP.keys_of(b.table, x[0], x[1], b.page, b.n_pages, 1)[1][0]
            b.k_pages.reshape(-1, kvh, hd)[row], b.v_pages.reshape(-1, kvh, hd)[row] = rows[0, i].cpu().numpy(), rows[1, i].cpu().numpy()
    assert np.array_equal(bits(ref["k_pages"]).reshape(-1), b.k_pages.reshape(-1).view(np.uint8))
    assert np.array_equal(bits(ref["v_pages"]).reshape(-1), b.v_pages.reshape(-1).view(np.uint8))
    run_prefill(b, kv32=kv is np.float32, dts=(torch.float16,))


# ---------------------------------------------------------------- refusals
def test_refusals():
    b = Batch([40, 20], [1, 1])
    d = b.dev()
    run = lambda **k: decode(b, dict(d, **k))  # noqa: E731
    for bad in (dict(q=d["q"].half()), dict(q=d["q"][:1].contiguous()), dict(q=d["q"].cpu()), dict(table=d["table"].long()),
                dict(table=d["table"].cpu()), dict(table=d["table"].t()), dict(key_len=d["key_len"][:1].contiguous()),
                dict(key_len=d["key_len"].cpu()), dict(k_pages=d["k_pages"].float()), dict(k_pages=d["k_pages"][:, :, :1]),
                dict(cos=d["cos"][:30].contiguous()), dict(cos=None), dict(gain=d["gain"].double())):
        with pytest.raises(ValueError):
            run(**bad)
    with pytest.raises(ValueError):
        decode(b, d, max_key_len=10 ** 6)
    with pytest.raises(ValueError):
        decode(b, d, out=torch.empty(2, 8, 128, device="cuda"))
    with pytest.raises(ValueError):
        decode(b, dict(d, k_new=d["k_new"].half()), append=True)
    with pytest.raises(ValueError):
        prefill(b, dict(d, cu=d["cu"][:2].contiguous()))
    with pytest.raises(ValueError):
        write(b, d, rows=(d["k_new"], d["v_new"].half()))
    with pytest.raises(sa._lib.G4AError):  # pages of 24 rows
        decode(b, dict(d, k_pages=torch.zeros(9, 24, 2, 256, dtype=torch.float16, device="cuda"),
                       v_pages=torch.zeros(9, 24, 2, 256, dtype=torch.float16, device="cuda")))
    with pytest.raises(RuntimeError):  # a reserved workspace that is too small
        prefill(b, d, workspace=sa.Workspace().reserve(16))
    x = torch.zeros(2 * 8 * 256 * 4, dtype=torch.uint8, device="cuda")
    with pytest.raises(sa._lib.G4AError):  # out over q
        prefill(b, dict(d, q=x.view(torch.float32).view(2, 8, 256)), out=x[:2 * 8 * 256 * 2].view(torch.float16).view(2, 8, 256))
