"""The paged operators at the edges of what they accept: offsets out of order over tables of just the
rows that the keys need, rows that are not finite, empty calls, long contexts."""
import numpy as np
import pytest
import torch

import slang_amd as sa
from paged_cases import Batch, bound, check
from test_gpu_paged import bits, decode, prefill, write, ws

pytestmark = pytest.mark.gpu
MAX_KEYS = 2048


def i32(x):
    return torch.tensor([int(v) for v in x], dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("hd", [256, 512])
@pytest.mark.parametrize("cu", [[0, 660, 0, 0], [0, 500, 5, 10], [0, 660, 20, 640, 3]])
def test_prefill_offsets_out_of_order_stay_in_the_rope_tables(hd, cu):
    """Tables of max_key_len rows with NaN behind them: no row behind is read (a q row rotated by one
    would make its outputs NaN; rows without a q of their own keep the workspace's zeros)."""
    keys, n = 700, len(cu) - 1
    b = Batch([keys], [660], hd=hd, kvh=1, pad=0)
    d = b.dev()
    tables = []
    for x in (d["cos"], d["sin"]):
        t = torch.full((keys + 700, hd // 2), float("nan"), device="cuda")
        t[:keys] = x[:keys]
        tables.append(t[:keys])
    w = ws().reserve(sa.paged_prefill_ws_bytes(660, n, keys, b.cfg(), page_size=16))
    w.buf.zero_()
    out = torch.zeros(660, 8, hd, dtype=torch.float16, device="cuda")
    over = dict(d, table=d["table"][:1].repeat(n, 1), key_len=i32([keys] * n), cu=i32(cu))
    prefill(b, over, rope_cos=tables[0], rope_sin=tables[1], max_key_len=keys, workspace=w, out=out)
    assert torch.isfinite(out).all()
    assert np.array_equal(bits(d["k_pages"]).reshape(-1), b.k_pages.reshape(-1).view(np.uint8))
    want, A, S = b.oracle()
    got = prefill(b, d, rope_cos=tables[0], rope_sin=tables[1], max_key_len=keys, workspace=w)
    check(got.cpu().numpy(), want, bound(want, A, S, q16=True, kv32=False, out16=True))


# ---------------------------------------------------------------- rows that are not finite
@pytest.mark.parametrize("keys", [[100], [1500], [20, 1500, 700, 0, 90]])  # one split; splits; a work list
@pytest.mark.parametrize("hd,kvh,kv", [(256, 2, np.float16), (512, 1, np.float16), (256, 1, np.float32)])
@pytest.mark.parametrize("what", ["q", "q inf", "k", "v"])
def test_decode_shows_what_is_not_finite(hd, kvh, kv, keys, what):
    """A query head, or an attended K row or V value, that is not finite makes its outputs NaN and no other,
    however the keys are split: through pages and over contiguous caches."""
    b = Batch(keys, [min(1, k) for k in keys], hd=hd, kvh=kvh, kv=kv, extra_cols=0)
    n, G, s = len(keys), 8 // kvh, int(np.argmax(keys))
    b.q = np.random.default_rng(1).standard_normal((n, 8, hd)).astype(np.float32)
    tokens = [(i, k - 1) for i, k in enumerate(keys)]
    out, A, S = b.oracle(tokens=tokens)
    tol = bound(out, A, S, q16=False, kv32=kv is np.float32, out16=True)
    bad = np.zeros(out.shape, bool)
    if what[0] == "q":
        b.q[s, 3, 7] = np.nan if what == "q" else np.inf
        bad[s, 3] = True
    else:
        p = keys[s] // 3
        pool = b.k_pages if what == "k" else b.v_pages
        pool[b.table[s, p // b.page], p % b.page, kvh - 1, 5] = np.nan
        bad[s, G * (kvh - 1):, slice(None) if what == "k" else 5] = True
    d = b.dev()
    got = [decode(b, d)]
    longest = max(keys)
    dense = [torch.zeros(n, longest, kvh, hd, dtype=d["k_pages"].dtype, device="cuda") for _ in range(2)]
    for i, k in enumerate(keys):
        at = [b.table[i, p // b.page] * b.page + p % b.page for p in range(k)]
        for x, pool in zip(dense, (d["k_pages"], d["v_pages"])):
            x[i, :k] = pool.view(-1, kvh, hd)[at]
    pos = torch.tensor([max(0, k - 1) for k in keys], device="cuda")
    got.append(sa.decode(d["q"], *dense, i32(keys), b.cfg(), q_gain=d["gain"], rope_cos=d["cos"][pos].contiguous(),
                         rope_sin=d["sin"][pos].contiguous(), workspace=ws()))
    for x, name in zip(got, ("paged", "contiguous")):
        x = x.float().cpu().numpy()
        assert np.isnan(x[bad]).all(), f"{name}: {np.isnan(x[bad]).sum()} of {bad.sum()} NaN, {(x[bad] == 0).sum()} zeros"
        assert (np.abs(x - out)[~bad] <= tol[~bad]).all(), name


@pytest.mark.parametrize("hd", [256, 512])
@pytest.mark.parametrize("keys,new", [([300, 90], [40, 20]), ([2000, 90], [10, 20])])  # whole blocks; pieces
def test_prefill_shows_what_is_not_finite(hd, keys, new):
    """A query head of one token, and a K row that every later token attends."""
    b = Batch(keys, new, hd=hd, kvh=1)
    out, A, S = (x.copy() for x in b.oracle())
    tol = bound(out, A, S, q16=True, kv32=False, out16=True)
    bad = np.zeros(out.shape, bool)
    b.q[2, 3, 7] = np.nan
    bad[2, 3] = True
    p = keys[1] - new[1] + 5  # row 5 of the second sequence's tokens
    b.k_pages[b.table[1, p // b.page], p % b.page, 0, 9] = np.nan
    bad[new[0] + 5:] = True
    got = prefill(b, b.dev()).float().cpu().numpy()
    assert np.isnan(got[bad]).all(), f"{np.isnan(got[bad]).sum()} of {bad.sum()} NaN"
    assert (np.abs(got - out)[~bad] <= tol[~bad]).all()


@pytest.mark.parametrize("hd,kvh,kv", [(256, 2, np.float16), (512, 1, np.float16), (256, 1, np.float32), (512, 1, np.float32)])
@pytest.mark.parametrize("keys", [[40, 90], [1000, 90]])  # one split; a work list
def test_decode_row_for_a_missing_page_may_hold_anything(hd, kvh, kv, keys):
    """A step's row whose page is not there is neither stored nor attended, whatever it holds."""
    b = Batch(keys, [1, 1], hd=hd, kvh=kvh, kv=kv, missing=[(0, (keys[0] - 1) // 16)])
    out, A, S = b.oracle()
    for junk in (np.nan, np.inf, -np.inf):
        d = b.dev()
        k, v = d["k_new"].clone(), d["v_new"].clone()
        k[0] = v[0] = float(junk)
        got = decode(b, dict(d, k_new=k, v_new=v), append=True, v_norm=False)[:1]
        check(got.cpu().numpy(), out[:1], bound(out, A, S, q16=False, kv32=kv is np.float32, out16=True)[:1], f"{junk}")
        assert not torch.isfinite(d["k_pages"]).all()  # the poison of the rows that nobody attends is still there


# ---------------------------------------------------------------- long bounds, large batches
@pytest.mark.parametrize("hd,kvh,kv,page,bound_keys,n", [(512, 8, np.float32, 16, 131072, 64), (512, 8, np.float16, 64, 1 << 18, 70),
                                                         (256, 1, np.float16, 32768, 1 << 30, 1), (256, 2, np.float16, 32768, 1 << 30, 3)])
def test_decode_long_bounds(hd, kvh, kv, page, bound_keys, n):
    """Short sequences under a bound whose rows pass 32-bit offsets."""
    keys = [1 + 13 * i % 90 for i in range(n)]
    b = Batch(keys, [1] * n, hd=hd, kvh=kvh, kv=kv, page=page, spare=1, extra_cols=0)
    table = np.full((n, bound_keys // page), -1, np.int32)
    table[:, :b.cols] = b.table
    out, A, S = b.oracle(rope=False)
    got = decode(b, b.dev(table=torch.from_numpy(table).cuda()), rope_cos=None, rope_sin=None, max_key_len=bound_keys)
    check(got.cpu().numpy(), out, bound(out, A, S, q16=False, kv32=kv is np.float32, out16=True))


@pytest.mark.parametrize("n,kvh,hd,kv,longest", [(33, 8, 256, np.float16, 3100), (65, 4, 256, np.float16, 3900), (300, 2, 256, np.float16, 10000),
                                                 (264, 1, 512, np.float16, 4500), (280, 1, 256, np.float32, 4700)])
@pytest.mark.parametrize("append", [False, True])
def test_decode_one_long_sequence_among_many(n, kvh, hd, kv, longest, append):
    """More pairs than workgroups that run at once, one long sequence and idle ones: the work list, whose
    partials show in the workspace. (scale 0.25: no weight is subnormal in f16.)"""
    keys = [1 + 29 * i % 70 for i in range(n)]
    keys[n // 2], keys[n - 1], keys[3] = longest, 0, 0
    b = Batch(keys, [1] * n, hd=hd, kvh=kvh, kv=kv, page=64)
    b.q = np.random.default_rng(1).standard_normal((n, 8, hd)).astype(np.float32)
    d = b.dev()
    w = ws().reserve(sa.paged_decode_ws_bytes(n, 1 << 16, b.cfg(), page_size=64, kv_f32=kv is np.float32))
    w.buf.zero_()
    new = {}
    if append:
        new = dict(k_new=torch.randn(n, kvh, hd, device="cuda"), v_new=torch.randn(n, kvh, hd, device="cuda"), v_norm=False)
    got = decode(b, d, rope_cos=None, rope_sin=None, cfg=b.cfg(scale=0.25), workspace=w, **new)
    assert w.buf.any()
    rows = [0, 3, n // 2, n // 2 + 1, n - 2, n - 1]
    want, A, S = b.oracle(q=b.q[rows], tokens=[(i, keys[i] - 1) for i in rows], rope=False, scale=0.25,
                          k_pages=d["k_pages"].cpu().numpy(), v_pages=d["v_pages"].cpu().numpy())
    check(got.cpu().numpy()[rows], want, bound(want, A, S, q16=False, kv32=kv is np.float32, out16=True))
    for i in rows:
        if append and keys[i]:
            p = keys[i] - 1
            at = int(b.table[i, p // 64]), p % 64
            assert torch.equal(d["k_pages"][at], new["k_new"][i].to(d["k_pages"].dtype))
            assert torch.equal(d["v_pages"][at], new["v_new"][i].to(d["v_pages"].dtype))


# ---------------------------------------------------------------- empty calls
@pytest.mark.parametrize("kv", [np.float16, np.float32])
def test_calls_without_tokens(kv):
    """A step that brings no prompt: nothing is written, the outputs are empty, wrong operands are refused."""
    b = Batch([40, 0], [0, 0], kv=kv)
    d = b.dev()
    none = dict(d, q=d["q"][:0], k_new=d["k_new"][:0], v_new=d["v_new"][:0])
    write(b, none)
    write(b, none, rows=(none["k_new"].half(), none["v_new"].half()))
    w = ws()
    got = prefill(b, none, workspace=w)
    assert got.shape == (0, 8, 256) and got.dtype is torch.float16 and w.buf is None
    out = torch.empty(0, 8, 256, device="cuda")
    assert prefill(b, none, workspace=w, out=out) is out
    for name in ("k_pages", "v_pages"):
        assert np.array_equal(bits(d[name]), getattr(b, name).reshape(-1).view(np.uint8).reshape(bits(d[name]).shape))
    with pytest.raises(ValueError):
        write(b, dict(none, cu=d["cu"][:2].contiguous()))
    with pytest.raises(ValueError):
        prefill(b, none, out=torch.empty(1, 8, 256, device="cuda"))
    with pytest.raises(ValueError):
        prefill(b, dict(none, q=none["q"].half()))
    empty = dict(none, table=d["table"][:0], key_len=d["key_len"][:0], cu=d["cu"][:1].contiguous())
    write(b, empty)
    for got in (decode(b, empty), decode(b, empty, append=True), prefill(b, empty)):
        assert got.shape == (0, 8, 256)


# ---------------------------------------------------------------- refusals of what would be read past its end
def test_gains_of_another_length_are_refused():
    b = Batch([40, 20], [1, 1])
    d = b.dev()
    for bad in (d["gain"][:255].contiguous(), d["gain"][:1], torch.ones(512, device="cuda"), torch.ones(2, 256, device="cuda")):
        for call in (lambda: decode(b, dict(d, gain=bad)), lambda: prefill(b, dict(d, gain=bad)),
                     lambda: write(b, dict(d, k_gain=bad)), lambda: decode(b, dict(d, k_gain=bad), append=True)):
            with pytest.raises(ValueError):
                call()
    out, A, S = b.oracle()
    got = decode(b, dict(d, gain=d["gain"].view(1, 256)))
    check(got.cpu().numpy(), out, bound(out, A, S, q16=False, kv32=False, out16=True))


def test_table_rows_too_far_apart_are_refused():
    """A row stride past 32 bits, which cut to them would read other entries."""
    b = Batch([40, 20], [1, 1], extra_cols=0)
    wide = torch.empty(2 ** 32 + 2 * b.cols, dtype=torch.int32, device="cuda")
    table = wide.as_strided((2, b.cols), (2 ** 32 + b.cols, 1))
    table.copy_(torch.from_numpy(b.table))
    d = b.dev(table=table)
    for call in (lambda: decode(b, d), lambda: prefill(b, d), lambda: write(b, d)):
        with pytest.raises(ValueError):
            call()


# ---------------------------------------------------------------- long contexts at scale 1
def long_tables(b, keys):
    c, s = sa.rope_tables(np.arange(keys), b.hd, 1e6, device="cpu")
    b.cos, b.sin = c.numpy(), s.numpy()


@pytest.mark.parametrize("hd,keys", [(256, 33000), (512, 20000)])
def test_prefill_long_history_at_scale_1(hd, keys):
    b = Batch([keys, 70], [37, 70], hd=hd, kvh=1, page=64)
    long_tables(b, keys)
    rows = [0, 17, 36, 37, 106]
    out, A, S = (x[rows] for x in b.oracle(tokens=[t if i in rows else None for i, t in enumerate(b.tokens())]))
    got = prefill(b, b.dev())
    check(got.cpu().numpy()[rows], out, bound(out, A, S, q16=True, kv32=False, out16=True))


@pytest.mark.parametrize("hd,kv,n", [(256, np.float16, 1), (256, np.float16, 128), (512, np.float16, 64), (256, np.float32, 128)])
def test_decode_long_context_at_scale_1(hd, kv, n):
    keys = 20000
    b = Batch([keys], [1], hd=hd, kvh=1, page=64, kv=kv)
    long_tables(b, keys)
    d = b.dev()
    q = np.random.default_rng(2).standard_normal((n, 8, hd)).astype(np.float32)
    lens = [keys - 17 * i for i in range(n)]
    got = decode(b, dict(d, q=torch.from_numpy(q).cuda(), table=d["table"].repeat(n, 1), key_len=i32(lens)))
    rows = sorted({0, n // 3, n - 1})
    want, A, S = b.oracle(q=q[rows], tokens=[(0, lens[i] - 1) for i in rows])
    check(got.cpu().numpy()[rows], want, bound(want, A, S, q16=False, kv32=kv is np.float32, out16=True))


@pytest.mark.parametrize("hd", [256, 512])
@pytest.mark.parametrize("kv", [np.float16, np.float32])
@pytest.mark.parametrize("call", ["decode", "prefill"])
def test_many_weak_keys_beside_a_strong_one(hd, kv, call):
    """Weights of 2^-26 of the largest, below f16's smallest number, whose values are all that the output
    holds: a strong key at the front of every 2048, one in each wave's blocks, with a value of zero."""
    keys, n, new = 16000, 64, 20
    b = Batch([keys], [1 if call == "decode" else new], hd=hd, kvh=1, page=64, kv=kv)
    p = np.arange(keys)
    strong = (p % 2048 < 64) & (p % 16 == 0)
    k, v = np.zeros((keys, 1, hd)), np.full((keys, 1, hd), 1024.0)
    k[strong, 0, 0], v[strong] = 1.0, 0.0
    at = b.table[0, p // 64] * 64 + p % 64
    b.k_pages.reshape(-1, 1, hd)[at], b.v_pages.reshape(-1, 1, hd)[at] = k, v
    b.q = np.zeros((n if call == "decode" else new, 8, hd), np.float32)
    b.q[..., 0] = 18.0
    d = b.dev()
    off = dict(q_gain=None, rope_cos=None, rope_sin=None)
    if call == "decode":
        lens = [keys - i for i in range(n)]
        got = decode(b, dict(d, table=d["table"].repeat(n, 1), key_len=i32(lens)), out_dtype=torch.float32, **off)
        tokens = [(0, x - 1) for x in lens]
    else:
        got, tokens = prefill(b, d, out_dtype=torch.float32, **off), b.tokens()
    rows = [0, 7, len(tokens) - 1]
    want, A, S = b.oracle(q=b.q[rows], tokens=[tokens[i] for i in rows], gain=False, rope=False)
    assert want.min() > 0.005
    tol = bound(want, A, S, q16=call == "prefill", kv32=kv is np.float32, out16=False, k16=call == "prefill" and kv is np.float32)
    if call == "prefill":
        # P of a key is off by at most 2^-25, where the largest is 2^4 or more: 2^-29 sum |v| / sum_t exp(s_t - max s)
        most = np.array([strong[:tokens[i][1] + 1].sum() for i in rows])
        tol = tol + (2.0 ** -29 * 1024 * keys / most)[:, None, None]
        assert (tol < want / 4).all()
    check(got.cpu().numpy()[rows], want, tol)


# ---------------------------------------------------------------- one split or many
@pytest.mark.parametrize("hd,kv,n,kvh,keys,one", [
    (256, np.float16, 1, 2, 128, True), (256, np.float16, 1, 2, 129, False), (256, np.float16, 64, 1, 320, True), (256, np.float16, 64, 1, 321, False),
    (512, np.float16, 1, 2, 64, True), (512, np.float16, 1, 2, 65, False), (512, np.float16, 32, 2, 161, False), (512, np.float16, 64, 2, 320, True),
    (256, np.float32, 1, 2, 64, True), (256, np.float32, 1, 2, 65, False), (256, np.float32, 64, 1, 160, True), (256, np.float32, 64, 1, 200, False),
    (512, np.float32, 1, 2, 32, True), (512, np.float32, 1, 2, 33, False), (512, np.float32, 32, 2, 81, False), (512, np.float32, 64, 2, 320, True)])
def test_decode_few_keys(hd, kv, n, kvh, keys, one):
    """Either side of the bounds below which a pair's keys are one split (no partials in the workspace), by
    the bytes of a row."""
    b = Batch([keys - i % 3 for i in range(n)], [1] * n, hd=hd, kvh=kvh, kv=kv)
    w = ws().reserve(sa.paged_decode_ws_bytes(n, keys, b.cfg(), page_size=16, kv_f32=kv is np.float32))
    w.buf.zero_()
    got = decode(b, b.dev(), workspace=w, max_key_len=keys)
    assert bool(w.buf.any()) != one
    out, A, S = b.oracle()
    check(got.cpu().numpy(), out, bound(out, A, S, q16=False, kv32=kv is np.float32, out16=True))


# ---------------------------------------------------------------- calls that the documents allow
@pytest.mark.parametrize("hd,kvh", [(256, 2), (512, 1)])
@pytest.mark.parametrize("window", [0, 60])
def test_f32_prefill_missing_and_shared_pages(hd, kvh, window):
    """f32 caches: pages that are not there, a prefix shared by two sequences, idle sequences, a loose bound."""
    b = Batch([100, 48, 150, 0, 90], [60, 48, 20, 0, 33], hd=hd, kvh=kvh, kv=np.float32, window=window, pad=3,
              missing=[(0, 0), (0, 4), (1, 0), (1, 1), (1, 2), (2, 6), (2, 9)])
    b.table[4, :2] = b.table[2, :2]
    k, v = b.k_pages.copy(), b.v_pages.copy()  # the shared pages hold rows for both sequences' windows
    r = np.random.default_rng(5)
    for pool in (k, v):
        pool[b.table[2, :2]] = r.standard_normal((2, 16, kvh, hd)) * (0.4 if pool is k else 1)
    out, A, S = b.oracle(k_pages=k, v_pages=v)
    live = np.array([t is not None for t in b.tokens()])
    table = np.pad(b.table, ((0, 0), (0, 20)), constant_values=-1)
    for max_key_len in (150, 300):
        got = prefill(b, b.dev(table=torch.from_numpy(table).cuda(), k_pages=torch.from_numpy(k).cuda(), v_pages=torch.from_numpy(v).cuda()),
                      max_key_len=max_key_len).cpu().numpy()
        check(got[live], out[live], bound(out, A, S, q16=True, kv32=True, out16=True, k16=True)[live])


@pytest.mark.parametrize("hd", [256, 512])
@pytest.mark.parametrize("keys,new", [([70, 200], [70, 33]), ([1900, 40], [9, 40])])  # whole blocks; pieces
@pytest.mark.parametrize("dt", [torch.float16, torch.float32])
def test_prefill_quantised_outputs(hd, keys, new, dt):
    b = Batch(keys, new, hd=hd, kvh=2)
    out, A, S = b.oracle()
    step = 0.015625
    got = prefill(b, b.dev(), cfg=b.cfg(out_q=step), out_dtype=dt).float().cpu().numpy()
    k = got / step
    assert (k == np.round(k)).all() and k.min() >= -128 and k.max() <= 127  # a step of 2^-6: exact in both types
    exact = np.clip(out, -128 * step, 127 * step)
    check(got, exact, bound(out, A, S, q16=True, kv32=False, out16=False) + step / 2)


@pytest.mark.parametrize("hd,kvh,kv", [(256, 2, np.float16), (512, 1, np.float32)])
def test_captured_appends(hd, kvh, kv):
    """Steps that append, captured once and replayed: each replay adds the next row, as the eager calls do."""
    keys, steps = [150, 1, 900], 4
    b = Batch([k + steps + 1 for k in keys], [1] * 3, hd=hd, kvh=kvh, kv=kv)
    rows = [torch.randn(steps + 1, 3, h, hd, device="cuda") for h in (8, kvh, kvh)]
    eager, graphed = b.dev(), b.dev()
    for d in (eager, graphed):
        d["key_len"] = i32(keys)
        d["q"], d["k_new"], d["v_new"] = (x[0].clone() for x in rows)
    w = ws().reserve(sa.paged_decode_ws_bytes(3, MAX_KEYS, b.cfg(), page_size=16, kv_f32=kv is np.float32))
    out = torch.zeros(3, 8, hd, dtype=torch.float16, device="cuda")
    decode(b, graphed, append=True, workspace=w, out=out)
    g, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=stream):
        decode(b, graphed, append=True, workspace=w, out=out)
    decode(b, eager, append=True)
    for i in range(1, steps + 1):
        for d in (eager, graphed):
            d["key_len"].add_(1)
            for name, x in zip(("q", "k_new", "v_new"), rows):
                d[name].copy_(x[i])
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            g.replay()
        torch.cuda.synchronize()
        want = decode(b, eager, append=True)
        torch.cuda.synchronize()
        assert torch.equal(out, want), f"step {i}"
        for name in ("k_pages", "v_pages"):
            assert np.array_equal(bits(eager[name]), bits(graphed[name])), f"step {i}: {name}"


def test_calls_from_two_threads():
    """Two threads, a stream and a workspace each, one config: the outputs are the calls' own."""
    import threading
    bs = [Batch([300 + 400 * s, 90], [3, 1], seed=s) for s in (0, 1)]
    cfg, outs, errors = bs[0].cfg(), [[], []], []
    ds = [b.dev() for b in bs]
    torch.cuda.synchronize()

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                w, dd = ws(), dict(ds[i], q=ds[i]["q"][2:4].contiguous())
                for _ in range(20):
                    outs[i].append((prefill(bs[i], ds[i], workspace=w, cfg=cfg), decode(bs[i], dd, workspace=w, cfg=cfg)))
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for b, o in zip(bs, outs):
        out, A, S = b.oracle()
        tol = bound(out, A, S, q16=True, kv32=False, out16=True)
        for x, y in o:
            check(x.cpu().numpy(), out, tol)
            check(y.cpu().numpy(), out[2:4], tol[2:4])


@pytest.mark.parametrize("kv", [np.float16, np.float32])
def test_table_of_more_columns_than_a_buffer_range_holds(kv):
    """2^30 columns, of whose bytes 32 bits keep none: the entries are still the sequence's."""
    b = Batch([200], [33], kv=kv)
    assert b.table[0, 0] != 0
    table = torch.full((1, 2 ** 30), -1, dtype=torch.int32, device="cuda")
    table[:, :b.cols] = torch.from_numpy(b.table)
    d = b.dev(table=table)
    out, A, S = b.oracle()
    got = prefill(b, d, max_key_len=1000)
    check(got.cpu().numpy(), out, bound(out, A, S, q16=True, kv32=kv is np.float32, out16=True, k16=kv is np.float32))
    got = decode(b, dict(d, q=d["q"][32:33].contiguous()), max_key_len=1000)
    check(got.cpu().numpy(), out[32:], bound(out, A, S, q16=False, kv32=kv is np.float32, out16=True)[32:])
    ref = b.dev()
    write(b, d, max_key_len=1000)
    write(b, ref)
    assert np.array_equal(bits(d["k_pages"]), bits(ref["k_pages"])) and np.array_equal(bits(d["v_pages"]), bits(ref["v_pages"]))
