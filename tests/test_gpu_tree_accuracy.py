"""paged_tree's scores are as exact as plain decoding's, at both head sizes and over both types of caches: neither q nor K is
rounded to f16."""
import numpy as np
import pytest
import torch

import oracle.branching as OB
import slang_amd as sa
from paged_cases import bound, check
from test_gpu_tree import Trees, tree

pytestmark = pytest.mark.gpu


def exact_scores(out, A, S, kv32, out16):
    """The bound with q as a pair of f16; over f32 caches K is one too: its own rounding and the product of the two remainders, 2^-22
    each, and remainders below f16's normal range, which for the keys here are less: 2^-20 of a score, the weights move by twice that."""
    return bound(out, A, S, q16=False, kv32=kv32, out16=out16) + (np.expm1(2 * 2.0 ** -20 * S) * A if kv32 else 0.0)


LAYOUTS = [dict(keys=[70, 129, 17], new=[70, 40, 17]),
           dict(keys=[1500, 20, 900, 1201], new=[40, 20, 130, 1], page=32),
           dict(keys=[100, 48, 150, 40], new=[60, 48, 20, 10], missing=[(0, 0), (0, 3), (1, 0), (1, 1), (1, 2), (2, 4), (3, 2)]),
           dict(keys=[1, 0, 64, 703], new=[1, 0, 64, 3], pad=5)]


@pytest.mark.parametrize("hd,kv", [(512, np.float16), (512, np.float32), (256, np.float32)])
@pytest.mark.parametrize("layout", range(len(LAYOUTS)))
@pytest.mark.parametrize("kvh", [1, 2, 4, 8])
@pytest.mark.parametrize("window", [0, 100, 5])
def test_scores_keep_their_bits(hd, kv, layout, kvh, window):
    b = Trees(hd=hd, kvh=kvh, window=window, kv=kv, seed=kvh + window, **LAYOUTS[layout])
    out, A, S = b.oracle()
    live, kv32 = b.live(), kv is np.float32
    for dt in (torch.float16, torch.float32):
        o = torch.full((max(1, b.T), b.nh, b.hd), 7.25, dtype=dt, device="cuda")
        got = tree(b, b.dev(), out=o).cpu().numpy()
        check(got[live], out[live], exact_scores(out, A, S, kv32, dt is torch.float16)[live])
        assert (got[~live] == 7.25).all()


@pytest.mark.parametrize("hd,kvh", [(512, 1), (512, 2), (256, 2)])
@pytest.mark.parametrize("window", [0, 40])
def test_appended_rows_over_f32_caches(hd, kvh, window):
    """Rows that the call stores are attended with their remainders too."""
    new, hist = [12, 1, 40, 7, 0], [100, 63, 17, 700, 0]
    b = Trees([a + h for a, h in zip(new, hist)], new, hd=hd, kvh=kvh, kv=np.float32, window=window, written=False, seed=window)
    d = b.dev()
    got = tree(b, d, append=True, out_dtype=torch.float32).cpu().numpy()
    b.k_pages, b.v_pages = d["k_pages"].cpu().numpy(), d["v_pages"].cpu().numpy()
    out, A, S = b.oracle()
    check(got, out, exact_scores(out, A, S, True, False))


@pytest.mark.parametrize("hd,kvh", [(256, 2), (512, 1)])
@pytest.mark.parametrize("kv", [np.float16, np.float32])
def test_a_token_alone_is_a_decode_step(hd, kvh, kv):
    """A tree of one token and the decode step that it stands for, within the sum of what each may be off."""
    keys = [1, 70, 640, 1500]
    b = Trees(keys, [1] * 4, hd=hd, kvh=kvh, kv=kv, kind="roots")
    out, A, S = b.oracle()
    d = b.dev()
    got = tree(b, d, out_dtype=torch.float32).cpu().numpy()
    ref = sa.paged_decode(d["q"], d["k_pages"], d["v_pages"], d["table"], d["key_len"], b.cfg(), workspace=sa.Workspace(), q_gain=d["gain"],
                          rope_cos=d["cos"], rope_sin=d["sin"], out_dtype=torch.float32).cpu().numpy()
    tol = exact_scores(out, A, S, kv is np.float32, False)
    check(got, out, tol)
    check(got, ref, 2 * tol)


@pytest.mark.parametrize("hd", [256, 512])
@pytest.mark.parametrize("junk", [1e6, np.inf, np.nan])
def test_keys_beyond_f16_in_an_f32_cache(hd, junk):
    """One that is attended shows as NaN, one that is masked reaches nobody; a V beyond f16 shows in all that attend it."""
    b = Trees([60], [20], hd=hd, kvh=1, kv=np.float32, seed=5)
    out, A, S = b.oracle()
    victim = 7
    hit = [i for i in range(20) if victim in OB.line(b.parents, i)]
    others = [i for i in range(20) if i not in hit]
    k = b.k_pages.copy()
    k[b.table[0, (40 + victim) // 16], (40 + victim) % 16] = junk
    got = tree(b, b.dev(k_pages=torch.from_numpy(k).cuda())).cpu().numpy()
    check(got[others], out[others], exact_scores(out, A, S, True, True)[others])
    assert np.isnan(got[hit]).all()
    v = b.v_pages.copy()
    v[b.table[0, 0], 3] = 1e6
    assert not np.isfinite(tree(b, b.dev(v_pages=torch.from_numpy(v).cuda())).cpu().numpy()).any()


@pytest.mark.parametrize("hd,kvh", [(256, 2), (512, 1)])
def test_weights_over_f32_caches_keep_their_bits(hd, kvh):
    """With V that f16 holds, an f32 output over an f32 cache has no rounding to f16 left: pairs' remainders (2^-22 of q, K and P,
    their products), f32 arithmetic on scores (2^-19), partials of 24 bits (2^-16). Four times below a half step of f16."""
    b = Trees([300, 70, 1500, 33], [20, 70, 9, 1], hd=hd, kvh=kvh, kv=np.float32, seed=4)
    b.v_pages = b.v_pages.astype(np.float16).astype(np.float32)
    out, A, S = b.oracle()
    got = tree(b, b.dev(), out_dtype=torch.float32).cpu().numpy()
    d = (2.0 ** -21 + 2.0 ** -20 + 2.0 ** -19) * S + 2.0 ** -20
    check(got, out, (np.expm1(2 * d) + 2.0 ** -16 + 2.0 ** -20) * A + 2.0 ** -24 * np.abs(out) + 2.0 ** -24)
