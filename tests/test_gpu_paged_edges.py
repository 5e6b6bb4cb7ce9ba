"""The paged operators at the edges of what they accept: offsets out of order over tables of just the
rows that the keys need, rows that are not finite, empty calls, long contexts."""
import numpy as np
import pytest
import torch

import slang_amd as sa
from paged_cases import Batch, bound, check
from test_gpu_paged import bits, decode, prefill, write, ws

pytestmark = pytest.mark.gpu


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
