"""What earlier tests of the calls that branch leave open: the walk over offsets that do not ascend, to the last word; q's
accuracy at head_dim 256 over all layouts; the same call twice."""
import numpy as np
import pytest
import torch

import oracle.branching as OB
import slang_amd as sa
from paged_cases import bound, check
from test_gpu_branching import dev, drafted
from test_gpu_tree import Trees, bits, tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cu", [[0, 40, 0, 40], [-5, 100, 3, 2 ** 31 - 1], [40, 40, 0, 0], [30, 10, 20, 45], [0, 0, -2 ** 31, 40]])
def test_accept_over_any_offsets(cu):
    """Offsets outside the packed rows are cut to them, one below its predecessor to that; no word beside the outputs changes."""
    n, keys, most = 40, [50, 60, 3], 7
    par, drafts, targets = drafted([n], 1)
    guarded = [torch.full((5,) + tail, 777, dtype=torch.int32, device="cuda") for tail in ((most,), (), (), ())]
    out = [t[1:4] for t in guarded]
    sa.tree_accept(dev(drafts), dev(targets), dev(par), dev(cu), dev(keys), max_path=most, out=out)
    for b in range(3):
        lo = min(max(cu[b], 0), n)
        hi = min(max(cu[b + 1], lo), n)
        want = OB.accept([keys[b]], [0, hi - lo], par[lo:hi], drafts[lo:hi], targets[lo:hi], most)
        assert [x[b].tolist() for x in out] == [w[0] for w in want], b
    for t in guarded:
        assert (t[0] == 777).all() and (t[4] == 777).all()


LAYOUTS = [dict(keys=[70, 129, 17], new=[70, 40, 17]),                                     # whole prompts and short trees
           dict(keys=[1500, 20, 900, 1201], new=[40, 20, 130, 1], page=32),                # histories cut into pieces
           dict(keys=[100, 48, 150, 40], new=[60, 48, 20, 10], missing=[(0, 0), (0, 3), (1, 0), (1, 1), (1, 2), (2, 4), (3, 2)]),
           dict(keys=[1, 0, 64, 703], new=[1, 0, 64, 3], pad=5)]


@pytest.mark.parametrize("layout", range(len(LAYOUTS)))
@pytest.mark.parametrize("kvh", [1, 2, 4, 8])
@pytest.mark.parametrize("window", [0, 100, 5])
@pytest.mark.parametrize("kv", [np.float16, np.float32])
def test_queries_of_256_keep_their_bits_everywhere(layout, kvh, window, kv):
    b = Trees(kvh=kvh, window=window, kv=kv, seed=kvh + window, **LAYOUTS[layout])
    out, A, S = b.oracle()
    live, kv32 = b.live(), kv is np.float32
    for dt in (torch.float16, torch.float32):
        got = tree(b, b.dev(), out_dtype=dt).cpu().numpy()
        check(got[live], out[live], bound(out, A, S, q16=False, kv32=kv32, out16=dt is torch.float16, k16=kv32)[live])


@pytest.mark.parametrize("hd,kvh", [(256, 2), (512, 1)])
@pytest.mark.parametrize("kv", [np.float16, np.float32])
def test_the_same_call_twice_is_the_same(hd, kvh, kv):
    """Nothing depends on which workgroup comes first: outputs and stored rows repeat to the bit."""
    b = Trees([1500, 20, 900, 601], [40, 20, 130, 1], hd=hd, kvh=kvh, kv=kv, page=32, written=False)
    first, ws = None, sa.Workspace()
    for _ in range(4):
        d = b.dev()
        got = [bits(tree(b, d, append=True, workspace=ws)), bits(d["k_pages"]), bits(d["v_pages"])]
        first = first or got
        assert all(np.array_equal(x, y) for x, y in zip(got, first))
