"""paged_fork on either side of the rules that choose between one workgroup and three launches: pages, rows, table entries."""
import numpy as np
import pytest
import torch

import oracle.branching as OB
import slang_amd as sa
from test_gpu_branching import beams, dev

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("groups,W,extra", [(50, 4, 0), (50, 4, 6), (256, 4, 0), (257, 4, 0), (5, 4, 0)])
@pytest.mark.parametrize("pages", [0, 12288, 12289])
def test_fork_is_the_same_in_either_form(groups, W, extra, pages):
    """200 rows of 80 and of 86 columns (32000 and 34400 entries of both tables), 1024 and 1028 rows, few."""
    page, n = 16, groups * W
    r = np.random.default_rng(groups + extra)
    prompts, grown = list(r.integers(1, 120, groups)), list(r.integers(0, 40, groups))
    table, keys, free, n_pages = beams(groups, W, prompts, grown, page, 3)
    cols = 80 + extra if groups == 50 else table.shape[1]
    table = np.pad(np.asarray(table), ((0, 0), (0, cols - table.shape[1])), constant_values=-1)
    if pages:
        if n_pages > pages:
            pytest.skip("the batch has more pages")
        free, n_pages = list(free) + list(range(n_pages, pages)), pages
    parent = np.arange(n) // W * W + r.integers(0, W, n)
    parent[3] = -1
    want = OB.fork([], table, keys, parent, free, 1, page, n_pages)
    free_t = np.full(n_pages, -1)
    free_t[:len(free)] = free
    got = sa.paged_fork([], dev(table), dev(keys), dev(parent), dev(free_t), dev([len(free)]), workspace=sa.Workspace(), n_pages=n_pages,
                        page_size=page)
    assert np.array_equal(got[0].cpu().numpy(), want[0]) and got[1].tolist() == want[1]
    assert got[3].tolist() == [len(want[2])]
    assert got[2].tolist() == [int(x) for x in want[2]] + [-1] * (n_pages - len(want[2]))
