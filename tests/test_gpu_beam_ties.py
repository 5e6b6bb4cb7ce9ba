"""beam_select: a row's scores do not depend on where the row lies, so equal beams tie and come in order."""
import numpy as np
import pytest
import torch

import oracle.branching as OB
import slang_amd as sa

pytestmark = pytest.mark.gpu


def row(V, dtype, seed):
    return (3 * np.random.default_rng(seed).standard_normal(V)).astype(dtype)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("cap", [0.0, 30.0, 100.0])
@pytest.mark.parametrize("V", [501, 4099, 32001, 262147])
def test_equal_beams_of_odd_rows_tie(V, cap, dtype):
    """Rows of an odd length begin at every alignment; equal ones have equal scores to the bit, and the first beam's come first."""
    W = 8
    x = torch.from_numpy(row(V, dtype, V)).cuda().repeat(W, 1)
    s = torch.zeros(1, W, device="cuda")
    score, parent, token = (t.cpu().numpy() for t in sa.beam_select(x, s, workspace=sa.Workspace(), cap=cap, n_out=20))
    want = OB.select(x.cpu().numpy(), s.cpu().numpy(), cap, 20)
    assert np.array_equal(parent, want[1]) and np.array_equal(token, want[2])
    assert (score[0, :8] == score[0, 0]).all() and (score[0, 8:16] == score[0, 8]).all()


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("V", [513, 20000])
def test_a_row_scores_alike_wherever_it_lies(V, dtype):
    x = row(V, dtype, V)
    want = None
    for stride in range(V, V + 9):
        t = torch.full((3, stride), float("nan"), dtype=torch.float16 if dtype is np.float16 else torch.float32, device="cuda")
        t[:, :V] = torch.from_numpy(x).cuda()
        got = sa.beam_select(t[:, :V], torch.zeros(3, 1, device="cuda"), workspace=sa.Workspace(), n_out=4, cap=30.0)
        want = got[0][0].clone() if want is None else want
        assert torch.equal(got[0], want.expand(3, 4)), f"rows {stride} apart"
