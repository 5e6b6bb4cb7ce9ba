"""paged_tree: the weights that sum to a row's denominator are the ones that multiply V."""
import numpy as np
import pytest
import torch

from test_gpu_tree import Trees, tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,kvh", [(256, 2), (512, 1)])
@pytest.mark.parametrize("kv", [np.float16, np.float32])
def test_a_leading_weight_keeps_its_share(hd, kvh, kv):
    """One key leads, behind the first tile, all others score 0; so many sequences that none is cut. The weights are powers of two
    but for the leader's, which is rounded by at most u = 2^-11 of itself. With the sum over rounded weights that moves an output
    by u w |v - out|, not by u w |v|. Scores in f32 (2^-19 and q's pair 2^-21 of at most 7.5) move weights by twice that."""
    n_seq, keys, row = 400, 70, 66
    b = Trees([keys] * n_seq, [1] * n_seq, hd=hd, kvh=kvh, kv=kv, kind="roots", page=16)
    r = np.random.default_rng(3)
    b.k_pages[:] = 0
    b.v_pages[:] = r.standard_normal(b.v_pages.shape).astype(np.float16)
    at = b.table[:, row // 16], row % 16
    b.k_pages[at[0], at[1], :, 0] = 1.0
    b.v_pages[at] = np.sign(b.v_pages[at])
    b.q[:] = 0
    b.q[..., 0] = r.uniform(6, 7.5, b.q.shape[:2])
    out, A, S = b.oracle(q_gain=None, cos=None, sin=None)
    got = tree(b, b.dev(), q_gain=None, rope_cos=None, rope_sin=None, out_dtype=torch.float32).cpu().numpy().astype(np.float64)
    lead = np.exp(b.q[..., :1].astype(np.float64))
    w = lead / (lead + keys - 1)
    v = np.repeat(b.v_pages[at].astype(np.float64), 8 // kvh, 1)
    tol = 2.0 ** -11 * w * np.abs(v - out) + np.expm1(2 * (2.0 ** -19 + 2.0 ** -21) * S) * A + 2.0 ** -22 * A + 2.0 ** -24 * np.abs(out)
    d = np.abs(got - out)
    assert (d <= tol).all(), f"off by {(d / tol).max():.2f} x the bound"
