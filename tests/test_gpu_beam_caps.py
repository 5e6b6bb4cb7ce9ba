"""beam_select's scores under caps of any size, against 64 bits."""
import numpy as np
import pytest
import torch

import oracle.branching as OB
import slang_amd as sa

pytestmark = pytest.mark.gpu

CAPS = [float(np.float32(c)) for c in (1e-40, 1e-30, 0.01, 30.0, 64.0, 64.5, 200.0, 1e3, 1e5, 1e6, 1e9, 1e17, 1e30, 2.9e38)]


def off(cap, largest):
    """Largest |score - exact| but for the last rounding: 2^-18 of the sums as without a cap, and twice (a logit's and the
    largest's) what x' is off by. Up to a cap of 64, cap - 2 cap r with r = 1 / (1 + e) <= 1/2 where a logit counts: r's and
    e's steps and e's argument give at most 2.5 2^-23 cap. Beyond, 4.5 2^-23 |x'|: below |x / cap| = 0.3 a series whose
    sum is rounded once, else tanh off by 1.3 2^-23 and at least 0.29."""
    return 2.0 ** -18 + 2.0 ** -23 * (5 * cap if cap <= 64 else 9 * largest)


@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("dtype,spread", [(np.float32, 3.0), (np.float16, 3.0), (np.float32, 30.0)])
def test_caps_of_any_size(cap, dtype, spread):
    W, V, n_out = 3, 5000, 6
    r = np.random.default_rng(11)
    x = (spread * r.standard_normal((2 * W, V))).astype(dtype)
    x[:, ::50] = 0.0
    s = np.array([[-1, -3, -2], [-0.5, -0.7, -4]], np.float32)
    got = [t.cpu().numpy() for t in sa.beam_select(torch.from_numpy(x).cuda(), torch.from_numpy(s).cuda(), workspace=sa.Workspace(),
                                                   cap=cap, n_out=n_out)]
    want = OB.select(x, s, cap, n_out)
    most = np.abs(cap * np.tanh(x.astype(np.float64) / cap)).max()
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])
    assert (np.abs(got[0] - want[0]) <= off(cap, most) + 2.0 ** -23 * np.abs(want[0])).all()


@pytest.mark.parametrize("cap", CAPS)
def test_caps_over_what_is_not_finite(cap):
    """-inf and NaN are no tokens under any cap; the type's extremes and +inf stay numbers."""
    r = np.random.default_rng(12)
    x = (3 * r.standard_normal((3, 700))).astype(np.float32)
    x[0, ::3], x[0, 1::3] = -np.inf, np.nan
    x[1, 5], x[1, 6] = -3.4028235e38, -np.inf
    x[2, [4, 600]] = np.inf
    s = np.array([[-1, -3, -2]], np.float32)
    got = [t.cpu().numpy() for t in sa.beam_select(torch.from_numpy(x).cuda(), torch.from_numpy(s).cuda(), workspace=sa.Workspace(),
                                                   cap=cap, n_out=5)]
    want = OB.select(x, s, cap, 5)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])
    # the largest |x'| that counts: that of +inf is the cap itself, from which every other token is far
    most = np.abs(cap * np.tanh(x[np.abs(x) < 1e30].astype(np.float64) / cap)).max()
    assert (np.abs(got[0] - want[0]) <= off(cap, most) + 2.0 ** -23 * np.abs(want[0])).all()
