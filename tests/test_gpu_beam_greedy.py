"""beam_select of width 1, which gives the tokens that drafts are checked against, beside the greedy step's own argmax."""
import numpy as np
import pytest
import torch

import slang_amd as sa
from slang_amd.decoder import softcap_argmax

pytestmark = pytest.mark.gpu


def test_width_one_is_the_greedy_steps_argmax():
    """beam_select of width 1 takes the largest logit, the lowest token of equal ones, with a cap or without; the greedy step
    caps in f32 first and takes the lowest token of those that this makes equal. They differ there and nowhere else."""
    V = 32000
    x = (4 * np.random.default_rng(5).standard_normal((9, V))).astype(np.float32)
    x[1, [700, 31]] = x[1].max() + 1   # equal logits
    x[2, [5, 900]] = 300, 400          # far above a cap of 30, where f32 makes them one
    x[3, 20000] = 200
    x[4] = 0
    logits = torch.from_numpy(x).cuda()
    zeros = torch.zeros(9, 1, device="cuda")
    for cap in (0.0, 30.0):
        token = sa.beam_select(logits, zeros, cap=cap, workspace=sa.Workspace())[2].view(-1).tolist()
        assert token == x.argmax(1).tolist()
        for i in range(9):
            capped = logits[i].clone()
            greedy = int(softcap_argmax(capped, cap))
            equal = (capped == capped.max()).nonzero().view(-1).tolist()
            assert greedy == equal[0]
            assert token[i] == greedy if i != 2 or cap == 0 else (token[i], greedy) == (900, 5)
