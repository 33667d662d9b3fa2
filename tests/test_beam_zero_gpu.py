"""Beam selection: -0.0 and 0.0 are equal logits and equal totals, so they are ordered as other equal ones are."""
import numpy as np
import pytest

from test_beam_gpu import select

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("V", [40, 5000, 50257])
def test_zeros_of_either_sign_go_to_the_lower_token(cuda, lib, dtype, V):
    torch = cuda
    W = 4
    x = np.full((W, V), -3.0, dtype)
    at = sorted(np.random.default_rng(V).choice(V, 9, replace=False))
    x[:, at] = np.where(np.arange(9) % 2 == 0, -0.0, 0.0)  # the lowest token has the negative one
    score = np.array([-1.0, -50.0, -50.0, -50.0], np.float32)
    token, parent, _, _ = select(torch, lib, torch.from_numpy(x).cuda(), torch.from_numpy(score).cuda(), None, 1, W, -1)
    assert token.tolist() == [int(i) for i in at[:W]] and parent.tolist() == [0] * W


def test_a_finished_beam_of_score_minus_zero_ties_with_zero(cuda, lib):
    torch = cuda
    x = np.full((2, 9), -np.inf, np.float32)
    x[1, 4] = 5.0  # one token: its total is its score, 0
    score, done = np.array([-0.0, 0.0], np.float32), np.array([1, 0], np.int32)
    token, parent, s, _ = select(torch, lib, torch.from_numpy(x).cuda(), torch.from_numpy(score).cuda(), torch.from_numpy(done).cuda(), 1, 2, 7)
    assert parent.tolist() == [0, 1] and token.tolist() == [7, 4] and s.tolist() == [0.0, 0.0]
