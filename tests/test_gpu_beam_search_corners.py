"""Corners of the beam selection against the 64-bit oracle (tolerances as in
test_gpu_beam_search.py)."""
import math

import pytest
import torch

from test_gpu_beam_search import BF16, F32, INF, check_select, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N,W,V,K", [(1, 1, 100, 4), (1, 4, 100, 16), (2, 3, 5000, 9), (40, 8, 9000, 8)])
@pytest.mark.parametrize("eos", [0, 2, 50, 99])
def test_finished_beams_without_a_score(cuda, N, W, V, K, eos):
    """A finished beam of score -inf: all of its tokens are equal, eos no better than others.
    (The sizes: joined in one launch, and by the merge.)"""
    x, s = make(N, W, V, BF16, V + eos)
    s[:] = -INF
    check_select(x, s, count=K, finished=torch.ones(N, W, dtype=torch.bool), eos=eos, dev=cuda)
    s[:, W - 1] = -3.0
    done = torch.zeros(N, W, dtype=torch.bool)
    done[:, 0] = done[:, W - 1] = True
    check_select(x, s, count=K, finished=done, eos=eos, dev=cuda)
