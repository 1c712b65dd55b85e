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


@pytest.mark.parametrize("V", [2 ** 31 - 1, 2 ** 31 - 8191])
def test_vocabularies_up_to_the_limit(cuda, V):
    """One beam whose last chunk ends past 2^31: few tokens allowed, at the row's ends, so that
    one counted twice shows (their logits, and so the sum, are small whole numbers)."""
    from llm_cuda.kernels.beam_search import beam_select

    x = torch.full((1, 1, V), -INF, dtype=BF16, device=cuda)
    at = torch.tensor([0, 7, 2 ** 30, V - 9, V - 8, V - 7, V - 2, V - 1])
    value = torch.tensor([1.0, 2.0, -1.0, 3.0, 0.5, 2.5, 4.0, 3.5])
    x[0, 0, at.to(cuda)] = value.to(BF16).to(cuda)
    scores, tokens, parents = beam_select(x, torch.zeros(1, 1, device=cuda), num_candidates=8)
    want, order = torch.log_softmax(value.double(), 0).sort(descending=True)
    assert torch.equal(tokens[0].cpu(), at[order]) and not parents.any()
    assert (scores[0].double().cpu() - want).abs().max().item() <= 1e-6 + 2 ** -24 * 8
