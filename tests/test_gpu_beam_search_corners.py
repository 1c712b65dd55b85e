"""Corners of the beam selection against the 64-bit oracle (tolerances as in
test_gpu_beam_search.py)."""
import math

import pytest
import torch
from torch.nn.functional import pad

from test_gpu_beam_search import BF16, F16, F32, INF, check_select, make

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


def definition(logits, scores, count, finished, eos):
    """The oracle's selection by torch's sorts, for sizes that its Python sort takes too long over
    (64 bits; no NaN)."""
    N, W, V = logits.shape
    x, s = logits.double(), scores.double().unsqueeze(-1)
    top = x.amax(-1, keepdim=True)
    below = x - top.nan_to_num(neginf=0.0)
    # (rows of equal alignment, so that equal ones have equal sums)
    value = s + (below - torch.logsumexp(pad(below, (0, -V % 64), value=-INF), -1, keepdim=True))
    value = torch.where(torch.isneginf(top) | torch.isneginf(s), -INF, value)
    if finished is not None:
        alone = torch.where(torch.arange(V, device=x.device) == eos, s, -INF)
        value = torch.where(finished.unsqueeze(-1), alone, value)
    value = value.view(N, W * V)
    # (the candidates by value, ties by index: all above the last one, then the lowest equal ones)
    least = value.topk(count).values[:, -1:]
    out = []
    for n in range(N):
        above = (value[n] > least[n]).nonzero()[:, 0]
        equal = (value[n] == least[n]).nonzero()[:count - len(above), 0]
        at = torch.cat([above, equal]).sort().values
        out.append(at[value[n, at].sort(descending=True, stable=True).indices])
    at = torch.stack(out)
    parents, tokens = at // V, at % V
    done = None if finished is None else torch.gather(finished, 1, parents) | (tokens == eos)
    return torch.gather(value, 1, at), tokens, parents, done


def check_large(logits, scores, count, finished=None, eos=None):
    from llm_cuda.kernels.beam_search import beam_select

    kw = {} if finished is None else dict(finished=finished, eos_token_id=eos)
    got = beam_select(logits, scores, num_candidates=count, **kw)
    want = definition(logits, scores, count, finished, eos)
    assert torch.equal(got[2], want[2]), "parents"
    assert torch.equal(got[1], want[1]), "tokens"
    fine = torch.isfinite(want[0])
    assert torch.equal(torch.isneginf(got[0]), torch.isneginf(want[0])) and torch.equal(fine, torch.isfinite(got[0]))
    assert ((got[0].double() - want[0]).abs()[fine] <= 1e-6 + 2 ** -24 * want[0][fine].abs()).all()
    if finished is not None:
        assert torch.equal(got[3], want[3])


def test_the_large_definition_is_the_oracles():
    from oracle.beam import beam_select as ref_select

    g = torch.Generator().manual_seed(0)
    x = torch.randint(-2, 3, (3, 4, 50), generator=g).float()
    x[0, 1] = x[2, :, 20:] = -INF
    s = torch.tensor([[-1.0, -1.0, -INF, -2.0]] * 3)
    done = torch.tensor([[False, True, False, False]] * 3)
    for count in (1, 7, 40):
        for a, b in zip(definition(x, s, count, done, 9), ref_select(x, s, count, done, 9)):
            assert torch.equal(a, b) or torch.allclose(a, b, rtol=1e-12, atol=0)


# Rows of several chunks of 8192 logits, enough of them that every CU has one: groups, beams,
# vocabulary (a whole chunk, one more token, odd tails)
LARGE = [(8, 8, 32769), (16, 8, 16385), (2, 64, 16384), (1, 128, 20011), (32, 2, 40000)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("N,W,V", LARGE)
def test_many_rows_of_several_chunks(cuda, N, W, V, dtype):
    g = torch.Generator(device=cuda).manual_seed(V)
    x = (torch.randn(N, W, V, generator=g, device=cuda) * 2.5).to(dtype)
    s = -10 * torch.rand(N, W, generator=g, device=cuda)
    for count in (1, min(W, 64), 64):
        check_large(x, s, count)
    # masked ones: half, nearly all, whole rows, one left, fewer left than candidates, dead beams
    y = x.masked_fill(torch.rand(x.shape, generator=g, device=cuda) < 0.5, -INF)
    y[0, 0], y[0, W - 1, :V - 1], y[N - 1, W // 2, 40:] = -INF, -INF, -INF
    t = s.clone()
    t[N - 1, 0] = -INF
    check_large(y, t, 64)
    y = x.masked_fill(torch.rand(x.shape, generator=g, device=cuda) < 0.9995, -INF)
    check_large(y, t, 64)
    check_large(torch.full_like(x, -INF), s, 64)
    # finished beams
    done = torch.rand(N, W, generator=g, device=cuda) < 0.3
    for eos in (0, V // 2, V - 1):
        check_large(x, s, 64, done, eos)
    check_large(x, s, 5, torch.ones_like(done), 3)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("N,W,V", LARGE)
def test_ties_of_several_chunks(cuda, N, W, V, dtype):
    g = torch.Generator(device=cuda).manual_seed(V)
    zero = torch.zeros(N, W, device=cuda)
    x = torch.zeros(N, W, V, dtype=dtype, device=cuda)
    for count in (3, 64):
        check_large(x, zero, count)
    x = torch.randint(-2, 3, (1, 1, V), generator=g, device=cuda).to(dtype).repeat(N, W, 1)
    check_large(x, zero, 64)
    # the best ones in few lanes of a chunk, its start or every lane in turn
    at = torch.arange(V, device=cuda)
    for stride, block in ((8192, 64), (2048, 8), (1024, 4), (8, 1)):
        hot = (at % stride) < block
        row = torch.where(hot, 3.0 + at.float() / V, -at.float() / V).to(dtype)
        for y in (row, row.flip(-1)):
            check_large(y.repeat(N, W, 1), zero, 64)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_undefined_rows_of_several_chunks(cuda, dtype):
    """NaN or +inf anywhere in a beam makes its values NaN, which rank first, lowest tokens first."""
    from llm_cuda.kernels.beam_search import beam_select

    N, W, V = 8, 8, 32769
    x = torch.randn(N, W, V, generator=torch.Generator().manual_seed(1)).to(dtype).to(cuda)
    s = torch.zeros(N, W, device=cuda)
    bad = [(0, 3, 0), (1, 7, V - 1), (2, 0, 8191), (3, 1, 8192), (4, 2, 20000), (5, 6, V - 2)]
    for n, w, at in bad:
        x[n, w, at] = math.nan if n % 2 else INF
    s[6, 4] = math.nan
    x[7] = math.nan
    got, tokens, parents = beam_select(x, s, num_candidates=64)
    want = [w for _, w, _ in bad] + [4, 0]
    assert got.isnan().all()
    assert torch.equal(tokens.cpu(), torch.arange(64).expand(N, 64))
    assert torch.equal(parents.cpu(), torch.tensor(want).view(N, 1).expand(N, 64))


def test_more_lists_than_are_held(cuda):
    """2048 and 1440 lists in a group: their best candidates are read again, and, where too
    many reach the bound, all of them are looked through."""
    g = torch.Generator(device=cuda).manual_seed(5)
    for W, V in ((128, 128256), (160, 65537)):
        x = torch.randn(1, W, V, generator=g, device=cuda) * 2.5
        s = -torch.rand(1, W, generator=g, device=cuda)
        check_large(x.to(BF16), s, 64)
        check_large(x, s, 7)
        check_large(torch.zeros_like(x), torch.zeros_like(s), 64)  # 2^24 equal values
        check_large(torch.full_like(x, -INF), s, 64)
        check_large(x.masked_fill(torch.rand(x.shape, generator=g, device=cuda) < 0.99995, -INF), s, 64)


@pytest.mark.parametrize("W,V,count", [(64, 20000, 64), (200, 3000, 64), (100, 30000, 64), (256, 9000, 40)])
def test_equal_values_in_many_lists(cuda, W, V, count):
    """More equal values than the merge gathers: equal beams whose best logits are all the same."""
    zero = torch.zeros(1, W, device=cuda)
    row = torch.zeros(V, device=cuda)
    row[::3] = 1.0
    check_large(row.to(BF16).repeat(1, W, 1), zero, count)
    check_large(row.repeat(1, W, 1), zero, count)
    best = torch.randint(0, 2, (1, W, V), generator=torch.Generator(device=cuda).manual_seed(1), device=cuda)
    best[..., 0] = 1
    check_large(best.sort(-1).values.float(), zero, count)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_one_beam_of_many_chunks(cuda, dtype):
    """More than 64 chunks in a row: a lane joins several of their sums."""
    g = torch.Generator(device=cuda).manual_seed(2)
    for V in (131073, 540001, 3000000):
        x = (torch.randn(1, 1, V, generator=g, device=cuda) * 3).to(dtype)
        for count in (1, 64):
            check_large(x, torch.full((1, 1), -2.0, device=cuda), count)


@pytest.mark.parametrize("dead", [-1e9, -1e30, torch.finfo(F32).min])
@pytest.mark.parametrize("W,V", [(4, 3000), (40, 20000)])
def test_beams_switched_off_by_a_large_score(cuda, W, V, dead):
    """Beams at a large negative score, as masks write it, beside a live one with few tokens left:
    the live tokens first, then as many others as are wanted, each once, at their beam's score."""
    from llm_cuda.kernels.beam_search import beam_select

    x, _ = make(1, W, V, F32, V)
    x[0, 0, 5:] = -INF
    s = torch.full((1, W), dead)
    s[0, 0] = -1.0
    best, tokens, parents = (t.cpu() for t in beam_select(x.to(cuda), s.to(cuda), num_candidates=32))
    live = torch.log_softmax(x[0, 0, :5].double(), 0) - 1.0
    want, order = live.sort(descending=True)
    assert torch.equal(tokens[0, :5], order) and not parents[0, :5].any()
    assert (best[0, :5].double() - want).abs().max() <= 2e-6
    assert (parents[0, 5:] > 0).all() and len(set(zip(parents[0].tolist(), tokens[0].tolist()))) == 32
    value = dead + torch.log_softmax(x[0].double(), -1)[parents[0, 5:], tokens[0, 5:]]
    assert ((best[0, 5:].double() - value).abs() <= 1e-6 + 2 ** -24 * value.abs()).all()
    top = (dead + torch.log_softmax(x[0, 1:].double(), -1)).flatten().topk(27).values
    assert ((best[0, 5:].double() - top).abs() <= 1e-6 + 2 ** -24 * top.abs()).all()
