"""Beam selection and cache reordering against the 64-bit oracle.

Tokens and parents have to be equal. Scores are rounded once to fp32 (2^-24
relative); the softmax sum's fp32 terms are off by at most 2^-22 each (two
roundings of the exponent's argument, |x - max| * 1.45 * 2^-24 * ln 2, and the
exponential's own) for arguments down to -4, which dominate the sum, and terms at
-80 by 2^-18 of a part below e^-76: below 1e-6 in the logsumexp together.
"""
import math

import pytest
import torch

from oracle.beam import beam_select as ref_select
from oracle.beam import kv_reorder as ref_reorder

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
INF = math.inf


def select(logits, scores, **kw):
    from llm_cuda.kernels.beam_search import beam_select

    got = beam_select(logits, scores, **kw)
    torch.cuda.synchronize()
    return got


def check_select(logits, scores, count=None, finished=None, eos=None, dev=None):
    count = logits.shape[1] if count is None else count
    kw = {} if finished is None else dict(finished=finished.to(dev), eos_token_id=eos)
    got = select(logits.to(dev), scores.to(dev), num_candidates=count, **kw)
    want = ref_select(logits, scores, count, finished, eos)
    assert got[0].dtype == F32 and got[1].dtype == torch.int64 and got[2].dtype == torch.int64
    assert torch.equal(got[2].cpu(), want[2]), "parents"
    assert torch.equal(got[1].cpu(), want[1]), "tokens"
    s, r = got[0].double().cpu(), want[0]
    assert torch.equal(s.isnan(), r.isnan())
    assert torch.equal(torch.isinf(s), torch.isinf(r))
    fine = torch.isfinite(r)
    assert ((s - r).abs()[fine] <= 1e-6 + 2 ** -24 * r[fine].abs()).all()
    if finished is not None:
        assert torch.equal(got[3].cpu(), want[3])


def make(N, W, V, dtype, seed, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(N, W, V, generator=g) * spread).to(dtype)
    return x, -10 * torch.rand(N, W, generator=g)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("N,W,V", [(1, 1, 1), (1, 4, 3), (2, 3, 64), (3, 2, 65), (1, 5, 255), (2, 4, 1000),
                                   (1, 8, 2049), (1, 2, 8191), (2, 2, 8193), (1, 3, 32000)])
def test_sizes_and_types(cuda, N, W, V, dtype):
    x, s = make(N, W, V, dtype, N * 1000 + V)
    check_select(x, s, dev=cuda, count=min(W, W * V))


@pytest.mark.parametrize("count", [1, 2, 5, 16, 31, 32, 33, 63, 64])
@pytest.mark.parametrize("W", [1, 4, 16])
def test_candidate_counts(cuda, count, W):
    x, s = make(2, W, 3001, BF16, count)
    check_select(x, s, count=count, dev=cuda)


def test_widest(cuda):
    x, s = make(1, 256, 700, BF16, 3)
    check_select(x, s, count=64, dev=cuda)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [50, 3000, 20000])
def test_ties_go_to_the_lowest_index(cuda, V, dtype):
    for count in (3, 64):
        x = torch.zeros(2, 3, V, dtype=dtype)
        check_select(x, torch.zeros(2, 3), count=count, dev=cuda)
        x[:, :, ::7] = 1.0
        x[1, 2] = x[1, 1] = -0.0
        check_select(x, torch.zeros(2, 3), count=count, dev=cuda)
        g = torch.Generator().manual_seed(V)
        x = torch.randint(-2, 3, (2, 3, V), generator=g).to(dtype)
        x[:, 1] = x[:, 0]
        check_select(x, torch.tensor([[-1.0, -1.0, -1.0], [-3.0, -3.0, -2.0]]), count=count, dev=cuda)


@pytest.mark.parametrize("V", [2000, 9000])
def test_best_values_in_few_lanes(cuda, V):
    """The best logits where one lane, or every lane in turn, holds many of them."""
    for stride, block in ((2048, 8), (1024, 4), (8, 1), (64, 64)):
        at = torch.arange(V)
        hot = (at % stride) < block
        x = torch.where(hot, 50.0 + at.float() / V, -at.float() / V).expand(1, 2, V).contiguous()
        for count in (8, 64):
            check_select(x, torch.tensor([[0.0, -0.001]]), count=count, dev=cuda)
            check_select(x.flip(-1), torch.tensor([[0.0, 0.0]]), count=count, dev=cuda)


def test_sorted_rows(cuda):
    up = torch.linspace(-5, 5, 8192).expand(1, 2, 8192).contiguous()
    for x in (up, up.flip(-1)):
        check_select(x, torch.tensor([[-1.0, -1.5]]), count=64, dev=cuda)


def test_masked_rows(cuda):
    x, s = make(2, 4, 9000, BF16, 1)
    x[0, 0] = -INF                      # no continuation at all
    x[0, 1, :8999] = -INF               # one
    x[0, 2, 10:] = -INF                 # fewer than the candidates
    x[1, :, ::2] = -INF
    x[1, 3] = torch.finfo(BF16).min     # the type's lowest value everywhere: uniform
    s[1, 1] = -INF
    for count in (1, 8, 64):
        check_select(x, s, count=count, dev=cuda)
    check_select(torch.full((1, 3, 500), -INF), torch.zeros(1, 3), count=20, dev=cuda)
    check_select(x, torch.full((2, 4), -INF), count=8, dev=cuda)


def test_a_forced_token_keeps_the_score(cuda):
    """Rows with one logit left have a log-probability of exactly 0: they tie with finished
    beams of the same score."""
    x = torch.full((1, 4, 6000), -INF)
    for w, at in enumerate((5999, 17, 2048, 300)):
        x[0, w, at] = 1.4745025634765625 * (w + 1)
    s = torch.tensor([[-1.0, -1.0, -1.0, -1.0]])
    for dtype in (F32, BF16):
        check_select(x.to(dtype), s, count=6, dev=cuda)
        done = torch.tensor([[False, True, False, True]])
        check_select(x.to(dtype), s, count=6, finished=done, eos=3, dev=cuda)
        got = select(x.to(dtype).to(cuda), s.to(cuda))
        assert (got[0] == -1.0).all()


def test_few_logits_left(cuda):
    """Constrained beams: so few tokens allowed that lists fill up with masked ones, with
    more candidates wanted than any list has."""
    for W, V, count, keep in ((27, 9176, 54, 0.001), (64, 4100, 64, 0.0005), (16, 20000, 32, 0.0001),
                              (200, 3000, 64, 0.001)):
        x, s = make(1, W, V, BF16, V)
        g = torch.Generator().manual_seed(W)
        x.masked_fill_(torch.rand(1, W, V, generator=g) > keep, -INF)
        check_select(x, s, count=count, dev=cuda)
        done = torch.rand(1, W, generator=g) < 0.3
        check_select(x, s, count=count, finished=done, eos=V // 2, dev=cuda)


def test_first_step(cuda):
    """Identical beams of which the first stands for all."""
    x, _ = make(2, 1, 5000, F16, 9)
    s = torch.tensor([[0.0, -INF, -INF, -INF]] * 2)
    check_select(x.expand(2, 4, 5000).contiguous(), s, dev=cuda)


def test_nan_and_inf(cuda):
    x, s = make(4, 3, 700, F32, 4)
    x[0, 1, 5] = math.nan
    x[1, 2, 699] = INF
    s[2, 0] = math.nan
    s[3, 1] = INF
    for count in (2, 10):
        check_select(x, s, count=count, dev=cuda)
    x[:] = math.nan
    check_select(x, s, count=64, dev=cuda)


@pytest.mark.parametrize("eos", [0, 17, 2999])
def test_finished_beams(cuda, eos):
    x, s = make(3, 4, 3000, BF16, 6)
    done = torch.tensor([[True, False, False, True], [True] * 4, [False] * 4])
    x[0, 0] = math.nan  # not read
    for count in (4, 8, 64):
        check_select(x, s, count=count, finished=done, eos=eos, dev=cuda)
    s[1, 2] = -INF
    check_select(x[:, :, :5].contiguous(), s, count=9, finished=done, eos=min(eos, 4), dev=cuda)


def test_strides(cuda):
    x, s = make(2, 3, 1001, BF16, 2)
    want = select(x.to(cuda), s.to(cuda))
    wide = torch.full((2, 3, 1500), 9.0, dtype=BF16, device=cuda)
    wide[:, :, 3:1004] = x.to(cuda)
    swapped = x.to(cuda).transpose(0, 1).contiguous().transpose(0, 1)
    spaced = torch.zeros(2, 3, 2002, dtype=BF16, device=cuda)[:, :, ::2]
    spaced.copy_(x)
    for view in (wide[:, :, 3:1004], swapped, spaced):
        got = select(view, s.to(cuda).t().contiguous().t())
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    same = select(x[:1, :1].to(cuda).expand(2, 3, 1001), torch.zeros(2, 3, device=cuda))
    assert torch.equal(same[1][0], same[1][1])


def test_equal_rows_tie_whatever_their_alignment(cuda):
    """Rows of an odd vocabulary start at every alignment; equal rows have equal values."""
    row = (torch.randn(5001, generator=torch.Generator().manual_seed(0)) * 3).to(F16)
    check_select(row.expand(1, 8, 5001).contiguous(), torch.full((1, 8), -2.0), count=16, dev=cuda)


# --------------------------------------------------------------------------
# Reordering
# --------------------------------------------------------------------------
def caches(L, N, W, M, P, Hkv, D, dtype, seed=0, spare=2):
    g = torch.Generator().manual_seed(seed)
    pool = N * W * M + spare
    table = torch.randperm(pool, generator=g)[:N * W * M].to(torch.int32).view(N * W, M)
    kp = torch.randn(L, pool, Hkv, P, D, generator=g).to(dtype)
    return kp, torch.randn(L, pool, Hkv, P, D, generator=g).to(dtype), table


def check_reorder(kp, vp, table, lens, parents, dev):
    from llm_cuda.kernels.beam_search import paged_kv_reorder

    k, v = kp.to(dev), vp.to(dev)
    old = table.to(dev)
    new = paged_kv_reorder(k, v, old, lens.to(dev), parents.to(dev))
    torch.cuda.synchronize()
    rk, rv, rt = ref_reorder(kp, vp, table, lens, parents)
    assert torch.equal(new.cpu(), rt) and torch.equal(old.cpu(), table)
    assert torch.equal(k.cpu(), rk) and torch.equal(v.cpu(), rv)
    return k, v, new


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("L,N,W,P,Hkv,D,t", [
    (1, 1, 1, 16, 2, 64, 20), (3, 2, 4, 16, 2, 64, 37), (2, 1, 8, 64, 8, 128, 63),
    (2, 3, 5, 16, 1, 7, 33), (1, 2, 4, 24, 2, 20, 50), (2, 2, 4, 16, 2, 64, 32),
    (1, 1, 4, 16, 2, 64, 0), (1, 1, 4, 16, 2, 64, 1), (2, 1, 70, 16, 1, 16, 19)])
def test_reorder(cuda, L, N, W, P, Hkv, D, t, dtype):
    M = t // P + 2
    kp, vp, table = caches(L, N, W, M, P, Hkv, D, dtype)
    g = torch.Generator().manual_seed(t)
    lens = torch.full((N * W,), t, dtype=torch.int32)
    for parents in (torch.randint(0, W, (N, W), generator=g), torch.zeros(N, W, dtype=torch.int64),
                    torch.full((N, W), W - 1), torch.arange(W).expand(N, W).contiguous(),
                    torch.arange(W).flip(0).expand(N, W).contiguous()):
        check_reorder(kp, vp, table, lens, parents, cuda)


def test_reorder_widest_and_full_table(cuda):
    kp, vp, table = caches(1, 1, 256, 2, 16, 1, 8, BF16)
    parents = torch.randint(0, 256, (1, 256), generator=torch.Generator().manual_seed(0))
    for t in (31, 32, 40):  # 40: past the capacity, which it stands for
        check_reorder(kp, vp, table, torch.full((256,), t, dtype=torch.int32), parents, cuda)
    check_reorder(kp, vp, table, torch.full((256,), -3, dtype=torch.int32), parents, cuda)


def test_reorder_out_of_range(cuda):
    """Parents outside the group stand for the sequence; pages outside the pool are left out."""
    kp, vp, table = caches(2, 2, 4, 3, 16, 2, 64, BF16)
    lens = torch.full((8,), 20, dtype=torch.int32)
    check_reorder(kp, vp, table, lens, torch.tensor([[-1, 0, 4, 2 ** 40], [1, 1, -2 ** 62, 1]]), cuda)
    table[1, 1], table[6, 1] = -1, kp.shape[1]
    check_reorder(kp, vp, table, lens, torch.tensor([[1, 1, 1, 0], [2, 0, 0, 0]]), cuda)


def test_reorder_views_and_out(cuda):
    from llm_cuda.kernels.beam_search import paged_kv_reorder

    kp, vp, table = caches(2, 2, 3, 3, 16, 2, 64, BF16)
    lens = torch.full((6,), 21, dtype=torch.int32)
    parents = torch.tensor([[0, 0, 2], [1, 1, 1]])
    rk, rv, rt = ref_reorder(kp, vp, table, lens, parents)
    both = torch.stack([kp, vp], 2).transpose(3, 4).contiguous().to(cuda)  # [L, N, 2, P, H, D]
    k, v = (both[:, :, i].transpose(2, 3) for i in range(2))
    out = torch.full((6, 5), -9, dtype=torch.int32, device=cuda)
    got = paged_kv_reorder(k, v, table.to(cuda), lens.to(cuda), parents.to(cuda), out=out[:, 1:4])
    assert got.data_ptr() == out[:, 1:4].data_ptr()
    assert torch.equal(out[:, 1:4].cpu(), rt) and (out[:, 0] == -9).all() and (out[:, 4] == -9).all()
    assert torch.equal(k.cpu(), rk) and torch.equal(v.cpu(), rv)
    # one layer, without its dimension
    k1, v1 = kp[0].clone().to(cuda), vp[0].clone().to(cuda)
    t1 = paged_kv_reorder(k1, v1, table.to(cuda), lens.to(cuda), parents.to(cuda))
    assert torch.equal(t1.cpu(), rt) and torch.equal(k1.cpu(), rk[0]) and torch.equal(v1.cpu(), rv[0])
    tbl = table.to(cuda)
    with pytest.raises(RuntimeError, match="overlaps"):
        paged_kv_reorder(k1, v1, tbl, lens.to(cuda), parents.to(cuda), out=tbl)


def test_reorder_twice_keeps_every_sequence(cuda):
    """Contents followed by hand over several steps: each sequence holds what its line of
    parents wrote."""
    N, W, M, P = 2, 4, 5, 8
    kp, vp, table = caches(1, N, W, M, P, 1, 8, F32)
    k, v, t = kp.to(cuda), vp.to(cuda), table.to(cuda)
    from llm_cuda.kernels.beam_search import paged_kv_reorder

    g = torch.Generator().manual_seed(1)
    held = [[] for _ in range(N * W)]
    for step in range(30):
        for b in range(N * W):
            mark = 1000.0 * step + b
            k[0, t[b, step // P].long(), 0, step % P] = mark
            v[0, t[b, step // P].long(), 0, step % P] = -mark
            held[b].append(mark)
        parents = torch.randint(0, W, (N, W), generator=g)
        lens = torch.full((N * W,), step + 1, dtype=torch.int32, device=cuda)
        t = paged_kv_reorder(k, v, t, lens, parents.to(cuda))
        held = [list(held[(b // W) * W + int(parents[b // W, b % W])]) for b in range(N * W)]
    for b in range(N * W):
        ids = t[b, torch.arange(30, device=cuda) // P].long()
        slot = torch.arange(30, device=cuda) % P
        assert k[0, ids, 0, slot, 0].tolist() == held[b]
        assert v[0, ids, 0, slot, 7].tolist() == [-m for m in held[b]]


def test_captured_step(cuda):
    """Selection and reordering in one captured graph, replayed on changing inputs with
    eager calls between, against eager calls."""
    from llm_cuda.kernels.beam_search import beam_select, paged_kv_reorder

    kp, vp, table = caches(2, 2, 4, 3, 16, 2, 64, BF16)
    k, v, t = kp.to(cuda), vp.to(cuda), table.to(cuda)
    lens = torch.full((8,), 20, dtype=torch.int32, device=cuda)
    x, s = (y.to(cuda) for y in make(2, 4, 3000, BF16, 0))

    def step():
        got = beam_select(x, s)
        return got, paged_kv_reorder(k, v, t, lens, got[2])

    step()
    k.copy_(kp)
    v.copy_(vp)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, new = step()
    for i in range(4):
        x.copy_(make(2, 4, 3000, BF16, 10 + i)[0])
        lens.fill_(5 + 9 * i)
        k.copy_(kp)
        v.copy_(vp)
        graph.replay()
        torch.cuda.synchronize()
        saved = k.clone(), v.clone()
        k.copy_(kp)
        v.copy_(vp)
        want, want_new = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(new, want_new)
        assert torch.equal(k, saved[0]) and torch.equal(v, saved[1])


@pytest.mark.parametrize("N,W,V,K", [(1, 4, 32000, 4), (3, 5, 1000, 8), (2, 24, 1397, 24), (1, 32, 700, 64), (40, 2, 999, 2)])
def test_one_launch_equals_two(cuda, monkeypatch, N, W, V, K):
    """The join by the last workgroup and the merge launch give the same bits, and leave the
    tickets at zero."""
    from llm_cuda.kernels import _ops

    for seed in range(4):
        x, s = make(N, W, V, BF16, seed)
        if seed == 3:
            s[:, 1:] = -INF  # one live beam
        done = torch.zeros(N, W, dtype=torch.bool)
        done[:, seed % W] = seed == 2
        check_select(x, s, count=K, finished=done, eos=7, dev=cuda)
        args = (x.to(cuda), s.to(cuda))
        kw = dict(num_candidates=K, finished=done.to(cuda), eos_token_id=7)
        one = select(*args, **kw)
        stream = torch.cuda.current_stream().cuda_stream
        assert not _ops._JOIN_COUNTERS[("beam_select", 0, stream)].any()
        with monkeypatch.context() as m:
            m.setattr(_ops, "_join_counters", lambda *key: None)
            two = select(*args, **kw)
        assert all(torch.equal(a, b) for a, b in zip(one, two))


def test_two_streams_at_once(cuda):
    """Calls on two streams in flight together, many of them, each with its own tickets."""
    from llm_cuda.kernels.beam_search import beam_select

    jobs = [tuple(y.to(cuda) for y in make(2, 4, 5000, BF16, s)) for s in range(2)]
    want = [beam_select(*j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(50):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(beam_select(*jobs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))


def test_reorder_overlapping_tables(cuda):
    """A table whose rows are one expanded row is read as such; an out that overlaps the
    table, or itself, is refused."""
    from llm_cuda.kernels.beam_search import paged_kv_reorder

    kp, vp, _ = caches(1, 1, 4, 3, 8, 1, 16, BF16)
    k, v = kp.to(cuda), vp.to(cuda)
    row = torch.tensor([[3, 1, 2]], dtype=torch.int32, device=cuda)
    lens = torch.full((4,), 16, dtype=torch.int32, device=cuda)  # whole pages: nothing is copied
    parents = torch.tensor([[2, 2, 0, 1]], device=cuda)
    new = paged_kv_reorder(k, v, row.expand(4, 3), lens, parents)
    assert torch.equal(new, row.repeat(4, 1))
    assert torch.equal(k.cpu(), kp) and torch.equal(v.cpu(), vp)
    pool = row.repeat(8, 1)
    for table, out in ((pool[:4], pool[:4]), (pool[:4], pool[3:7]), (pool[3:7], pool[:4]),
                       (pool[:4], torch.empty(1, 3, dtype=torch.int32, device=cuda).expand(4, 3))):
        with pytest.raises(RuntimeError if out.stride(0) else ValueError):
            paged_kv_reorder(k, v, table, lens, parents, out=out)
    assert torch.equal(paged_kv_reorder(k, v, pool[:4], lens, parents, out=pool[4:]), row.repeat(4, 1))
