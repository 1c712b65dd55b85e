"""Attention of sequences that share a prefix against the 64-bit oracle.

Tolerance of an output element. Scores: D products summed in fp32 are off by at
most D * 2^-24 * sum |q_d k_d| * scale; for N(0, 1) rows of D <= 256 that is
below 1e-4 (256 * 6e-8 * 256 * 0.8 * 0.0625 = 2e-4 at D 256 as a bound no sum
comes near). An error of d in the scores moves a softmax mean by at most 2 d *
max|v|. Weights rounded to the data type (2^-8 relative in bf16, 2^-11 in f16)
move it by that times max|v|, and the result is rounded once more.
"""
import math

import pytest
import torch

from oracle.beam import shared_prefix_decode

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (BF16, F16, F32)}


def make(N, W, Hq, Hkv, D, P, plens, slens, dtype, seed=0, spare=3):
    """Shuffled pages, unused table entries at -1, and NaN in every slot that holds no token."""
    g = torch.Generator().manual_seed(seed)
    B = N * W
    need_p = [-(-n // P) for n in plens]
    need_s = [-(-n // P) for n in slens]
    pool = sum(need_p) + sum(need_s) + spare
    order = torch.randperm(pool, generator=g).to(torch.int32)
    kp = torch.randn(pool, Hkv, P, D, generator=g).to(dtype)
    vp = torch.randn(pool, Hkv, P, D, generator=g).to(dtype)
    used = torch.zeros(pool, P, dtype=torch.bool)
    at = 0

    def table(rows, need, lens):
        nonlocal at
        t = torch.full((rows, max(need + [1])), -1, dtype=torch.int32)
        for r in range(rows):
            t[r, :need[r]] = order[at:at + need[r]]
            at += need[r]
            for i in range(lens[r]):
                used[int(t[r, i // P]), i % P] = True
        return t

    pt, bt = table(N, need_p, plens), table(B, need_s, slens)
    for pages in (kp, vp):
        pages.transpose(1, 2)[~used] = math.nan
    q = torch.randn(B, Hq, 1, D, generator=g).to(dtype)
    return (q, kp, vp, pt, torch.tensor(plens, dtype=torch.int32), bt,
            torch.tensor(slens, dtype=torch.int32))


def check(args, got, scale=None):
    q, kp, vp = args[:3]
    out, lse = got
    ref, ref_lse = shared_prefix_decode(*args, scale=scale)
    D = q.shape[-1]
    assert out.shape == q.shape and out.dtype == q.dtype
    out, lse = out.double().cpu().reshape(ref.shape), lse.double().cpu()
    empty = torch.isneginf(ref_lse)
    assert torch.equal(torch.isneginf(lse), empty)
    assert not out[empty].any()
    assert torch.isfinite(out).all()
    vmax = vp[~vp.isnan()].abs().max().item()
    half = HALF_ULP[q.dtype]
    score = 1e-4 * max(1.0, (scale or D ** -0.5) * D ** 0.5)
    err = (out - ref).abs() - half * ref.abs()
    limit = vmax * (2 * score + (half if q.dtype != F32 else 0.0))
    assert err.max().item() <= limit, (err.max().item(), limit)
    if (~empty).any():
        d = (lse - ref_lse)[~empty].abs() - 2e-6 * ref_lse[~empty].abs()
        assert d.max().item() <= score


def run(args, dev, **kw):
    from llm_cuda.kernels.triton.decode_attention import shared_prefix_decode_attention

    got = shared_prefix_decode_attention(*(t.to(dev) for t in args), return_lse=True, **kw)
    torch.cuda.synchronize()
    return got


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("Hq,Hkv,D", [(32, 8, 128), (16, 8, 64), (8, 2, 32), (4, 1, 72), (6, 2, 256),
                                      (3, 1, 20), (40, 1, 64), (2, 2, 7)])
def test_head_layouts_and_types(cuda, Hq, Hkv, D, dtype):
    args = make(2, 3, Hq, Hkv, D, 16, [150, 37], [5, 40, 0, 17, 1, 64], dtype)
    check(args, run(args, cuda))


@pytest.mark.parametrize("P", [1, 8, 16, 24, 32, 48, 64, 128, 256])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_page_sizes(cuda, P, dtype):
    args = make(2, 2, 8, 2, 64, P, [129, 300], [1, 33, 130, 64], dtype, seed=P)
    check(args, run(args, cuda))


@pytest.mark.parametrize("plen", [0, 1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 500, 1025])
@pytest.mark.parametrize("dtype,D", [(BF16, 128), (F16, 64), (F32, 64)])
def test_prefix_lengths(cuda, plen, dtype, D):
    args = make(1, 3, 8, 2, D, 32, [plen], [0, 1, 70], dtype, seed=plen)
    check(args, run(args, cuda))


@pytest.mark.parametrize("W", [1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 40, 70])
def test_group_widths(cuda, W):
    lens = [(5 * i) % 21 for i in range(2 * W)]
    args = make(2, W, 8, 2, 64, 16, [100, 260], lens, BF16, seed=W)
    check(args, run(args, cuda))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_no_tokens_at_all(cuda, dtype):
    args = make(2, 2, 8, 2, 64, 16, [0, 20], [0, 3, 0, 0], dtype)
    check(args, run(args, cuda))
    none = list(args)
    none[3], none[5] = args[3][:, :0], args[5][:, :0]  # tables without columns: lengths clamp to 0
    out, lse = run(none, cuda)
    assert not out.any() and torch.isneginf(lse).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_lengths_are_clamped_and_bad_pages_skipped(cuda, dtype):
    q, kp, vp, pt, pl, bt, sl = make(2, 2, 8, 2, 64, 16, [64, 128], [32, 48, 16, 48], dtype)
    pt[1, 3], bt[1, 1] = -5, kp.shape[0]  # entries outside the pool
    args = (q, kp, vp, pt, pl, bt, sl)
    check(args, run(args, cuda))
    long = (q, kp, vp, pt, torch.tensor([64, 10 ** 6], dtype=torch.int32), bt,
            torch.tensor([-7, 48, 16, 2 ** 31 - 1], dtype=torch.int32))
    check(long, run(long, cuda))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("scale", [0.02, 0.5])
def test_scale(cuda, dtype, scale):
    args = make(1, 4, 8, 2, 64, 16, [200], [9, 0, 30, 2], dtype)
    check(args, run(args, cuda, scale=scale), scale)


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (F16, 72), (F32, 64)])
def test_strides_and_dims(cuda, dtype, D):
    """Pools that are views of a larger buffer (kv heads beside tokens), q as a
    transposed projection, q without the token dimension, unaligned q."""
    from llm_cuda.kernels.triton.decode_attention import shared_prefix_decode_attention as op

    args = make(2, 3, 8, 2, D, 16, [150, 37], [5, 40, 0, 17, 1, 64], dtype)
    ref, ref_lse = run(args, cuda)
    q, kp, vp, *rest = (t.to(cuda) for t in args)
    both = torch.stack([kp, vp], dim=1).permute(0, 1, 3, 2, 4).contiguous()  # [N, 2, P, H, D]
    kv, vv = (both[:, i].transpose(1, 2) for i in range(2))
    wide = torch.empty(q.shape[0], 1, 2 * 8 * D, dtype=dtype, device=cuda)
    qv = wide[..., 8 * D:].view(-1, 1, 8, D).transpose(1, 2)
    qv.copy_(q)
    rest[0] = torch.cat([rest[0], rest[0]], 1)[:, :rest[0].shape[1]]  # row stride > width
    out, lse = op(qv, kv, vv, *rest, return_lse=True)
    assert torch.equal(out, ref) and torch.equal(lse, ref_lse)
    assert torch.equal(op(qv.squeeze(2), kv, vv, *rest), ref.squeeze(2))
    odd = torch.empty(q.numel() + 1, dtype=dtype, device=cuda)[1:].view(q.shape)
    odd.copy_(q)
    check(args, op(odd, kp, vp, *rest, return_lse=True))


def test_a_step_in_the_scores_at_every_tile(cuda):
    """Keys whose scores rise by more than the lazy-rescale threshold every 64 tokens."""
    for dtype, D in ((BF16, 128), (F16, 64), (F32, 64)):
        q, kp, vp, pt, pl, bt, sl = make(1, 4, 8, 2, D, 64, [640], [200, 64, 130, 1], dtype)
        q = (torch.ones_like(q) + 0.1 * torch.randn(q.shape)).to(dtype)
        for row, length in ((pt[0], 640), (bt[0], 200)):
            for i in range(-(-length // 64)):
                page = kp[int(row[i])]
                page[~page.isnan()] = (page + 6.0 * i * D ** -0.5)[~page.isnan()].to(dtype)
        args = (q, kp, vp, pt, pl, bt, sl)
        check(args, run(args, cuda), None)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_equals_the_paged_decode_of_one_table(cuda, dtype):
    """Whole prefix pages followed by own pages in one block table: the same result
    as paged_decode_attention over it, up to rounding."""
    from llm_cuda.kernels.triton.decode_attention import paged_decode_attention

    args = make(2, 4, 8, 2, 64, 32, [128, 128], [40, 3, 33, 64, 1, 2, 3, 63], dtype)
    out, lse = run(args, cuda)
    q, kp, vp, pt, pl, bt, sl = (t.to(cuda) for t in args)
    both = torch.cat([pt.repeat_interleave(4, 0), bt], 1).contiguous()
    one, one_lse = paged_decode_attention(q, kp, vp, both, sl + 128, return_lse=True)
    assert (out - one).abs().max().item() <= (0.05 if dtype == BF16 else 1e-3)
    assert (lse - one_lse).abs().max().item() <= 1e-3


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_nan_reaches_the_output_of_its_sequence_alone(cuda, dtype):
    q, kp, vp, pt, pl, bt, sl = make(1, 4, 4, 2, 64, 16, [200], [30, 30, 30, 30], dtype)
    vp[int(bt[1, 0]), 0, 3] = math.nan
    q[2, 0] = math.nan
    out, lse = run((q, kp, vp, pt, pl, bt, sl), cuda)
    bad = out.isnan().any(-1).squeeze(-1).cpu()
    want = torch.zeros(4, 4, dtype=torch.bool)
    want[1, :2] = True  # the heads of kv head 0
    want[2, 0] = True
    assert torch.equal(bad, want)
    assert torch.equal(lse.isnan().cpu(), torch.tensor([[False] * 4] * 2 + [[True] + [False] * 3] + [[False] * 4]))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_captured_and_replayed(cuda, dtype):
    """Replays follow lengths and tables that change in place, with eager work of
    another shape between them."""
    from llm_cuda.kernels.triton.decode_attention import shared_prefix_decode_attention as op

    args = [t.to(cuda) for t in make(1, 8, 8, 2, 64, 16, [300], [100] * 8, dtype)]
    other = [t.to(cuda) for t in make(2, 3, 4, 2, 64, 16, [90, 10], [7] * 6, dtype, seed=5)]
    kp, vp = args[1], args[2]
    for t in (kp, vp):
        t.copy_(torch.nan_to_num(t, nan=0.25))
    op(*args, return_lse=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out, lse = op(*args, return_lse=True)
    for step in range(4):
        args[4].fill_(300 - 37 * step)
        args[6].copy_(torch.randint(0, 101, (8,), dtype=torch.int32))
        args[0].normal_()
        graph.replay()
        op(*other)
        want, want_lse = op(*args, return_lse=True)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D,W,plen,cap", [(128, 4, 300, 20), (64, 4, 9, 20), (32, 1, 70, 0), (128, 8, 900, 130),
                                          (64, 5, 0, 3)])
def test_one_launch_equals_two(cuda, monkeypatch, dtype, D, W, plen, cap):
    """The join by the last workgroup and the merge launch give the same bits, and leave the
    tickets at zero."""
    from llm_cuda.kernels import _ops
    from llm_cuda.kernels.triton.decode_attention import shared_prefix_decode_attention as op

    for seed in range(6):
        lens = [(7 * seed + 3 * i) % (cap + 1) for i in range(2 * W)]
        args = [t.to(cuda) for t in make(2, W, 8, 2, D, 8, [plen, plen // 2], lens, dtype, seed=seed)]
        one = op(*args, return_lse=True)
        torch.cuda.synchronize()
        stream = torch.cuda.current_stream().cuda_stream
        assert not _ops._JOIN_COUNTERS[("shared_prefix", 0, stream)].any()
        with monkeypatch.context() as m:
            m.setattr(_ops, "_join_counters", lambda *key: None)
            two = op(*args, return_lse=True)
        assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])


def test_two_streams_at_once(cuda):
    """Calls on two streams in flight together, many of them, each with its own tickets."""
    from llm_cuda.kernels.triton.decode_attention import shared_prefix_decode_attention as op

    jobs = [[t.to(cuda) for t in make(2, 4, 8, 2, 64, 16, [300, 90], [3 * i for i in range(8)], BF16, seed=s)]
            for s in range(2)]
    want = [op(*j, return_lse=True) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(50):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(op(*jobs[i], return_lse=True))
    torch.cuda.synchronize()
    for i in range(2):
        for out, lse in got[i]:
            assert torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])


def test_another_stream(cuda):
    args = make(1, 8, 8, 2, 64, 16, [300], [30] * 8, BF16)
    want, want_lse = run(args, cuda)
    from llm_cuda.kernels.triton.decode_attention import shared_prefix_decode_attention as op

    dev = [t.to(cuda) for t in args]
    torch.cuda.synchronize()
    got = []
    for s in (torch.cuda.Stream(), torch.cuda.Stream()):
        with torch.cuda.stream(s):
            got.append(op(*dev, return_lse=True))
    torch.cuda.synchronize()
    for out, lse in got:
        assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_offsets_past_32_bits(cuda):
    """Pages whose byte and element offsets lie past 2^32."""
    Hkv, P, D = 2, 64, 128
    pages = 2 ** 32 // (Hkv * P * D) + 40  # 4.3e9 elements: 8.6 GB a pool
    kp = torch.empty(pages, Hkv, P, D, dtype=BF16, device=cuda)
    vp = torch.empty_like(kp)
    args = make(1, 4, 8, Hkv, D, P, [200], [70, 1, 64, 0], BF16, spare=0)
    n = args[1].shape[0]
    kp[-n:], vp[-n:] = args[1].to(cuda), args[2].to(cuda)
    moved = list(t.to(cuda) for t in args)
    want, want_lse = run(args, cuda)
    moved[1], moved[2] = kp, vp
    for i in (3, 5):
        moved[i] = torch.where(moved[i] >= 0, moved[i] + (pages - n), moved[i])
    out, lse = run(moved, cuda)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_forward_only(cuda):
    from llm_cuda.kernels.triton.decode_attention import shared_prefix_decode_attention as op

    args = [t.to(cuda) for t in make(1, 2, 4, 2, 64, 16, [20], [3, 4], F32)]
    args[0].requires_grad_(True)
    with pytest.raises(NotImplementedError, match="shared_prefix_decode"):
        op(*args).sum().backward()


def test_expanded_tables(cuda):
    """One row of a table or of lengths for all groups or sequences, without a copy of it."""
    from llm_cuda.kernels.triton.decode_attention import shared_prefix_decode_attention as op

    args = [t.to(cuda) for t in make(3, 2, 8, 2, 64, 16, [100] * 3, [20] * 6, BF16)]
    q, kp, vp, ptab, plens, btab, slens = args
    wide = op(q, kp, vp, ptab[:1].expand(3, -1), plens[:1].expand(3), btab[:1].expand(6, -1), slens[:1].expand(6))
    full = op(q, kp, vp, ptab[:1].repeat(3, 1), plens[:1].repeat(3), btab[:1].repeat(6, 1), slens[:1].repeat(6))
    assert torch.equal(wide, full)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("W,plen", [(1, 2700), (2, 3900), (3, 2100)])
def test_many_ranges(cuda, monkeypatch, dtype, W, plen):
    """Long prefixes of few rows, with tickets and without: right, and the same bits."""
    from llm_cuda.kernels import _ops
    from llm_cuda.kernels.triton.decode_attention import shared_prefix_decode_attention as op

    args = [t.to(cuda) for t in make(1, W, 8, 2, 64, 64, [plen], [5 + 40 * i for i in range(W)], dtype)]
    check([t.cpu() for t in args], run([t.cpu() for t in args], cuda))
    one = op(*args, return_lse=True)
    with monkeypatch.context() as m:
        m.setattr(_ops, "_join_counters", lambda *key: None)
        two = op(*args, return_lse=True)
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
