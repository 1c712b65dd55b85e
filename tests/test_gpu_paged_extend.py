"""Attention of the newest tokens over the paged cache against the 64-bit oracle.

Tolerance of an output element. Scores: D products summed in fp32 are off by at most D *
2^-24 * sum |q_d k_d| * scale, below 1e-4 for N(0, 1) rows of D <= 256 (a bound that no
sum comes near); an error of d in the scores moves a softmax mean by at most 2 d times
the weighted mean of |v|. Weights are kept to 2^-15 relative or better, and the result is
rounded once: half a step of its type. lse: the score's error and 2^-21 of its size.
"""
import math

import pytest
import torch

from oracle.speculative import paged_extend as oracle

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
I32 = torch.int32


def make(lens, T, Hq, Hkv, D, P, dtype, queries=None, seed=0, spare=3, width=None):
    """Shuffled pages, unused table entries at -1, and NaN in every slot that holds no token."""
    g = torch.Generator().manual_seed(seed)
    B = len(lens)
    need = [-(-n // P) for n in lens]
    pool = sum(need) + spare
    order = torch.randperm(pool, generator=g).to(I32)
    kp = torch.randn(pool, Hkv, P, D, generator=g).to(dtype)
    vp = torch.randn(pool, Hkv, P, D, generator=g).to(dtype)
    table = torch.full((B, max(need + [1]) if width is None else width), -1, dtype=I32)
    used, at = torch.zeros(pool, P, dtype=torch.bool), 0
    for b in range(B):
        table[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
        pos = torch.arange(lens[b])
        used[table[b, pos // P].long(), pos % P] = True
    for pages in (kp, vp):
        pages.transpose(1, 2)[~used] = math.nan
    q = torch.randn(B, T, Hq, D, generator=g).to(dtype).transpose(1, 2)
    return dict(q=q, key_pages=kp, value_pages=vp, block_table=table,
                seq_lens=torch.tensor(lens, dtype=I32),
                query_lens=None if queries is None else torch.tensor(queries, dtype=I32))


def run(args, dev, **kw):
    from llm_cuda.kernels.triton.decode_attention import paged_extend_attention

    got = paged_extend_attention(**{k: None if t is None else t.to(dev) for k, t in args.items()},
                                 return_lse=True, **kw)
    torch.cuda.synchronize()
    return got


def check(args, got, scale=None, want=None):
    q = args["q"]
    out, lse = got
    ref, ref_lse, size = oracle(**args, scale=scale) if want is None else want
    assert out.shape == q.shape and out.dtype == q.dtype and lse.dtype == F32
    out, lse = out.double().cpu(), lse.double().cpu()
    empty = torch.isneginf(ref_lse)
    assert torch.equal(torch.isneginf(lse), empty)
    assert not out[empty].any() and torch.isfinite(out).all()
    score = 1e-4 * max(1.0, (scale or q.shape[-1] ** -0.5) * q.shape[-1] ** 0.5)
    weight = {BF16: 2 ** -15, F16: 2 ** -19, F32: 2 ** -22}[q.dtype]
    half = torch.finfo(q.dtype).eps / 2
    over = (out - ref).abs() - half * ref.abs() - (2 * score + weight) * size
    assert over.max().item() <= 2.0 ** -25, over.max().item()  # (the least step of f16)
    if (~empty).any():
        d = (lse - ref_lse)[~empty].abs() - 2 ** -21 * ref_lse[~empty].abs()
        assert d.max().item() <= score


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 1, 64), (8, 2, 128), (8, 8, 32), (6, 2, 80), (5, 1, 256), (3, 3, 17),
                                      (40, 1, 64)])
def test_layouts(cuda, Hq, Hkv, D, dtype):
    args = make([70, 5, 131], 5, Hq, Hkv, D, 16, dtype, seed=D)
    check(args, run(args, cuda))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("P", [1, 3, 8, 16, 64, 256])
def test_page_sizes(cuda, P, dtype):
    args = make([100, 64, 65, 7], 4, 8, 2, 64, P, dtype, seed=P)
    check(args, run(args, cuda))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T", [1, 2, 3, 7, 8, 9, 16, 17, 31, 33, 64, 65, 100])
def test_query_counts(cuda, T, dtype):
    args = make([T, T + 1, T + 63, 200 + T], T, 8, 2, 64, 16, dtype, seed=T)
    check(args, run(args, cuda))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,G", [(5, 4), (12, 4), (40, 4), (5, 8), (24, 8), (3, 16), (9, 16)])
def test_long_contexts(cuda, T, G, dtype):
    args = make([3000, 777, 1], T, 2 * G, 2, 128, 64, dtype, seed=T * G)
    check(args, run(args, cuda))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T,Hq", [(6, 8), (20, 8), (40, 16)])
def test_ragged_queries(cuda, T, Hq, dtype):
    """Unequal and absent queries, more queries than tokens, lengths of 0 and 1, values out of range."""
    lens = [100, 50, 64, 1, 0, 3, 90, 33]
    args = make(lens, T, Hq, 2, 64, 16, dtype, queries=[T, 1, 0, 1, T, T, 3, T - 1], seed=T)
    check(args, run(args, cuda))
    args["query_lens"] = torch.tensor([T + 9, -1, -2 ** 31, 2 ** 31 - 1, T, 2, 3, 1], dtype=I32)
    check(args, run(args, cuda))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_lengths_past_the_table_are_cut(cuda, dtype):
    args = make([64, 32], 3, 4, 2, 64, 16, dtype)
    args["seq_lens"] = torch.tensor([2 ** 31 - 1, -5], dtype=I32)
    check(args, run(args, cuda))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [2, 30])
def test_pages_outside_the_pool_are_skipped(cuda, T, dtype):
    args = make([200, 130], T, 8, 2, 64, 16, dtype, seed=3)
    args["block_table"][0, 3] = -1
    args["block_table"][0, 12] = args["key_pages"].shape[0]
    args["block_table"][1, :] = -7
    check(args, run(args, cuda))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T,Hq,lens", [(5, 8, [70, 9]), (16, 8, [90, 16]), (40, 16, [100, 41]),
                                       (70, 8, [200, 75])])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_tokens_ahead_have_no_part(cuda, T, Hq, lens, bad, dtype):
    """What K and V hold at a token is nothing to the queries before it."""
    args = make(lens, T, Hq, 2, 64, 16, dtype, seed=T)
    want = oracle(**args)
    for b, n in enumerate(lens):
        first = n - T + 2  # tokens from the third query on (the second's is first - 1)
        for t in {first, first + 1, n - 1}:
            page = int(args["block_table"][b, t // 16])
            args["key_pages"][page, :, t % 16] = bad
            args["value_pages"][page, :, t % 16, ::3] = bad
    out, lse = run(args, cuda)
    for i in range(2):
        part = dict(args, q=args["q"][:, :, i:i + 1])
        check(part, (out[:, :, i:i + 1], lse[:, :, i:i + 1]),
              want=tuple(w[:, :, i:i + 1] for w in want))
    assert (~torch.isfinite(out[:, :, -1].float())).any()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T,Hq", [(3, 8), (20, 16)])
def test_infinite_values_stay_infinite(cuda, T, Hq, dtype):
    args = make([90, 40], T, Hq, 2, 64, 16, dtype, seed=T)
    args["value_pages"][int(args["block_table"][0, 1]), 0, 3, 5] = math.inf
    args["value_pages"][int(args["block_table"][1, 0]), 1, 2, 7] = -math.inf
    out = run(args, cuda)[0].double().cpu()
    ref = oracle(**args)[0]
    assert torch.equal(torch.isposinf(out), torch.isposinf(ref)) and torch.isposinf(ref).any()
    assert torch.equal(torch.isneginf(out), torch.isneginf(ref)) and torch.isneginf(ref).any()
    assert not out.isnan().any()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,Hq", [(4, 8), (12, 8), (33, 16)])
def test_rising_scores(cuda, T, Hq, dtype):
    """Scores that rise by 9 in log2 every 16 tokens: the running maximum moves all along."""
    args = make([400, 150], T, Hq, 2, 64, 16, dtype, seed=7)
    args["q"] = torch.ones_like(args["q"])
    for b, n in enumerate((400, 150)):
        for t in range(n):
            page = int(args["block_table"][b, t // 16])
            args["key_pages"][page, :, t % 16] *= 0.05
            args["key_pages"][page, :, t % 16] += 0.78 * (t // 16)
    got = run(args, cuda)
    # (scores up to 160: their fp32 sums are off by up to 64 * 2^-24 * 160 * 1.1)
    ref, ref_lse, size = oracle(**args)
    d = 64 * 2 ** -24 * 176
    half = torch.finfo(dtype).eps / 2
    over = (got[0].double().cpu() - ref).abs() - half * ref.abs() - (2 * d + 2 ** -15) * size
    assert over.max().item() <= 0
    assert ((got[1].double().cpu() - ref_lse).abs() <= d + 2 ** -21 * ref_lse.abs()).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_strides(cuda, dtype):
    """Projection views, expanded tables and lengths, pools inside a larger one, an odd offset."""
    args = {k: None if t is None else t.to(cuda) for k, t in
            make([60, 60], 6, 8, 2, 64, 16, dtype, seed=1).items()}
    want = run(args, cuda)
    g = torch.Generator().manual_seed(5)
    kp, vp = args["key_pages"], args["value_pages"]
    big = torch.zeros(kp.shape[0], 3, 2, 24, 72, dtype=dtype, device=cuda)
    big[:, 0, :, :16, :64], big[:, 2, :, :16, :64] = kp, vp
    moved = dict(args, key_pages=big[:, 0, :, :16, :64], value_pages=big[:, 2, :, :16, :64])
    q2 = torch.zeros(2, 8, 6, 131, dtype=dtype, device=cuda)
    q2[..., 1:65] = args["q"]
    moved["q"] = q2[..., 1:65]
    got = run(moved, cuda)
    check({k: None if t is None else t.cpu() for k, t in args.items()}, got)
    wide = torch.full((2, 2 * args["block_table"].shape[1]), -9, dtype=I32, device=cuda)
    wide[:, ::2] = args["block_table"]
    assert torch.equal(run(dict(args, block_table=wide[:, ::2]), cuda)[0], want[0])
    one = dict(args, block_table=args["block_table"][:1].expand(2, -1))
    assert torch.equal(run(one, cuda)[0][:1], want[0][:1])
    assert torch.equal(run(dict(args, q=args["q"].transpose(2, 3).contiguous().transpose(2, 3)), cuda)[0], want[0])
    del g


def test_scale_and_empty_calls(cuda):
    from llm_cuda.kernels.triton.decode_attention import paged_extend_attention

    args = make([60, 30], 3, 4, 2, 64, 16, BF16, seed=2)
    check(args, run(args, cuda, scale=0.3), scale=0.3)
    check(args, run(args, cuda, scale=-0.1), scale=-0.1)
    dev = {k: None if t is None else t.to(cuda) for k, t in args.items()}
    none = dict(dev, q=dev["q"][:, :, :0])
    out, lse = paged_extend_attention(**none, return_lse=True)
    assert out.shape == (2, 4, 0, 64) and lse.shape == (2, 4, 0)
    out = paged_extend_attention(dev["q"][:0], dev["key_pages"], dev["value_pages"], dev["block_table"][:0],
                                 dev["seq_lens"][:0])
    assert out.shape == (0, 4, 3, 64)
    empty = dict(dev, block_table=dev["block_table"][:, :0])
    out, lse = paged_extend_attention(**empty, return_lse=True)
    assert not out.any() and torch.isneginf(lse).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_one_query_is_a_decode(cuda, dtype):
    """T = 1 against the one-token entry."""
    from llm_cuda.kernels.triton.decode_attention import paged_decode_attention

    args = make([300, 17, 64], 1, 8, 2, 128, 32, dtype, seed=4)
    out, lse = run(args, cuda)
    dev = {k: None if t is None else t.to(cuda) for k, t in args.items()}
    o1, l1 = paged_decode_attention(dev["q"], dev["key_pages"], dev["value_pages"], dev["block_table"],
                                    dev["seq_lens"], return_lse=True)
    check(args, (out, lse))
    eps = torch.finfo(dtype).eps
    assert ((out - o1).float().abs() <= 2 * eps * o1.float().abs() + 4 * eps).all()
    assert ((lse[..., 0] - l1).abs() <= 1e-4 + 2 ** -20 * l1.abs()).all()


def test_backward_raises(cuda):
    args = {k: None if t is None else t.to(cuda) for k, t in make([20], 2, 4, 2, 64, 16, F32).items()}
    args["q"].requires_grad_(True)
    out, _ = run(args, cuda)
    with pytest.raises(NotImplementedError):
        out.sum().backward()


@pytest.mark.parametrize("T,lens", [(4, [200, 90]), (40, [400, 90])])
def test_graph_replays(cuda, T, lens):
    """Captured calls follow the device-side lengths; eager calls run between the replays."""
    from llm_cuda.kernels.triton.decode_attention import paged_extend_attention

    dev = {k: None if t is None else t.to(cuda) for k, t in make(lens, T, 8, 2, 64, 16, BF16, seed=6).items()}
    dev["query_lens"] = torch.full((2,), T, dtype=I32, device=cuda)
    paged_extend_attention(**dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out, lse = paged_extend_attention(**dev, return_lse=True)
    for step in range(4):
        dev["seq_lens"].copy_(torch.tensor([n - 7 * step for n in lens], dtype=I32))
        dev["query_lens"].copy_(torch.tensor([T - step, 1 + step], dtype=I32))
        graph.replay()
        want = paged_extend_attention(**dev, return_lse=True)
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_calls_on_two_streams(cuda):
    from llm_cuda.kernels.triton.decode_attention import paged_extend_attention

    many = [{k: None if t is None else t.to(cuda) for k, t in
             make([500 + 40 * i, 90], 5, 8, 2, 128, 16, BF16, seed=i).items()} for i in range(4)]
    want = [paged_extend_attention(**a) for a in many]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in many]
    for _ in range(5):
        got = []
        for a, s in zip(many, streams):
            with torch.cuda.stream(s):
                got.append(paged_extend_attention(**a))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
