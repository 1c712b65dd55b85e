"""Verification of drafted tokens against the 64-bit definition: tokens and counts are equal.

Whether a draft stands is a comparison of numbers that the kernel has to 1e-6 relative, and
the new token a place on a running sum in 64 bits (off by some 2^-45); random numbers that
fall closer than that to a border are replaced, which hardly any do.
"""
import math

import pytest
import torch

from oracle.speculative import distribution, verify_draft as oracle

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
I32 = torch.int32


def make(B, K, V, dtype, seed, drawn=True, near=0.7, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, K + 1, V, generator=g) * spread
    hot = torch.randint(0, V, (B, K + 1, 8), generator=g)
    x.scatter_add_(2, hot, 7 * torch.rand(B, K + 1, 8, generator=g))
    y = (x[:, :K] + near * torch.randn(B, K, V, generator=g)).to(dtype)
    noise = -torch.log(-torch.log(torch.rand(B, K, V, generator=g).clamp(1e-9, 1 - 1e-6)))
    d = (y.float() + noise).argmax(-1) if K else torch.zeros(B, 0, dtype=torch.int64)
    return dict(logits=x.to(dtype), draft_tokens=d, uniforms=torch.rand(B, K + 1, generator=g),
                draft_logits=y if drawn and K else None, draft_lens=None, temperature=1.0)


def on(dev, args):
    return {k: t.to(dev) if isinstance(t, torch.Tensor) else t for k, t in args.items()}


def check(args, dev, margin=True):
    from llm_cuda.kernels.speculative import verify_draft_tokens

    tokens, accepted, close, near = oracle(**args)
    g = torch.Generator().manual_seed(99)
    while margin and (close < 4e-6 or near < 1e-11):
        args["uniforms"] = torch.rand(args["uniforms"].shape, generator=g)
        tokens, accepted, close, near = oracle(**args)
    got, count = verify_draft_tokens(**on(dev, args))
    torch.cuda.synchronize()
    assert got.dtype == torch.int64 and count.dtype == I32
    assert torch.equal(count.cpu(), accepted), "accepted"
    assert torch.equal(got.cpu(), tokens), "tokens"
    return accepted


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (1, 4, 3), (3, 2, 64), (2, 5, 65), (4, 3, 1000), (2, 4, 2047),
                                   (2, 3, 2048), (1, 7, 2049), (3, 2, 8191), (1, 3, 32000)])
@pytest.mark.parametrize("drawn", [True, False])
def test_sizes_and_types(cuda, B, K, V, dtype, drawn):
    # (few tokens: flat rows, or nothing is ever in doubt)
    check(make(B, K, V, dtype, B * 100 + K * 10 + V, drawn), cuda, margin=V > 16)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [1, 17, 5000, 128256])
def test_sampling_without_drafts(cuda, V, dtype):
    check(make(5, 0, V, dtype, V), cuda, margin=V > 16)


@pytest.mark.parametrize("temperature", [1.0, 0.7, 1.9, 0.05, 1e-30, 0.0, -1.0, math.inf, math.nan])
@pytest.mark.parametrize("drawn", [True, False])
def test_temperatures(cuda, temperature, drawn):
    args = make(4, 3, 3000, BF16, 5, drawn)
    args["temperature"] = temperature
    check(args, cuda, margin=1e-3 < temperature < math.inf)


def test_temperatures_of_each_sequence(cuda):
    args = make(6, 3, 2500, F16, 6)
    args["temperature"] = torch.tensor([1.0, 0.0, 0.6, math.nan, math.inf, 2.5])
    check(args, cuda, margin=False)


def test_many_acceptances_and_refusals(cuda):
    seen = set()
    for near in (0.0, 0.3, 1.0, 4.0):
        args = make(24, 6, 1200, BF16, int(10 * near), near=near)
        seen |= set(check(args, cuda).tolist())
    assert seen == set(range(7))


def test_equal_distributions_accept(cuda):
    """p = q: u < 1 always accepts, at every temperature."""
    for t in (1.0, 0.5, 0.0):
        args = make(8, 5, 999, F32, 3, near=0.0)
        args["logits"][:, :5] = args["draft_logits"]
        args["temperature"] = t
        if t == 0:
            args["draft_tokens"] = args["draft_logits"].argmax(-1)
        args["uniforms"][:, :5] = 1 - 2.0 ** -24
        assert (check(args, cuda, margin=False) == 5).all()


def test_ragged_drafts(cuda):
    args = make(7, 4, 1500, BF16, 8, near=0.2)
    args["draft_lens"] = torch.tensor([4, 0, 1, 3, -2, 99, 2], dtype=I32)
    check(args, cuda)
    # rows past the drafts are not looked at
    for b, n in enumerate([4, 0, 1, 3, 0, 4, 2]):
        args["logits"][b, n + 1:] = math.nan
        args["draft_logits"][b, n:] = math.inf
        args["draft_tokens"][b, n:] = -5
    check(args, cuda, margin=False)


def test_drafts_outside_the_vocabulary_are_refused(cuda):
    for drawn in (True, False):
        args = make(4, 3, 700, F32, 9, drawn)
        args["draft_tokens"][0, 0], args["draft_tokens"][1, 1] = -1, 700
        args["draft_tokens"][2, 2], args["draft_tokens"][3, 0] = 2 ** 40, -2 ** 40
        accepted = check(args, cuda, margin=False)
        assert accepted[0] == 0 and accepted[3] == 0


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("drawn", [True, False])
def test_banned_tokens(cuda, dtype, drawn):
    """Logits of -inf: most tokens, all but one, whole chunks, the drafted token, all."""
    args = make(6, 3, 5000, dtype, 10, drawn)
    x = args["logits"]
    keep = torch.rand(x.shape[1:], generator=torch.Generator().manual_seed(1)) < 0.001
    x[0] = torch.where(keep, x[0], -math.inf)
    x[1, 0, :], x[1, 0, 4321] = -math.inf, 2.0
    x[2, :, :4096] = -math.inf
    x[3, 0, args["draft_tokens"][3, 0]] = -math.inf
    x[4] = -math.inf
    if drawn:
        args["draft_logits"][5, 0] = -math.inf
        args["draft_logits"][0, :, 100:] = -math.inf
    check(args, cuda, margin=False)


@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("t", [1.0, 0.0])
def test_rows_without_finite_largest(cuda, drawn, t):
    """NaN and +inf: all mass on the first largest logit, NaN the largest."""
    args = make(6, 2, 3000, F32, 11, drawn)
    args["temperature"] = t
    x = args["logits"]
    x[0, 0, 2500] = x[0, 0, 2900] = math.nan
    x[1, 0, 17] = x[1, 0, 5] = math.inf
    x[2, :, 1000] = math.inf
    x[2, :, 2999] = math.nan
    x[3, 0] = math.nan
    args["draft_tokens"][2, 0] = 2999  # (stands)
    if drawn:
        args["draft_logits"][4, 0, 44] = math.nan
        args["draft_tokens"][4, 0] = 44
        args["draft_logits"][5, 0, 2048] = math.inf
    check(args, cuda, margin=False)


def test_ties_go_to_the_first(cuda):
    args = make(3, 2, 4100, BF16, 12)
    args["temperature"] = 0.0
    args["logits"][0, 0, [4099, 2047, 2048]] = 40.0
    args["logits"][1, 0] = 0.0
    args["logits"][2, 0, [9, 8]] = 40.0
    args["draft_tokens"][0, 0], args["draft_tokens"][2, 0] = 2048, 8
    accepted = check(args, cuda, margin=False)
    assert accepted[0] == 0 and accepted[2] >= 1


def test_extreme_uniforms(cuda):
    """0, and the largest float below 1: the first and the last token of weight."""
    for drawn in (True, False):
        args = make(4, 2, 3000, F32, 13, drawn)
        args["logits"][:, :, 2990:] = -math.inf
        args["logits"][:, :, :7] = -math.inf
        args["uniforms"][:2] = 0.0
        args["uniforms"][2:] = 1 - 2.0 ** -24
        check(args, cuda, margin=False)


def test_a_vanishing_residual_samples_the_target(cuda):
    """A refused draft whose distributions agree (it has no mass in either)."""
    args = make(2, 1, 2000, F32, 14, near=0.0)
    args["logits"][:, 0] = args["draft_logits"][:, 0]
    args["logits"][:, 0, 5] = args["draft_logits"][:, 0, 5] = -math.inf
    args["draft_tokens"][:] = 5
    assert not check(args, cuda, margin=False).any()


def test_tokens_are_distributed_as_the_target(cuda):
    """The first token of 1 draft, over evenly spaced random numbers: a grid of n x n points
    takes each token's probability to within 3 intervals of either axis."""
    from llm_cuda.kernels.speculative import verify_draft_tokens

    V, n = 7, 128
    g = torch.Generator().manual_seed(15)
    x, y = torch.randn(2, V, generator=g), torch.randn(V, generator=g)
    p, q = distribution(x[0], 1.0), distribution(y, 1.0)
    u = (torch.arange(n) + 0.5) / n
    share = torch.zeros(V, dtype=torch.float64)
    for d in range(V):
        B = n * n
        uni = torch.stack([u.repeat_interleave(n), u.repeat(n)], 1)
        tokens, accepted = verify_draft_tokens(
            x.expand(B, 2, V).to(cuda), torch.full((B, 1), d, device=cuda), uni.to(cuda),
            draft_logits=y.expand(B, 1, V).to(cuda))
        first = torch.bincount(tokens[:, 0].cpu(), minlength=V).double() / B
        share += q[d] * first
    assert ((share - p).abs() <= 3.0 / n).all()


def test_strides(cuda):
    from llm_cuda.kernels.speculative import verify_draft_tokens

    args = on(cuda, make(3, 3, 1001, BF16, 16))
    want = verify_draft_tokens(**args)
    wide = torch.zeros(3, 9, 1500, dtype=BF16, device=cuda)
    wide[:, 1::2, 3:1004][:, :4] = args["logits"]
    moved = dict(args, logits=wide[:, 1::2, 3:1004][:, :4],
                 draft_logits=args["draft_logits"].transpose(0, 1).contiguous().transpose(0, 1),
                 draft_tokens=args["draft_tokens"].T.contiguous().T, uniforms=args["uniforms"].T.contiguous().T)
    got = verify_draft_tokens(**moved)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = verify_draft_tokens(**dict(args, logits=args["logits"].transpose(1, 2).contiguous().transpose(1, 2)))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_empty_batch_and_backward(cuda):
    from llm_cuda.kernels.speculative import verify_draft_tokens

    args = on(cuda, make(2, 2, 50, F32, 17))
    tokens, accepted = verify_draft_tokens(
        args["logits"][:0], args["draft_tokens"][:0], args["uniforms"][:0])
    assert tokens.shape == (0, 3) and accepted.shape == (0,)
    tokens, _ = verify_draft_tokens(**dict(args, logits=args["logits"].clone().requires_grad_(True)))
    assert not tokens.requires_grad


def test_graph_replays_and_streams(cuda):
    from llm_cuda.kernels.speculative import verify_draft_tokens

    many = [on(cuda, make(3, 4, 9000, BF16, 20 + i)) for i in range(3)]
    want = [verify_draft_tokens(**a) for a in many]
    held = {k: t.clone() if isinstance(t, torch.Tensor) else t for k, t in many[0].items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = verify_draft_tokens(**held)
    for _ in range(2):
        for a, w in zip(many, want):
            for k, t in a.items():
                if isinstance(t, torch.Tensor):
                    held[k].copy_(t)
            graph.replay()
            verify_draft_tokens(**a)
            torch.cuda.synchronize()
            assert torch.equal(out[0], w[0]) and torch.equal(out[1], w[1])
    streams = [torch.cuda.Stream() for _ in many]
    for _ in range(5):
        got = []
        for a, s in zip(many, streams):
            with torch.cuda.stream(s):
                got.append(verify_draft_tokens(**a))
        torch.cuda.synchronize()
        for x, w in zip(got, want):
            assert torch.equal(x[0], w[0]) and torch.equal(x[1], w[1])
