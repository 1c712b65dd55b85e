"""Attention of the newest tokens in every form that a call's sizes choose, with ranges of
several whole tiles: rows that see unequal numbers of tokens, a maximum that moves all along,
and queries that are none. Tolerances: see test_gpu_paged_extend.py."""
import math

import pytest
import torch

from test_gpu_paged_extend import BF16, F16, F32, I32, check, make, run

pytestmark = pytest.mark.gpu

# type, sequences, queries, query heads, kv heads, head_dim, most tokens, ranges of a tile at most
FORMS = [
    (BF16, 3, 5, 8, 2, 64, 1700, 64),     # up to 32 rows: streams, four waves to a range
    (F16, 160, 3, 16, 4, 64, 330, 1),     # two
    (BF16, 400, 3, 16, 4, 64, 330, 1),    # one
    (BF16, 130, 5, 32, 4, 64, 520, 1),    # up to 64 rows: half tiles, one range
    (F16, 130, 5, 32, 4, 128, 520, 1),
    (BF16, 8, 7, 64, 8, 128, 2100, 8),    # several
    (F16, 6, 33, 8, 8, 64, 2900, 11),
    (BF16, 130, 12, 32, 4, 64, 520, 1),   # more rows: 128 a tile, one range
    (F16, 3, 70, 16, 4, 128, 4500, 64),   # several
    (F32, 70, 5, 16, 4, 64, 330, 1),      # fp32, one range
    (F32, 3, 20, 8, 2, 128, 1700, 64),    # several
    (BF16, 6, 9, 12, 4, 40, 520, 64),     # head_dim that is none of the kernels'
    (BF16, 6, 9, 12, 4, 17, 520, 64),     # one row a wave
]
IDS = [f"{str(f[0])[6:]}-{'-'.join(map(str, f[1:]))}" for f in FORMS]


def ragged(B, T, top, seed):
    """Lengths and queries: absent ones, more queries than tokens, the longest, and the rest."""
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(top // 3, top + 1, (B,), generator=g)
    queries = torch.randint(1, T + 1, (B,), generator=g)
    lens[0], queries[0] = top, max(1, T - 1)
    if B > 5:
        lens[2], queries[3], lens[4], queries[4] = 0, 0, T - 1, T
        queries[5] = -7
    else:
        queries[1], lens[2], queries[2] = 0, T - 1, T
    return lens.tolist(), queries.tolist()


def whole(args):
    """Output, logsumexp and sum_t p_t |v_t| in 64 bits, a sequence at a time."""
    q, kp, vp = args["q"], args["key_pages"], args["value_pages"]
    B, Hq, T, D = q.shape
    Hkv, P = kp.shape[1:3]
    out, size = torch.zeros(2, B, Hq, T, D, dtype=torch.float64)
    lse = torch.full((B, Hq, T), -math.inf, dtype=torch.float64)
    for b in range(B):
        L, n = max(0, int(args["seq_lens"][b])), min(max(0, int(args["query_lens"][b])), T)
        at, i = torch.arange(L), torch.arange(T).view(T, 1)
        seen = (at <= L - n + i) & (i < n)
        some = seen.any(1)
        if not some.any():
            continue
        page = args["block_table"][b, at // P].long()
        k, v = (p[page, :, at % P].double().permute(1, 0, 2).contiguous() for p in (kp, vp))
        x = torch.matmul(q[b].double().reshape(Hkv, -1, D), k.transpose(1, 2).contiguous()) / math.sqrt(D)
        x = x.view(Hq, T, L).masked_fill(~seen, -math.inf)
        lse[b, :, some] = torch.logsumexp(x[:, some], -1)
        p = torch.exp(x - torch.where(some.view(T, 1), lse[b].unsqueeze(-1), 0.0)).view(Hkv, -1, L)
        out[b], size[b] = torch.matmul(p, v).view(Hq, T, D), torch.matmul(p, v.abs()).view(Hq, T, D)
    return out, lse, size


def build(form, seed, page=16):
    """The call, of the ranges that the form says."""
    from llm_cuda import _native

    dtype, B, T, Hq, Hkv, D, top, ranges = form
    lens, queries = ragged(B, T, top, seed)
    args = make(lens, T, Hq, Hkv, D, page, dtype, queries=queries, seed=seed)
    cap = args["block_table"].shape[1] * page
    need = _native.size("lc_paged_extend_workspace_bytes", B, T, Hq, Hkv, D, cap, _native.lc_dtype(args["q"]))
    assert need // (B * Hq * T * (D + 1) * 4) <= ranges  # (the workspace holds all ranges' outputs)
    return args


@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_every_form(cuda, form):
    args = build(form, 1)
    check(args, run(args, cuda), want=whole(args))


@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_every_form_with_rising_scores(cuda, form):
    """Scores that rise by 2.3 in log2 every 32 tokens: past 2^8 within a range, again and again."""
    args = build(form, 2)
    dtype, P, D = form[0], 16, form[5]
    args["q"] = torch.ones_like(args["q"])
    step = 1.6 / math.sqrt(D)
    for b, n in enumerate(args["seq_lens"].tolist()):
        at = torch.arange(n)
        page = args["block_table"][b, at // P].long()
        k = args["key_pages"][page, :, at % P].float() * 0.05 + step * (at // 32).view(-1, 1, 1)
        args["key_pages"][page, :, at % P] = k.to(dtype)
    out, lse = (t.double().cpu() for t in run(args, cuda))
    ref, ref_lse, size = whole(args)
    # (a score is a sum of D products, each below the largest |k|: its fp32 sum is off by at most
    # D * 2^-24 times their absolute sum)
    top = args["key_pages"].float().nan_to_num().abs().sum(-1).max().item() / math.sqrt(D)
    d = D * 2 ** -24 * top
    half, least = torch.finfo(dtype).eps / 2, 2.0 ** -25
    weight = {BF16: 2 ** -15, F16: 2 ** -19, F32: 2 ** -22}[dtype]
    empty = torch.isneginf(ref_lse)
    assert torch.equal(torch.isneginf(lse), empty) and not out[empty].any()
    assert ((out - ref).abs() <= half * ref.abs() + (2 * d + weight) * size + least).all()
    assert ((lse - ref_lse)[~empty].abs() <= d + 2 ** -21 * ref_lse[~empty].abs()).all()


@pytest.mark.parametrize("bad", [math.inf, math.nan, "largest"])
@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_rows_that_are_no_queries_may_hold_anything(cuda, form, bad):
    """Rows past a sequence's queries, and queries before its first token: zeros, lse -inf."""
    args = build(form, 3)
    T = form[2]
    i = torch.arange(T)
    n = args["query_lens"].clamp(0, T).view(-1, 1)
    dead = (i >= n) | (args["seq_lens"].view(-1, 1) - n + i < 0)
    assert dead.any() and not dead.all()
    want = whole(args)
    bad = torch.finfo(form[0]).max if bad == "largest" else bad
    args["q"] = torch.where(dead.view(len(n), 1, T, 1), torch.tensor(bad, dtype=form[0]), args["q"])
    check(args, run(args, cuda), want=want)
