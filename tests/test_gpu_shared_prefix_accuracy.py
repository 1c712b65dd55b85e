"""Rounding of the shared-prefix attention's 16-bit outputs, and its tiles of many rows,
against the definition in 64 bits.

A 16-bit output is rounded once, which is uniform over a step of the type there: its
mean square is the mean of step^2 / 12. Everything before it is kept to 2^-16 of each
weight or better (fp32 sums, weights in two parts) and moves the output by less than a
hundredth of that, so the root mean square over n outputs is that of the rounding, to
within its own scatter: a relative 1 / sqrt(n) or so, below 2% for the 4096 outputs and
more of these cases. 10% are allowed. (Weights of one part double the mean square; one
wrong V row of 4000 makes it 50 times as large.)
"""
import math

import pytest
import torch

from test_gpu_shared_prefix import BF16, F16, make, run

pytestmark = pytest.mark.gpu


def definition(q, kp, vp, pt, pl, bt, sl, scale=None):
    """out [B, Hq, D] and lse [B, Hq] in 64 bits; tokens of pages outside the pool are left out."""
    B, Hq, _, D = q.shape
    pages, Hkv, P, _ = kp.shape
    N, G = pt.shape[0], Hq // Hkv
    scale = D ** -0.5 if scale is None else scale

    def tokens(pool, row, n):
        at = torch.arange(n)
        page = row[at // P].long()
        live = (page >= 0) & (page < pages)
        return pool[page[live], :, at[live] % P].double()  # [tokens, Hkv, D]

    def attend(rows, k, v):
        x = rows.double() @ k.T * scale
        if not len(k):
            return torch.zeros(rows.shape, dtype=torch.float64), torch.full(rows.shape[:1], -math.inf).double()
        return torch.softmax(x, -1) @ v, torch.logsumexp(x, -1)

    out = torch.zeros(B, Hq, D, dtype=torch.float64)
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64)
    W = B // N
    for n in range(N):
        ks, vs = (tokens(p, pt[n], int(pl[n])) for p in (kp, vp))
        for h in range(Hkv):
            heads = slice(h * G, (h + 1) * G)
            seqs = slice(n * W, (n + 1) * W)
            o, m = attend(q[seqs, heads, 0].reshape(W * G, D), ks[:, h], vs[:, h])
            out[seqs, heads], lse[seqs, heads] = o.view(W, G, D), m.view(W, G)
    for b in range(B):
        ks, vs = (tokens(p, bt[b], int(sl[b])) for p in (kp, vp))
        for h in range(Hkv if len(ks) else 0):
            heads = slice(h * G, (h + 1) * G)
            o, m = attend(q[b, heads, 0], ks[:, h], vs[:, h])
            both = torch.logaddexp(lse[b, heads], m)
            out[b, heads] = (out[b, heads] * (lse[b, heads] - both).exp().unsqueeze(-1)
                             + o * (m - both).exp().unsqueeze(-1))
            lse[b, heads] = both
    return out, lse


def check_rounding(args, got, scale=None):
    want, want_lse = definition(*args, scale=scale)
    dtype = args[0].dtype
    out = got[0].double().cpu().reshape(want.shape)
    info = torch.finfo(dtype)
    step = torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=info.tiny)))) * info.eps
    rounding = (step.square().mean() / 12).sqrt().item()
    rms = (out - want).square().mean().sqrt().item()
    assert rms <= 1.1 * rounding, f"{rms / rounding:.2f} times the output's rounding"
    live = torch.isfinite(want_lse)
    lse = got[1].double().cpu()
    assert torch.equal(torch.isfinite(lse), live)
    # (64 bits against fp32 sums of D <= 128 products and of the weights: as in the other tests)
    assert ((lse - want_lse)[live].abs() <= 1e-4 + 2e-6 * want_lse[live].abs()).all()


# beams, query heads, kv heads, head_dim; rows of a prefix per kv head
LAYOUTS = [(4, 32, 8, 128), (8, 8, 2, 64), (12, 8, 2, 128), (16, 8, 2, 72), (32, 8, 2, 128),
           (40, 8, 2, 64), (5, 40, 1, 128)]  # 16, 32, 48, 64, 128, 160, 200


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("W,Hq,Hkv,D", LAYOUTS)
def test_outputs_are_rounded_once(cuda, W, Hq, Hkv, D, dtype):
    args = make(1, W, Hq, Hkv, D, 64, [2500], [(37 * i) % 400 for i in range(W)], dtype, seed=W)
    check_rounding(args, run(args, cuda))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_own_tokens_alone_are_rounded_once(cuda, dtype):
    args = make(4, 3, 8, 2, 128, 32, [0] * 4, [300 + 117 * i for i in range(12)], dtype)
    check_rounding(args, run(args, cuda))


@pytest.mark.parametrize("dtype", [BF16, F16, torch.float32])
@pytest.mark.parametrize("W,Hq,Hkv,D", [(4, 8, 2, 64), (12, 8, 2, 128), (40, 8, 2, 64)])
def test_infinite_values_stay_infinite(cuda, W, Hq, Hkv, D, dtype):
    """An infinite V entry makes that element of its sequences infinite, not NaN: every weight is
    above 0. (A score at the maximum among them, whose weight has no remainder.)"""
    args = make(1, W, Hq, Hkv, D, 16, [200], [(5 * i) % 37 for i in range(W)], dtype, seed=W)
    q, kp, vp, pt, pl, bt, sl = args
    kp[int(pt[0, 1])] = 0  # (equal scores)
    vp[int(pt[0, 1]), 0, :4, 3] = math.inf
    vp[int(pt[0, 5]), 1, 7, 5] = -math.inf
    vp[int(bt[3, 0]), 0, 2, 9] = math.inf  # 15 tokens
    out = run(args, cuda)[0].cpu().view(W, Hkv, Hq // Hkv, D)
    want = definition(*args)[0].view(out.shape)
    assert torch.equal(torch.isposinf(out), torch.isposinf(want)) and torch.isposinf(want).any()
    assert torch.equal(torch.isneginf(out), torch.isneginf(want)) and torch.isneginf(want).any()
    assert not out.isnan().any()
