"""The tiles of a prefix with more than 32 rows per kv head: ranges of several tiles, whose
buffers take turns and whose reference maxima move, against the definition in 64 bits."""
import pytest
import torch

from test_gpu_shared_prefix import BF16, F16, F32, make, run
from test_gpu_shared_prefix_accuracy import check_rounding, definition

pytestmark = pytest.mark.gpu


def range_tokens(q, pt, kp, length):
    """Tokens of the ranges that a prefix of `length` tokens is cut into, from the workspace
    that a call without own tokens needs: fp32 outputs and logsumexps of every range."""
    from llm_cuda import _native as nat

    B, Hq, D = q.shape[0], q.shape[1], q.shape[-1]
    need = nat.load().lc_shared_prefix_decode_workspace_bytes(
        B, pt.shape[0], Hq, kp.shape[1], D, pt.shape[1] * kp.shape[2], 0, nat.lc_dtype(q))
    ranges = [s for s in range(1, 65)
              if (B * Hq * s * D * 4 + 255) // 256 * 256 + B * Hq * s * 4 == need]
    assert len(ranges) == 1
    each = -(-length // ranges[0])
    return -(-each // 64) * 64


@pytest.mark.parametrize("dtype", [BF16, F32])  # (products of f16 values stay within fp32)
@pytest.mark.parametrize("W", [4, 10, 24])  # 16, 40, 96 rows of a prefix
def test_rows_without_a_score_keep_no_reference(cuda, W, dtype):
    """Odd heads have scores below any finite fp32 value in the first two tiles of every
    range, then ones far below 0; even heads' scores rise steeply in the second tile."""
    tiles, D = 4, 64
    length = 64 * 64 * tiles
    q, kp, vp, pt, pl, bt, sl = make(1, W, 4, 1, D, 64, [length], [0] * W, F32, seed=W)
    kp = kp.nan_to_num(0.0) * 0.1
    q *= 0.1
    q[..., :3] = 0
    q[:, 1::2, :, 0], q[:, 1::2, :, 1], q[:, ::2, :, 2] = -1e30, -64.0, 16.0
    in_range = torch.arange(length) // 64 % tiles
    keys = kp[pt[0].long()].view(length, D)
    keys[:, 0] = torch.where(in_range < 2, 1e30, 0.0)
    keys[:, 1] = torch.where(in_range >= 2, 32.0, 0.0)
    keys[:, 2] = torch.where(in_range >= 1, 8.0, 0.0)
    kp[pt[0].long()] = keys.view(-1, 1, 64, D)
    args = (q.to(dtype), kp.to(dtype), vp.nan_to_num(0.0).to(dtype), pt, pl, bt, sl)
    assert range_tokens(args[0], pt, kp, length) == 64 * tiles
    got = run(args, cuda)
    want, want_lse = definition(*args)
    assert ((got[1].double().cpu() - want_lse).abs() <= 1e-3 + 2e-6 * want_lse.abs()).all()
    # (scores of up to 2048 * 0.125: fp32 sums are off by 2^-24 of them, 3e-5)
    half = torch.finfo(dtype).eps / 2
    err = (got[0].double().cpu().reshape(want.shape) - want).abs()
    assert (err <= half * want.abs() + 1e-3 * vp.nan_to_num(0.0).abs().max()).all()


# beams of 4 heads (rows of a prefix: 40, 64: tiles of 64 rows; 72, 128, 136: of 128), then
# head_dim, type and tiles of a range
WIDTHS = [10, 16, 18, 32, 34]
FORMS = [(64, BF16, 3), (64, F16, 5), (72, BF16, 4), (72, F16, 3), (128, BF16, 5), (128, F16, 6), (64, BF16, 2),
         (128, BF16, 1)]


def tiled(W, D, dtype, tiles, P=64, seed=0):
    """One prompt whose ranges hold `tiles` tiles, the last one less, and short own tokens."""
    length = 64 * 64 * tiles - 100 if tiles > 1 else 64
    args = make(1, W, 4, 1, D, P, [length], [(7 * i) % 40 for i in range(W)], dtype, seed=seed)
    each = range_tokens(args[0], args[3], args[1], length)
    assert each == tiles * 64
    return args


@pytest.mark.parametrize("D,dtype,tiles", FORMS)
@pytest.mark.parametrize("W", WIDTHS)
def test_ranges_of_several_tiles(cuda, W, D, dtype, tiles):
    args = tiled(W, D, dtype, tiles, P=16 if W == 16 else 64, seed=W + tiles)
    check_rounding(args, run(args, cuda))


@pytest.mark.parametrize("D,dtype,tiles", FORMS[:-1])
@pytest.mark.parametrize("W", WIDTHS)
def test_scores_that_rise_in_every_tile(cuda, W, D, dtype, tiles):
    """By 8 nats a tile, 2^11.5 in the weights: the reference maximum has to move each time."""
    q, kp, vp, pt, pl, bt, sl = tiled(W, D, dtype, tiles)
    q = (torch.ones_like(q) + 0.1 * torch.randn(q.shape, generator=torch.Generator().manual_seed(W))).to(dtype)
    for i, page in enumerate(pt[0].tolist()):
        rise = 8.0 * (i % tiles) * D ** -0.5
        kp[page] = torch.where(kp[page].isnan(), kp[page], (kp[page] + rise).to(dtype))
    args = (q, kp, vp, pt, pl, bt, sl)
    check_rounding(args, run(args, cuda))


@pytest.mark.parametrize("P", [16, 64])
@pytest.mark.parametrize("D,dtype,tiles", FORMS[:-2])
@pytest.mark.parametrize("W", [10, 34])
def test_pages_outside_the_pool(cuda, W, D, dtype, tiles, P):
    """Entries outside the pool: a range's first tile, its last, a whole range, single pages."""
    args = tiled(W, D, dtype, tiles, P)
    pt, pages, per = args[3], args[1].shape[0], 64 // P
    for first, count in ((0, 1), (tiles - 1, 1), (tiles, tiles), (4 * tiles + 1, tiles - 1)):
        pt[0, first * per:(first + count) * per] = -1
    pt[0, 3::7 * per + 1] = pages
    pt[0, 5::11 * per + 2] = 2 ** 31 - 1
    check_rounding(args, run(args, cuda))
