"""Beam search without a GPU: refusals of the entry points, workspace sizes, and
the oracle against closed forms."""
import math

import pytest
import torch

from oracle import beam as oracle

I32, I64 = torch.int32, torch.int64


def attention_args(**kw):
    a = dict(q=torch.zeros(4, 4, 1, 16), key_pages=torch.zeros(6, 2, 8, 16),
             value_pages=torch.zeros(6, 2, 8, 16), prefix_table=torch.zeros(2, 1, dtype=I32),
             prefix_lens=torch.zeros(2, dtype=I32), block_table=torch.zeros(4, 1, dtype=I32),
             seq_lens=torch.zeros(4, dtype=I32))
    a.update(kw)
    return a


@pytest.mark.parametrize("change,error", [
    (dict(q=torch.zeros(4, 4, 2, 16)), ValueError),
    (dict(q=torch.zeros(4, 3, 1, 16)), ValueError),
    (dict(q=torch.zeros(4, 4, 1, 8)), ValueError),
    (dict(q=torch.zeros(4, 4, 1, 16, dtype=torch.float16)), TypeError),
    (dict(value_pages=torch.zeros(6, 2, 4, 16)), ValueError),
    (dict(key_pages=torch.zeros(6, 8, 16), value_pages=torch.zeros(6, 8, 16)), ValueError),
    (dict(prefix_table=torch.zeros(3, 1, dtype=I32), prefix_lens=torch.zeros(3, dtype=I32)), ValueError),
    (dict(prefix_table=torch.zeros(0, 1, dtype=I32), prefix_lens=torch.zeros(0, dtype=I32)), ValueError),
    (dict(prefix_lens=torch.zeros(1, dtype=I32)), ValueError),
    (dict(prefix_lens=torch.zeros(2, dtype=I64)), TypeError),
    (dict(prefix_table=torch.zeros(2, 1, dtype=I64)), TypeError),
    (dict(block_table=torch.zeros(3, 1, dtype=I32)), ValueError),
    (dict(block_table=torch.zeros(4, dtype=I32)), ValueError),
    (dict(seq_lens=torch.zeros(4, dtype=torch.float32)), TypeError),
    (dict(q=torch.zeros(4, 4, 1, 16, dtype=torch.float64), key_pages=torch.zeros(6, 2, 8, 16, dtype=torch.float64),
          value_pages=torch.zeros(6, 2, 8, 16, dtype=torch.float64)), TypeError),
    (dict(), RuntimeError),  # host tensors
])
def test_attention_refuses(change, error):
    from llm_cuda.kernels.triton.decode_attention import shared_prefix_decode_attention

    with pytest.raises(error):
        shared_prefix_decode_attention(**attention_args(**change))


@pytest.mark.parametrize("kw,error", [
    (dict(logits=torch.zeros(4, 10)), ValueError),
    (dict(scores=torch.zeros(2, 3)), ValueError),
    (dict(scores=torch.zeros(2, 4, dtype=torch.float64)), TypeError),
    (dict(num_candidates=0), ValueError),
    (dict(num_candidates=65), ValueError),
    (dict(logits=torch.zeros(2, 4, 2), num_candidates=9), ValueError),
    (dict(logits=torch.zeros(2, 0, 2), scores=torch.zeros(2, 0)), ValueError),
    (dict(logits=torch.zeros(1, 257, 2), scores=torch.zeros(1, 257), num_candidates=1), ValueError),
    (dict(logits=torch.zeros(1).expand(1, 256, 2 ** 23), scores=torch.zeros(1, 256), num_candidates=4), ValueError),
    (dict(finished=torch.zeros(2, 4, dtype=torch.bool)), ValueError),
    (dict(finished=torch.zeros(2, 4, dtype=torch.uint8), eos_token_id=1), TypeError),
    (dict(finished=torch.zeros(2, 3, dtype=torch.bool), eos_token_id=1), TypeError),
    (dict(finished=torch.zeros(2, 4, dtype=torch.bool), eos_token_id=10), ValueError),
    (dict(finished=torch.zeros(2, 4, dtype=torch.bool), eos_token_id=-1), ValueError),
    (dict(logits=torch.zeros(2, 4, 10, dtype=torch.float64)), TypeError),
    (dict(), RuntimeError),
])
def test_selection_refuses(kw, error):
    from llm_cuda.kernels.beam_search import beam_select

    args = dict(logits=torch.zeros(2, 4, 10), scores=torch.zeros(2, 4))
    args.update(kw)
    with pytest.raises(error):
        beam_select(**args)


@pytest.mark.parametrize("kw,error", [
    (dict(key_pages=torch.zeros(2, 8, 16)), ValueError),
    (dict(value_pages=torch.zeros(1, 9, 2, 8, 16)), ValueError),
    (dict(value_pages=torch.zeros(1, 8, 2, 8, 16, dtype=torch.float16)), TypeError),
    (dict(value_pages=torch.zeros(1, 8, 8, 2, 16).transpose(2, 3)), ValueError),
    (dict(key_pages=torch.zeros(1, 8, 2, 16, 8).transpose(3, 4), value_pages=torch.zeros(1, 8, 2, 16, 8).transpose(3, 4)), ValueError),
    (dict(key_pages=torch.zeros(1, 8, 2, 8, 16, requires_grad=True)), NotImplementedError),
    (dict(block_table=torch.zeros(4, 2, dtype=I64)), TypeError),
    (dict(seq_lens=torch.zeros(4, dtype=I64)), TypeError),
    (dict(seq_lens=torch.zeros(2, dtype=I32)), ValueError),
    (dict(parents=torch.zeros(2, 2, dtype=I32)), TypeError),
    (dict(parents=torch.zeros(4, dtype=I64)), TypeError),
    (dict(parents=torch.zeros(2, 3, dtype=I64)), ValueError),
    (dict(key_pages=torch.zeros(1, 1, 2, 8, 16).expand(1, 8, 2, 8, 16),
          value_pages=torch.zeros(1, 1, 2, 8, 16).expand(1, 8, 2, 8, 16)), ValueError),
    (dict(), RuntimeError),
])
def test_reordering_refuses(kw, error):
    from llm_cuda.kernels.beam_search import paged_kv_reorder

    args = dict(key_pages=torch.zeros(1, 8, 2, 8, 16), value_pages=torch.zeros(1, 8, 2, 8, 16),
                block_table=torch.zeros(4, 2, dtype=I32), seq_lens=torch.zeros(4, dtype=I32),
                parents=torch.zeros(2, 2, dtype=I64))
    args.update(kw)
    with pytest.raises(error):
        paged_kv_reorder(**args)


def test_arguments_rejected_before_launch():
    """Negative status and a message from the C entries; no launch, so no GPU needed."""
    from llm_cuda import _native

    lib = _native.load()
    buf = torch.zeros(1 << 16, dtype=torch.uint8)
    base = (buf.data_ptr() + 255) // 256 * 256

    def attend(B=4, N=2, Hq=4, Hkv=2, D=16, P=8, pages=6, ppages=1, pages_seq=1, ws=1 << 15, dtype=0,
               pt_stride=1, wp=base, cnt=None):
        return lib.lc_shared_prefix_decode_fwd(
            base, 64, 16, base, base, 256, 128, 16, pages, base, pt_stride, ppages, base, base, 1,
            pages_seq, base, base, 64, 16, None, wp, ws, cnt, B, N, Hq, Hkv, D, P, 0.25, dtype, None)

    for bad in (dict(B=5), dict(N=0), dict(B=-1), dict(B=65536), dict(Hq=3), dict(D=0), dict(D=257),
                dict(P=0), dict(pages=0), dict(ppages=-1), dict(pt_stride=0), dict(ws=8), dict(dtype=7),
                dict(ppages=1 << 30, pt_stride=1 << 30), dict(wp=base + 4), dict(wp=None), dict(cnt=base + 2)):
        assert attend(**bad) < 0, bad
        assert b"lc_shared_prefix_decode_fwd" in lib.lc_last_error()
    assert attend(B=0, N=0) == 0 and attend(B=0) == 0

    def select(groups=2, W=4, V=10, K=4, fin=None, eos=0, ws=1 << 15, dtype=0, wp=base, cnt=None):
        return lib.lc_beam_select(base, 40, 10, base, fin, eos, groups, W, V, K, base, base, base, None,
                                  wp, ws, cnt, dtype, None)

    for bad in (dict(groups=-1), dict(W=0), dict(W=257), dict(V=0), dict(W=256, V=1 << 23), dict(K=0),
                dict(K=65), dict(W=1, V=2, K=3), dict(fin=base, eos=10), dict(fin=base, eos=-1),
                dict(ws=100), dict(dtype=3), dict(wp=base + 16), dict(wp=None), dict(cnt=base + 1)):
        assert select(**bad) < 0, bad
        assert b"lc_beam_select" in lib.lc_last_error()
    assert select(groups=0) == 0

    def reorder(L=1, pages=8, M=2, N=2, W=2, H=2, D=16, P=8, dtype=0, out=base + 4096, stride=2):
        return lib.lc_paged_kv_reorder(base, base, 2048, 256, 128, 16, L, pages, base, stride, out, stride,
                                       M, base, base, N, W, H, D, P, dtype, None)

    for bad in (dict(L=-1), dict(L=40000), dict(pages=-1), dict(M=-1), dict(N=-1), dict(W=0), dict(W=257),
                dict(H=0), dict(D=0), dict(P=0), dict(dtype=9), dict(out=base), dict(out=base + 12),
                dict(stride=1), dict(M=1 << 30, stride=1 << 30), dict(out=None)):
        assert reorder(**bad) < 0, bad
        assert b"lc_paged_kv_reorder" in lib.lc_last_error()
    assert reorder(N=0) == 0 and reorder(M=0) == 0


def test_workspace_sizes():
    from llm_cuda import _native

    lib = _native.load()
    assert lib.lc_shared_prefix_decode_workspace_bytes(4, 3, 4, 2, 16, 8, 8, 0) == -1
    assert lib.lc_shared_prefix_decode_workspace_bytes(4, 2, 4, 3, 16, 8, 8, 0) == -1
    assert lib.lc_shared_prefix_decode_workspace_bytes(0, 2, 4, 2, 16, 8, 8, 0) == 0
    # both parts present: at least one range each of fp32 output and logsumexp per row
    assert lib.lc_shared_prefix_decode_workspace_bytes(4, 2, 4, 2, 16, 8, 8, 0) >= 4 * 4 * 2 * (16 + 1) * 4
    assert lib.lc_beam_select_workspace_bytes(1, 4, 0, 4) == -1
    assert lib.lc_beam_select_workspace_bytes(0, 4, 10, 4) == 0


def test_empty_batches_launch_nothing():
    """No sequence, no group: shapes only (checked before any device question)."""
    lib_free = torch.zeros(0, 4, 10)
    from llm_cuda.kernels.beam_search import beam_select

    with pytest.raises(RuntimeError):  # host tensors are refused all the same
        beam_select(lib_free, torch.zeros(0, 4))


def test_oracle_selection_by_hand():
    x = torch.log(torch.tensor([[[0.5, 0.25, 0.25], [0.1, 0.6, 0.3]]]))
    s = torch.log(torch.tensor([[0.2, 0.8]]))
    best, tok, par, _ = oracle.beam_select(x, s, 4)
    # 0.8 * (0.1, 0.6, 0.3) = 0.08, 0.48, 0.24; 0.2 * (0.5, 0.25, 0.25) = 0.1, 0.05, 0.05
    assert tok.tolist() == [[1, 2, 0, 0]] and par.tolist() == [[1, 1, 0, 1]]
    assert torch.allclose(best.exp(), torch.tensor([[0.48, 0.24, 0.1, 0.08]], dtype=torch.float64))
    done = torch.tensor([[True, False]])
    best, tok, par, fin = oracle.beam_select(x, s, 4, done, 2)
    assert par.tolist() == [[1, 1, 0, 1]] and tok.tolist() == [[1, 2, 2, 0]]
    assert fin.tolist() == [[False, True, True, False]]


def test_oracle_selection_special_rows():
    x = torch.zeros(1, 3, 4)
    x[0, 0] = -math.inf
    x[0, 1, 2] = math.nan
    best, tok, par, _ = oracle.beam_select(x, torch.zeros(1, 3), 9)
    assert par.tolist() == [[1, 1, 1, 1, 2, 2, 2, 2, 0]] and tok.tolist() == [[0, 1, 2, 3, 0, 1, 2, 3, 0]]
    assert best[0, :4].isnan().all() and best[0, 8] == -math.inf


def test_oracle_attention_is_one_softmax():
    """The union of prefix and own tokens equals plain attention over their concatenation."""
    g = torch.Generator().manual_seed(0)
    kp, vp = torch.randn(5, 1, 4, 8, generator=g), torch.randn(5, 1, 4, 8, generator=g)
    q = torch.randn(2, 2, 1, 8, generator=g)
    out, lse = oracle.shared_prefix_decode(
        q, kp, vp, torch.tensor([[2, 0]], dtype=I32), torch.tensor([6], dtype=I32),
        torch.tensor([[1], [4]], dtype=I32), torch.tensor([3, 0], dtype=I32))
    k = torch.cat([kp[2, 0], kp[0, 0, :2], kp[1, 0, :3]]).double()
    v = torch.cat([vp[2, 0], vp[0, 0, :2], vp[1, 0, :3]]).double()
    p = torch.softmax(q[0, 1, 0].double() @ k.T / 8 ** 0.5, -1)
    assert torch.allclose(out[0, 1], p @ v)
    p = torch.softmax(q[1, 0, 0].double() @ k[:6].T / 8 ** 0.5, -1)
    assert torch.allclose(out[1, 0], p @ v[:6])
    assert torch.allclose(lse[1, 0], torch.logsumexp(q[1, 0, 0].double() @ k[:6].T / 8 ** 0.5, -1))


def test_oracle_reordering_by_hand():
    kp = torch.arange(6.0).view(1, 6, 1, 1, 1).expand(1, 6, 1, 2, 1).clone()
    table = torch.tensor([[0, 3], [1, 4], [2, 5]], dtype=I32)
    k, _, t = oracle.kv_reorder(kp, kp.clone(), table, torch.full((3,), 3, dtype=I32), torch.tensor([[2, 2, 0]]))
    # beam 0 is 2's first child, beam 1 its second (takes childless 1's page), beam 2 continues 0
    assert t.tolist() == [[2, 5], [2, 4], [0, 3]]
    assert k[0, 4, 0].flatten().tolist() == [5.0, 4.0] and k[0, 3, 0].flatten().tolist() == [3.0, 3.0]
