"""Speculative decoding without a GPU: refusals of the entry points, workspace sizes, and
the oracle against closed forms."""
import math

import pytest
import torch

from oracle import speculative as oracle
from oracle.attention import causal_attention

I32, I64 = torch.int32, torch.int64


def extend_args(**kw):
    a = dict(q=torch.zeros(3, 4, 2, 16), key_pages=torch.zeros(6, 2, 8, 16),
             value_pages=torch.zeros(6, 2, 8, 16), block_table=torch.zeros(3, 2, dtype=I32),
             seq_lens=torch.zeros(3, dtype=I32))
    a.update(kw)
    return a


@pytest.mark.parametrize("change,error", [
    (dict(q=torch.zeros(3, 4, 16)), ValueError),
    (dict(q=torch.zeros(3, 3, 2, 16)), ValueError),
    (dict(q=torch.zeros(3, 0, 2, 16)), ValueError),
    (dict(q=torch.zeros(3, 4, 2, 8)), ValueError),
    (dict(q=torch.zeros(3, 4, 2, 16, dtype=torch.float16)), TypeError),
    (dict(value_pages=torch.zeros(6, 2, 4, 16)), ValueError),
    (dict(key_pages=torch.zeros(6, 8, 16), value_pages=torch.zeros(6, 8, 16)), ValueError),
    (dict(block_table=torch.zeros(2, 2, dtype=I32)), ValueError),
    (dict(block_table=torch.zeros(3, dtype=I32)), ValueError),
    (dict(block_table=torch.zeros(3, 2, dtype=I64)), TypeError),
    (dict(seq_lens=torch.zeros(2, dtype=I32)), ValueError),
    (dict(seq_lens=torch.zeros(3)), TypeError),
    (dict(query_lens=torch.zeros(2, dtype=I32)), ValueError),
    (dict(query_lens=torch.zeros(3, dtype=I64)), TypeError),
    (dict(q=torch.zeros(3, 4, 2, 16, dtype=torch.float64), key_pages=torch.zeros(6, 2, 8, 16, dtype=torch.float64),
          value_pages=torch.zeros(6, 2, 8, 16, dtype=torch.float64)), TypeError),
    (dict(), RuntimeError),  # host tensors
])
def test_extend_refuses(change, error):
    from llm_cuda.kernels.triton.decode_attention import paged_extend_attention

    with pytest.raises(error):
        paged_extend_attention(**extend_args(**change))


@pytest.mark.parametrize("kw,error", [
    (dict(logits=torch.zeros(2, 10)), ValueError),
    (dict(logits=torch.zeros(2, 3, 10)), ValueError),
    (dict(logits=torch.zeros(2, 4, 0)), ValueError),
    (dict(logits=torch.zeros(2, 0, 10), draft_tokens=torch.zeros(2, 0, dtype=I64), uniforms=torch.zeros(2, 0)), ValueError),
    (dict(logits=torch.zeros(2, 4, 10, dtype=torch.float64)), TypeError),
    (dict(draft_tokens=torch.zeros(2, 3, dtype=I32)), TypeError),
    (dict(draft_tokens=torch.zeros(2, 4, dtype=I64)), ValueError),
    (dict(uniforms=torch.zeros(2, 3)), ValueError),
    (dict(uniforms=torch.zeros(2, 4, dtype=torch.float64)), TypeError),
    (dict(draft_logits=torch.zeros(2, 4, 10)), ValueError),
    (dict(draft_logits=torch.zeros(2, 3, 10, dtype=torch.float16)), TypeError),
    (dict(draft_lens=torch.zeros(3, dtype=I32)), ValueError),
    (dict(draft_lens=torch.zeros(2, dtype=I64)), TypeError),
    (dict(temperature=torch.ones(3)), ValueError),
    (dict(temperature=torch.ones(2, dtype=torch.float64)), TypeError),
    (dict(), RuntimeError),
])
def test_verification_refuses(kw, error):
    from llm_cuda.kernels.speculative import verify_draft_tokens

    args = dict(logits=torch.zeros(2, 4, 10), draft_tokens=torch.zeros(2, 3, dtype=I64),
                uniforms=torch.zeros(2, 4))
    args.update(kw)
    with pytest.raises(error):
        verify_draft_tokens(**args)


POOL_ERRORS = [
    (dict(key_pages=torch.zeros(2, 8, 16)), ValueError),
    (dict(value_pages=torch.zeros(1, 9, 2, 8, 16)), ValueError),
    (dict(value_pages=torch.zeros(1, 8, 2, 8, 16, dtype=torch.float16)), TypeError),
    (dict(value_pages=torch.zeros(1, 8, 8, 2, 16).transpose(2, 3)), ValueError),
    (dict(key_pages=torch.zeros(1, 8, 2, 16, 8).transpose(3, 4), value_pages=torch.zeros(1, 8, 2, 16, 8).transpose(3, 4)), ValueError),
    (dict(key_pages=torch.zeros(1, 8, 2, 8, 16, requires_grad=True)), NotImplementedError),
    (dict(key_pages=torch.zeros(1, 1, 2, 8, 16).expand(3, 8, 2, 8, 16),
          value_pages=torch.zeros(1, 1, 2, 8, 16).expand(3, 8, 2, 8, 16)), ValueError),
    (dict(block_table=torch.zeros(4, 2, dtype=I64)), TypeError),
    (dict(block_table=torch.zeros(3, 2, dtype=I32)), ValueError),
    (dict(seq_lens=torch.zeros(4, dtype=I64)), TypeError),
    (dict(seq_lens=torch.zeros(2, dtype=I32)), ValueError),
    (dict(page_refs=torch.zeros(8, dtype=I64)), TypeError),
    (dict(page_refs=torch.zeros(7, dtype=I32)), ValueError),
    (dict(), RuntimeError),
]


def pool_args(**kw):
    a = dict(key_pages=torch.zeros(1, 8, 2, 8, 16), value_pages=torch.zeros(1, 8, 2, 8, 16),
             block_table=torch.zeros(4, 2, dtype=I32), seq_lens=torch.zeros(4, dtype=I32),
             page_refs=torch.zeros(8, dtype=I32))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,error", POOL_ERRORS + [
    (dict(new_lens=torch.zeros(4, dtype=I64)), TypeError), (dict(new_lens=torch.zeros(3, dtype=I32)), ValueError)])
def test_resize_refuses(kw, error):
    from llm_cuda.kernels.page_pool import paged_kv_resize

    with pytest.raises(error):
        paged_kv_resize(**pool_args(**{"new_lens": torch.zeros(4, dtype=I32), **kw}))


@pytest.mark.parametrize("kw,error", POOL_ERRORS + [
    (dict(parents=torch.zeros(4, dtype=I32)), TypeError), (dict(parents=torch.zeros(2, 2, dtype=I64)), TypeError)])
def test_fork_refuses(kw, error):
    from llm_cuda.kernels.page_pool import paged_kv_fork

    with pytest.raises(error):
        paged_kv_fork(**pool_args(**{"parents": torch.zeros(4, dtype=I64), **kw}))


@pytest.mark.parametrize("kw,error", POOL_ERRORS)
def test_compact_refuses(kw, error):
    from llm_cuda.kernels.page_pool import paged_kv_compact

    with pytest.raises(error):
        paged_kv_compact(**pool_args(**kw))


def test_arguments_rejected_before_launch():
    """Negative status and a message from the C entries; no launch, so no GPU needed."""
    from llm_cuda import _native

    lib = _native.load()
    buf = torch.zeros(1 << 16, dtype=torch.uint8)
    base = (buf.data_ptr() + 255) // 256 * 256

    def extend(B=2, T=3, Hq=4, Hkv=2, D=16, P=8, pages=6, M=1, ts=1, ws=1 << 15, wp=base, dtype=0, q=base, qs=64):
        return lib.lc_paged_extend_fwd(q, qs, 16, 16, base, base, 256, 128, 16, pages, base, ts, M, base, None,
                                       base, 64, 16, 16, None, wp, ws, B, T, Hq, Hkv, D, P, 0.25, dtype, None)

    for bad in (dict(B=-1), dict(B=65536), dict(T=-1), dict(T=1 << 20), dict(Hq=3), dict(D=0), dict(D=257), dict(P=0),
                dict(pages=0), dict(M=-1), dict(ts=0), dict(M=1 << 30, ts=1 << 30), dict(ws=8), dict(wp=base + 4),
                dict(wp=None), dict(dtype=7), dict(q=None), dict(qs=-1), dict(B=60000, T=1 << 19)):
        assert extend(**bad) < 0, bad
        assert b"lc_paged_extend_fwd" in lib.lc_last_error()
    assert extend(B=0) == 0 and extend(T=0) == 0

    def verify(B=2, K=3, V=10, dtype=0, ws=1 << 15, wp=base, x=base, u=base, xs=40, d=base):
        return lib.lc_verify_draft_tokens(x, xs, 10, None, 0, 0, d, u, None, None, 1.0, B, K, V, base, base, wp, ws,
                                          dtype, None)

    for bad in (dict(B=-1), dict(K=-1), dict(K=256), dict(V=0), dict(V=1 << 31), dict(dtype=7), dict(ws=8),
                dict(wp=base + 4), dict(wp=None), dict(x=None), dict(u=None), dict(xs=-1), dict(d=None),
                dict(B=1 << 24)):
        assert verify(**bad) < 0, bad
        assert b"lc_verify_draft_tokens" in lib.lc_last_error()
    assert verify(B=0) == 0

    def resize(B=4, L=1, N=8, M=2, ts=2, Hkv=2, D=16, P=8, dtype=0, ws=1 << 15, wp=base, kp=base, refs=base,
               out_refs=base + 64, table=base, out=base + 4096, lens=base, missing=base, sp=256):
        return lib.lc_paged_kv_resize(kp, base, 2048, sp, 128, 16, L, N, table, ts, M, lens, lens, refs, out,
                                      out_refs, missing, wp, ws, B, Hkv, D, P, dtype, None)

    def fork(B=4, R=4, L=1, N=8, M=2, ts=2, wp=base, ws=1 << 15, parents=base, out=base + 4096, out_refs=base + 64):
        return lib.lc_paged_kv_fork(base, base, 2048, 256, 128, 16, L, N, base, ts, M, base, parents, base, out, base,
                                    out_refs, base, wp, ws, B, R, 2, 16, 8, 0, None)

    def compact(B=4, N=8, M=2, ts=2, wp=base, ws=1 << 15, page_map=base, out=base + 4096, out_refs=base + 64):
        return lib.lc_paged_kv_compact(base, base, 2048, 256, 128, 16, 1, N, base, ts, M, base, base, out, out_refs,
                                       page_map, wp, ws, B, 2, 16, 8, 0, None)

    for bad in (dict(B=-1), dict(B=1 << 20), dict(L=-1), dict(L=32768), dict(N=-1), dict(N=1 << 31), dict(M=-1),
                dict(ts=1), dict(Hkv=0), dict(D=0), dict(P=0), dict(M=1 << 28, ts=1 << 28), dict(dtype=3), dict(ws=8),
                dict(wp=base + 4), dict(wp=None), dict(kp=None), dict(refs=None), dict(out_refs=base), dict(table=None),
                dict(out=base), dict(lens=None), dict(missing=None), dict(sp=-1), dict(D=1 << 25)):
        assert resize(**bad) < 0, bad
        assert b"lc_paged_kv_resize" in lib.lc_last_error()
    for bad in (dict(R=-1), dict(R=1 << 20), dict(M=0, ts=0), dict(parents=None), dict(wp=None), dict(ws=8),
                dict(out=base), dict(out_refs=base)):
        assert fork(**bad) < 0, bad
    for bad in (dict(page_map=None), dict(wp=None), dict(ws=8), dict(out=base), dict(out_refs=base), dict(ts=1)):
        assert compact(**bad) < 0, bad


def test_workspace_sizes():
    from llm_cuda import _native

    lib = _native.load()
    assert lib.lc_paged_extend_workspace_bytes(2, 3, 5, 2, 16, 64, 0) == -1
    assert lib.lc_paged_extend_workspace_bytes(-1, 3, 4, 2, 16, 64, 0) == -1
    assert lib.lc_verify_draft_tokens_workspace_bytes(2, 3, 0) == -1
    assert lib.lc_verify_draft_tokens_workspace_bytes(2, -1, 5) == -1
    assert lib.lc_verify_draft_tokens_workspace_bytes(2, 3, 5000) > 0
    assert lib.lc_paged_kv_resize_workspace_bytes(-1, 2, 3) == -1
    assert lib.lc_paged_kv_fork_workspace_bytes(2, -1, 3) == -1
    assert lib.lc_paged_kv_compact_workspace_bytes(-1) == -1
    # the lists hold what a call can hand out: never more than the pool
    assert lib.lc_paged_kv_resize_workspace_bytes(1000, 1000, 16) < 64 << 10


def test_oracle_extend_is_causal_attention():
    """The newest tokens' rows are the last rows of a causal attention."""
    g = torch.Generator().manual_seed(0)
    L, T, Hq, Hkv, D, P = 21, 4, 4, 2, 16, 8
    k, v = (torch.randn(1, Hkv, L, D, generator=g) for _ in range(2))
    q = torch.randn(1, Hq, L, D, generator=g)
    table = torch.tensor([[4, 0, 2]], dtype=I32)
    kp, vp = torch.zeros(5, Hkv, P, D), torch.zeros(5, Hkv, P, D)
    for t in range(L):
        kp[table[0, t // P], :, t % P], vp[table[0, t // P], :, t % P] = k[0, :, t], v[0, :, t]
    out, lse, size = oracle.paged_extend(q[:, :, -T:], kp, vp, table, torch.tensor([L]))
    ref = causal_attention(q, k, v)
    ref = ref[0] if isinstance(ref, tuple) else ref
    assert (out - ref[:, :, -T:]).abs().max() < 1e-5 and (size >= out.abs() - 1e-12).all()
    assert torch.isfinite(lse).all()


def test_oracle_verification_of_known_numbers():
    """Two tokens: p = (3/4, 1/4), q = (1/4, 3/4); draft 1 stands for u < 1/3, else the residual
    is all on token 0."""
    x = torch.log(torch.tensor([[[0.75, 0.25], [0.5, 0.5]]]))
    y = torch.log(torch.tensor([[[0.25, 0.75]]]))
    d = torch.tensor([[1]])
    tokens, accepted, _, _ = oracle.verify_draft(x, d, torch.tensor([[0.33, 0.6]]), y)
    assert accepted.tolist() == [1] and tokens.tolist() == [[1, 1]]
    tokens, accepted, _, _ = oracle.verify_draft(x, d, torch.tensor([[0.34, 0.99]]), y)
    assert accepted.tolist() == [0] and tokens.tolist() == [[0, -1]]
    tokens, accepted, _, _ = oracle.verify_draft(x, d, torch.tensor([[0.24, 0.4]]))
    assert accepted.tolist() == [1] and tokens.tolist() == [[1, 0]]
    assert oracle.distribution(torch.tensor([1.0, math.nan, math.inf]), 1.0).tolist() == [0, 1, 0]
    assert oracle.distribution(torch.tensor([-math.inf] * 3), 1.0).tolist() == [1, 0, 0]


def test_oracle_pool_keeps_its_counts():
    """Growing, forking and compaction leave the counts those of the table."""
    P, N = 4, 12
    kp = torch.arange(N).float().view(1, N, 1, 1, 1).expand(1, N, 1, P, 2).contiguous()
    table = torch.full((2, 4), -1, dtype=I32)
    table[0, :2] = torch.tensor([7, 3])
    table[1, :1] = 11
    lens, refs = torch.tensor([6, 4], dtype=I32), torch.zeros(N, dtype=I32)
    refs[[7, 3, 11]] = 1
    t, n, r, missing, kp2, _ = oracle.kv_fork(kp, kp, table, lens, torch.tensor([0, 0, 1]), refs)
    assert t.tolist() == [[7, 3, -1, -1], [7, 0, -1, -1], [11, -1, -1, -1]] and n.tolist() == [6, 6, 4]
    assert r.tolist() == [1, 0, 0, 1, 0, 0, 0, 2, 0, 0, 0, 1] and int(missing) == 0
    assert kp2[0, 0, 0, :, 0].tolist() == [3, 3, 0, 0]  # two slots of page 3
    t2, r2, missing, _, _ = oracle.kv_resize(kp2, kp2, t, n, torch.tensor([4, 9, 5], dtype=I32), r)
    assert t2.tolist() == [[7, -1, -1, -1], [7, 0, 1, -1], [11, 2, -1, -1]]
    assert r2.tolist() == [1, 1, 1, 0, 0, 0, 0, 2, 0, 0, 0, 1]
    t3, r3, where, kp4, _ = oracle.kv_compact(kp2, kp2, t2, torch.tensor([4, 9, 5]), r2)
    assert where.tolist() == [0, 1, 2, -1, -1, -1, -1, 3, -1, -1, -1, 4]
    assert t3.tolist() == [[3, -1, -1, -1], [3, 0, 1, -1], [4, 2, -1, -1]] and r3.tolist()[:6] == [1, 1, 1, 2, 1, 0]
    assert kp4[0, 3, 0, 0, 0] == 7 and kp4[0, 4, 0, 0, 0] == 11
