"""The operators of speculative decoding at large sizes: chunks of hundreds of tokens, hundreds
of sequences, and data past 2^31 elements and 4 GiB (tensors of which little is written)."""
import math

import pytest
import torch

from oracle import speculative as oracle
from test_gpu_paged_extend import check, make, run
from test_gpu_verify_draft import make as make_verify, on

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
I32 = torch.int32


def dense(args):
    """The oracle's three results with one matrix product per sequence."""
    q, kp, vp = args["q"], args["key_pages"], args["value_pages"]
    B, Hq, T, D = q.shape
    P, Hkv = kp.shape[2], kp.shape[1]
    out, lse, size = (torch.zeros(B, Hq, T, D, dtype=torch.float64), torch.full((B, Hq, T), -math.inf).double(),
                      torch.zeros(B, Hq, T, D, dtype=torch.float64))
    for b in range(B):
        L = int(args["seq_lens"][b])
        n = T if args["query_lens"] is None else int(args["query_lens"][b])
        at = torch.arange(L)
        page = args["block_table"][b, at // P].long()
        k = kp[page, :, at % P].double().permute(1, 0, 2)
        v = vp[page, :, at % P].double().permute(1, 0, 2)
        x = q[b, :, :n].double().reshape(Hkv, -1, D) @ k.transpose(1, 2).contiguous() / math.sqrt(D)
        x = x.view(Hq, n, L).masked_fill(at.view(1, L) > (L - n + torch.arange(n)).view(n, 1), -math.inf)
        p = torch.softmax(x, -1).view(Hkv, -1, L)
        out[b, :, :n], size[b, :, :n] = (p @ v).view(Hq, n, D), (p @ v.abs()).view(Hq, n, D)
        lse[b, :, :n] = torch.logsumexp(x, -1)
    return out, lse, size


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T,lens,Hq,Hkv,D", [(640, [1500, 640], 8, 2, 128), (333, [333, 900, 2000], 4, 1, 64),
                                             (129, [4000], 16, 2, 128)])
def test_chunks(cuda, T, lens, Hq, Hkv, D, dtype):
    args = make(lens, T, Hq, Hkv, D, 32, dtype, queries=[T - 7 * i for i in range(len(lens))], seed=T)
    check(args, run(args, cuda), want=dense(args))


@pytest.mark.parametrize("B,T,top", [(300, 3, 60), (160, 5, 300), (260, 1, 700)])
def test_many_sequences(cuda, B, T, top):
    lens = torch.randint(T, top, (B,), generator=torch.Generator().manual_seed(B)).tolist()
    args = make(lens, T, 8, 2, 64, 16, BF16, seed=B)
    check(args, run(args, cuda), want=dense(args))


@pytest.mark.parametrize("dtype,T", [(BF16, 5), (BF16, 40), (F32, 3)])
def test_pages_past_4_gib(cuda, dtype, T):
    from llm_cuda.kernels.triton.decode_attention import paged_extend_attention

    small = make([70, 200], T, 8, 2, 64, 16, dtype, seed=3)
    n, pages = small["key_pages"].shape[0], 2 ** 31 // (2 * 16 * 64) + 1000
    big = [torch.empty(pages, 2, 16, 64, dtype=dtype, device=cuda) for _ in range(2)]
    at = pages - 1 - torch.arange(n)
    for to, name in zip(big, ("key_pages", "value_pages")):
        to[at.to(cuda)] = small[name].to(cuda)
    table = torch.where(small["block_table"] >= 0, at[small["block_table"].clamp(min=0).long()].to(I32), -1)
    out = paged_extend_attention(small["q"].to(cuda), *big, table.to(cuda), small["seq_lens"].to(cuda), return_lse=True)
    torch.cuda.synchronize()
    check(small, out)


def test_copies_past_4_gib(cuda):
    """Two layers of 2.1 billion elements each; pages copied from the end to the front."""
    from llm_cuda.kernels.page_pool import paged_kv_compact, paged_kv_fork

    P, D = 16, 64
    N = 2 ** 31 // (P * D) + 500
    pools = [torch.empty(2, N, 1, P, D, dtype=BF16, device=cuda) for _ in range(2)]
    used = torch.tensor([N - 1, N - 7, N - 300, 5], device=cuda)
    for i, pool in enumerate(pools):
        pool[:, used] = torch.randn(2, 4, 1, P, D, device=cuda, generator=torch.Generator(cuda).manual_seed(i)).to(BF16)
    was = [pool[:, used].clone() for pool in pools]
    refs = torch.zeros(N, dtype=I32, device=cuda)
    refs[used] = 1
    table = used.to(I32).view(2, 2)
    lens = torch.tensor([2 * P, P + 3], dtype=I32, device=cuda)
    t, r, page_map = paged_kv_compact(*pools, table, lens, refs)
    # (4 in use: 5, N - 300, N - 7, N - 1 in order into 0 to 3)
    where = page_map[used].long()
    assert where.tolist() == [3, 2, 1, 0]
    assert torch.equal(t.view(-1).long(), where)
    for pool, old in zip(pools, was):
        assert torch.equal(pool[:, where], old)
    refs[[0, 1, 2, 3]] = 1
    t, l, r, missing = paged_kv_fork(*pools, table, lens, torch.tensor([1, 1], device=cuda), refs)
    assert int(missing) == 0 and l.tolist() == [P + 3, P + 3] and t[0].tolist() == table[1].tolist()
    assert t[1, 0] == table[1, 0] and t[1, 1] == 4
    for pool, old in zip(pools, was):
        assert torch.equal(pool[:, 4, :, :3], old[:, 3, :, :3])


def test_logits_past_2_31_elements(cuda):
    from llm_cuda.kernels.speculative import verify_draft_tokens

    args = make_verify(2, 2, 3001, BF16, 5)
    want = oracle.verify_draft(**args)
    assert want[2] > 4e-6 and want[3] > 1e-11
    args = on(cuda, args)
    far = 2 ** 31 + 8
    buf = torch.empty(far + 2 ** 20, dtype=BF16, device=cuda)
    x = buf.as_strided((2, 3, 3001), (far, 3001, 1))
    y = buf.as_strided((2, 2, 3001), (far, 3001, 1), 2 ** 19)
    x.copy_(args["logits"])
    y.copy_(args["draft_logits"])
    tokens, accepted = verify_draft_tokens(**dict(args, logits=x, draft_logits=y))
    torch.cuda.synchronize()
    assert torch.equal(tokens.cpu(), want[0]) and torch.equal(accepted.cpu(), want[1])
