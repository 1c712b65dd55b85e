"""Resizing, forking and compaction of a page pool against the oracle: everything is equal,
the pools' contents bit for bit."""
import pytest
import torch

from oracle import speculative as oracle

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
I32, I64 = torch.int32, torch.int64


def make(lens, P, dtype=BF16, layers=2, Hkv=2, D=16, spare=6, width=None, share=0, twins=(), seed=0):
    """Rows on shuffled pages; every odd row shares the first `share` whole pages of the row
    before it, and the rows in `twins` all of its pages (their lengths are equal)."""
    g = torch.Generator().manual_seed(seed)
    held = [-(-n // P) for n in lens]
    M = (max(held + [0]) + 2) if width is None else width
    table = torch.full((len(lens), M), -1, dtype=I64)
    used = 0
    for b, h in enumerate(held):
        s = 0
        if b in twins:
            s = h
        elif b % 2:
            s = min(share, lens[b] // P, lens[b - 1] // P)
        table[b, :s] = table[b - 1, :s]
        table[b, s:h] = torch.arange(used, used + h - s)
        used += h - s
    N = used + spare
    order = torch.randperm(N, generator=g)
    refs = torch.bincount(order[table[table >= 0]], minlength=N).to(I32)
    # entries that are not held say anything
    table = torch.where(table >= 0, order[table.clamp(min=0)] if N else table,
                        torch.randint(-3, N + 3, table.shape, generator=g)).to(I32)
    shape = (layers, N, Hkv, P, D)
    return dict(key_pages=torch.randn(shape, generator=g).to(dtype),
                value_pages=torch.randn(shape, generator=g).to(dtype), block_table=table,
                seq_lens=torch.tensor(lens, dtype=I32), page_refs=refs)


def on(dev, args):
    return {k: t.to(dev) for k, t in args.items()}


def same(got, want, names):
    torch.cuda.synchronize()
    for g, w, name in zip(got, want, names):
        if g.is_floating_point():
            view = torch.int32 if g.dtype == F32 else torch.int16
            assert torch.equal(g.cpu().view(view), w.view(view)), name
        else:
            assert g.dtype == w.dtype and torch.equal(g.cpu(), w), name


def check(op, args, dev):
    from llm_cuda.kernels import page_pool

    want = {"resize": oracle.kv_resize, "fork": oracle.kv_fork, "compact": oracle.kv_compact}[op](**args)
    given = on(dev, args)
    before = {k: given[k].clone() for k in given if not k.endswith("pages")}
    got = {"resize": page_pool.paged_kv_resize, "fork": page_pool.paged_kv_fork,
           "compact": page_pool.paged_kv_compact}[op](**given)
    names = {"resize": ("table", "refs", "missing"), "fork": ("table", "lens", "refs", "missing"),
             "compact": ("table", "refs", "map")}[op]
    same((*got, given["key_pages"], given["value_pages"]), want, (*names, "keys", "values"))
    assert all(torch.equal(given[k], t) for k, t in before.items()), "inputs"
    return got


def consistent(table, lens, refs, P):
    """The counts are those of the table's held entries."""
    N = refs.shape[0]
    held = torch.arange(table.shape[1]) < ((lens.cpu() + P - 1) // P).unsqueeze(1)
    named = table.cpu()[held].long()
    assert torch.equal(torch.bincount(named, minlength=N).to(I32), refs.cpu())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("P,D", [(16, 64), (1, 8), (5, 24), (64, 128), (8, 3)])
def test_resize(cuda, P, D, dtype):
    lens = [0, 1, P, P + 1, 3 * P - 1, 2 * P, 40, 41]
    args = make(lens, P, dtype, D=D, spare=60, share=2, seed=P)
    for change in (1, 5, P, 2 * P + 1, -1, -P, -1000):
        now = torch.tensor([max(0, n + change) for n in lens], dtype=I32)
        table, refs, missing = check("resize", dict(args, new_lens=now), cuda)
        cut = now.clamp(max=table.shape[1] * P)
        consistent(table, cut, refs, P)
        assert int(missing) == 0


def test_resize_up_and_down_at_once(cuda):
    args = make([10, 50, 0, 33, 64, 17, 17, 5], 16, share=1, spare=9, seed=1)
    args["new_lens"] = torch.tensor([11, 3, 40, 33, 0, 64, -5, 2 ** 31 - 1], dtype=I32)
    check("resize", args, cuda)


@pytest.mark.parametrize("dtype,D", [(BF16, 32), (F32, 5)])
def test_resize_copies_a_shared_page_before_it_is_written(cuda, dtype, D):
    lens = [30, 30, 30, 48, 48, 7, 7, 1, 1]
    args = make(lens, 16, dtype, D=D, spare=20, twins=(1, 2, 4, 6, 8), seed=2)
    for now in ([31] * 3 + [49] * 2 + [8, 7, 2, 2], [30] * 3 + [48, 49, 7, 40, 0, 1], [16] * 3 + [48] * 2 + [9] * 4):
        table, refs, _ = check("resize", dict(args, new_lens=torch.tensor(now, dtype=I32)), cuda)
        consistent(table, torch.tensor(now), refs, 16)


@pytest.mark.parametrize("spare", [0, 1, 3, 7])
def test_resize_without_enough_pages(cuda, spare):
    lens = [20, 20, 9, 0]
    args = make(lens, 8, twins=(1,), spare=spare, seed=3)
    args["new_lens"] = torch.tensor([30, 22, 17, 10], dtype=I32)  # 1 + 1, 1, 1, 2
    _, _, missing = check("resize", args, cuda)
    assert int(missing) == max(0, 6 - spare)


def test_negative_counts_are_not_free(cuda):
    args = make([5, 9], 8, spare=8, seed=4)
    free = (args["page_refs"] == 0).nonzero().view(-1)
    args["page_refs"][free[::2]] = -1
    check("resize", dict(args, new_lens=torch.tensor([20, 20], dtype=I32)), cuda)
    check("compact", args, cuda)


def test_entries_outside_the_pool_pass(cuda):
    args = make([40, 40, 20], 8, share=3, spare=9, seed=5)
    args["block_table"][0, 1], args["block_table"][1, 4], args["block_table"][2, 2] = -4, 10 ** 6, -1
    check("resize", dict(args, new_lens=torch.tensor([41, 12, 21], dtype=I32)), cuda)
    check("fork", dict(args, parents=torch.tensor([2, 2, 0, 1, 1])), cuda)
    check("compact", args, cuda)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("P,D", [(16, 64), (1, 8), (5, 24), (64, 128), (8, 3)])
def test_fork(cuda, P, D, dtype):
    lens = [0, 1, P, P + 1, 3 * P - 1, 2 * P]
    args = make(lens, P, dtype, D=D, spare=20, share=1, seed=P)
    for parents in ([0, 1, 2, 3, 4, 5], [4, 4, 4, 1, 4, 2], [5, 3, 3], [1] * 12, [], [-1, 6, 4, 2 ** 40, -2 ** 40, 4]):
        table, lens_now, refs, missing = check("fork", dict(args, parents=torch.tensor(parents, dtype=I64)), cuda)
        consistent(table, lens_now, refs, P)
        assert int(missing) == 0


def test_fork_without_enough_pages(cuda):
    args = make([20, 9, 16], 8, spare=2, seed=6)
    _, _, _, missing = check("fork", dict(args, parents=torch.tensor([0, 0, 1, 1, 0, 2, 2, 1])), cuda)
    assert int(missing) == 2


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("spare", [0, 1, 40])
def test_compact(cuda, spare, dtype):
    args = make([70, 3, 0, 16, 33, 48, 1], 16, dtype, spare=spare, share=1, seed=spare)
    table, refs, page_map = check("compact", args, cuda)
    consistent(table, args["seq_lens"], refs, 16)
    n = int((args["page_refs"] != 0).sum())
    assert (refs[:n] != 0).all() and not refs[n:].any()


def test_compact_twice_from_the_same_state(cuda):
    """The old places keep their contents: a compaction that was not taken can run again."""
    from llm_cuda.kernels.page_pool import paged_kv_compact

    args = on(cuda, make([70, 3, 30], 16, spare=12, seed=7))
    first = paged_kv_compact(**args)
    keys = args["key_pages"].clone()
    again = paged_kv_compact(**args)
    assert all(torch.equal(a, b) for a, b in zip(first, again)) and torch.equal(keys, args["key_pages"])


@pytest.mark.parametrize("N", [1, 15, 16, 17, 1023, 16384, 16400, 50001])
def test_large_pools(cuda, N):
    """Pools of up to several passes; the free pages at the front, at the end, and scattered."""
    g = torch.Generator().manual_seed(N)
    for where in ("front", "end", "scattered"):
        count = max(1, N // 5)
        free = {"front": torch.arange(count), "end": torch.arange(N - count, N),
                "scattered": torch.randperm(N, generator=g)[:count]}[where]
        refs = torch.randint(1, 4, (N,), generator=g).to(I32)
        refs[free] = 0
        pages = torch.arange(N, dtype=F32).view(1, N, 1, 1, 1)
        live = refs.nonzero().view(-1)
        table = torch.full((3, 1200), -1, dtype=I32)
        lens = torch.tensor([0, min(len(live), 700), 0], dtype=I32)
        table[1, :int(lens[1])] = live[:int(lens[1])].to(I32)
        args = dict(key_pages=pages.clone(), value_pages=-pages, block_table=table, seq_lens=lens, page_refs=refs)
        check("compact", args, cuda)
        check("resize", dict(args, new_lens=torch.tensor([1000, 710, 5], dtype=I32)), cuda)


@pytest.mark.parametrize("B", [1, 1023, 1025, 3000])
def test_large_batches(cuda, B):
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 20, (B,), generator=g).tolist()
    args = make(lens, 4, layers=1, Hkv=1, D=8, spare=3 * B, width=8, share=2, seed=B)
    now = torch.tensor(lens, dtype=I32) + torch.randint(-6, 9, (B,), generator=g).to(I32)
    table, refs, missing = check("resize", dict(args, new_lens=now), cuda)
    assert int(missing) == 0
    consistent(table, now.clamp(min=0), refs, 4)
    parents = torch.randint(-1, B, (B + 7,), generator=g)
    table, lens_now, refs, missing = check("fork", dict(args, parents=parents), cuda)
    if int(missing) == 0:  # (8 children of one row ask for more pages than there are)
        consistent(table, lens_now, refs, 4)
    check("compact", args, cuda)


def test_layouts_of_pools(cuda):
    """One layer without its dimension, pools inside a larger tensor, heads and slots swapped in
    memory, and an odd offset."""
    from llm_cuda.kernels.page_pool import paged_kv_compact, paged_kv_fork

    base = make([30, 17], 8, BF16, layers=3, Hkv=2, D=16, spare=5, seed=8)
    parents = torch.tensor([0, 0, 1, 1, 1])
    want = oracle.kv_fork(**base, parents=parents)
    N = base["key_pages"].shape[1]

    def inside(t, odd):
        big = torch.zeros(3, N, 9, 3, 25, dtype=BF16, device=cuda)
        part = big.transpose(2, 3)[:, :, 1:3, 1:9, odd:odd + 16]
        part.copy_(t.to(cuda))
        return part

    for odd in (0, 1):
        args = on(cuda, base)
        args["key_pages"], args["value_pages"] = inside(base["key_pages"], odd), inside(base["value_pages"], odd)
        got = paged_kv_fork(**args, parents=parents.to(cuda))
        same((*got, args["key_pages"], args["value_pages"]), want, ("table", "lens", "refs", "missing", "k", "v"))
    flat = on(cuda, dict(base, key_pages=base["key_pages"][1], value_pages=base["value_pages"][1]))
    got = paged_kv_compact(**flat)
    want = oracle.kv_compact(**dict(base, key_pages=base["key_pages"][1], value_pages=base["value_pages"][1]))
    same((*got, flat["key_pages"], flat["value_pages"]), want, ("table", "refs", "map", "k", "v"))


def test_strided_tables_and_empty_calls(cuda):
    from llm_cuda.kernels import page_pool

    base = make([30, 17, 9], 8, spare=5, seed=9)
    args = on(cuda, base)
    now = torch.tensor([31, 25, 3], dtype=I32)
    want = oracle.kv_resize(**base, new_lens=now)
    wide = torch.full((3, 2 * base["block_table"].shape[1]), 77, dtype=I32, device=cuda)
    wide[:, 1::2] = args["block_table"]
    args["block_table"] = wide[:, 1::2]
    both = torch.stack([base["seq_lens"], now], 1).to(cuda)
    args["seq_lens"] = both[:, 0]
    got = page_pool.paged_kv_resize(**args, new_lens=both[:, 1])
    same(got, want[:3], ("table", "refs", "missing"))
    none = dict(args, block_table=args["block_table"][:0], seq_lens=args["seq_lens"][:0])
    table, refs, missing = page_pool.paged_kv_resize(**none, new_lens=both[:0, 1])
    assert table.shape[0] == 0 and torch.equal(refs, args["page_refs"]) and int(missing) == 0
    table, refs, page_map = page_pool.paged_kv_compact(**none)
    assert table.shape[0] == 0 and int((refs != 0).sum()) == int((args["page_refs"] != 0).sum())
    table, lens, refs, _ = page_pool.paged_kv_fork(**none, parents=torch.tensor([0, -1], device=cuda))
    assert (table == -1).all() and not lens.any() and torch.equal(refs, args["page_refs"])


def test_graph_replays(cuda):
    """A round of growing, shrinking and forking, captured, follows the inputs' contents."""
    from llm_cuda.kernels import page_pool

    base = make([30, 17, 44], 8, spare=20, seed=10)
    args = on(cuda, base)
    now = torch.tensor([33, 20, 45], dtype=I32, device=cuda)
    parents = torch.tensor([0, 0, 2], device=cuda)
    k0, v0 = args["key_pages"].clone(), args["value_pages"].clone()

    def round_():
        t, r, m = page_pool.paged_kv_resize(**args, new_lens=now)
        t2, l2, r2, m2 = page_pool.paged_kv_fork(args["key_pages"], args["value_pages"], t, now, parents, r)
        t3, r3, pm = page_pool.paged_kv_compact(args["key_pages"], args["value_pages"], t2, l2, r2)
        return t, r, m, t2, l2, r2, m2, t3, r3, pm

    round_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = round_()
    for step in range(4):
        now.copy_(torch.tensor([33 + 3 * step, 20 - 5 * step, 45 + step], dtype=I32))
        parents.copy_(torch.tensor([step % 3, 0, 2]))
        args["key_pages"].copy_(k0)
        args["value_pages"].copy_(v0)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out] + [args["key_pages"].clone(), args["value_pages"].clone()]
        args["key_pages"].copy_(k0)
        args["value_pages"].copy_(v0)
        want = list(round_()) + [args["key_pages"], args["value_pages"]]
        assert all(torch.equal(a, b) for a, b in zip(got, want)), step


@pytest.mark.parametrize("Hkv,P,D,layers", [(8, 64, 128, 4), (2, 16, 32, 3)])
def test_whole_pages_of_real_sizes(cuda, Hkv, P, D, layers):
    args = make([150, 150, 90, 300, 64, 1], P, BF16, layers=layers, Hkv=Hkv, D=D, spare=30, share=1, seed=11)
    check("compact", args, cuda)
    check("fork", dict(args, parents=torch.tensor([0, 0, 0, 2, 2, 3, 3, 3, 5, 5])), cuda)


def test_counts_that_are_not_aligned(cuda):
    """page_refs from the second element of a buffer, in a pool of several passes."""
    from llm_cuda.kernels import page_pool

    g = torch.Generator().manual_seed(3)
    N = 20011
    refs = (torch.rand(N, generator=g) < 0.9).to(I32)
    live = refs.nonzero().view(-1).to(I32)
    pages = torch.arange(N, dtype=F32).view(1, N, 1, 1, 1)
    base = dict(key_pages=pages.clone(), value_pages=-pages, block_table=live[:600].view(2, 300).contiguous(),
                seq_lens=torch.tensor([100, 300], dtype=I32), page_refs=refs)
    now = torch.tensor([300, 20], dtype=I32)
    for name, want, more in (("resize", oracle.kv_resize(**base, new_lens=now), dict(new_lens=now)),
                             ("compact", oracle.kv_compact(**base), {})):
        args = on(cuda, dict(base, **more))
        args["page_refs"] = torch.cat([refs[:1], refs]).to(cuda)[1:]
        got = getattr(page_pool, f"paged_kv_{name}")(**args)
        same((*got, args["key_pages"], args["value_pages"]), want, ("table", "refs", "third", "k", "v"))


def test_a_pool_without_pages(cuda):
    from llm_cuda.kernels import page_pool

    pool = torch.empty(2, 0, 1, 4, 8, device=cuda)
    none = torch.zeros(0, dtype=I32, device=cuda)
    table, lens = torch.full((3, 5), -1, dtype=I32, device=cuda), torch.zeros(3, dtype=I32, device=cuda)
    t, refs, missing = page_pool.paged_kv_resize(pool, pool, table, lens, lens + 7, none)
    assert (t == -1).all() and refs.numel() == 0 and int(missing) == 6
    t, n, refs, missing = page_pool.paged_kv_fork(pool, pool, table, lens, torch.tensor([0, 0], device=cuda), none)
    assert t.shape == (2, 5) and not n.any() and int(missing) == 0
    t, refs, page_map = page_pool.paged_kv_compact(pool, pool, table, lens, none)
    assert (t == -1).all() and page_map.numel() == 0
