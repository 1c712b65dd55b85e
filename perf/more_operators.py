"""Performance cases of speculative decoding over a pool of pages: inputs, the plain
form, the framework's call, its work and its 64-bit result.

  extend    attention of the newest tokens of every sequence over the paged cache
            (`paged_extend_attention`): drafted tokens under verification, chunks of
            a prompt;
  verify    which drafted tokens stand, and the token after them
            (`verify_draft_tokens`);
  resize    sequences take pages as they grow and give them back
            (`paged_kv_resize`);
  fork      the batch becomes continuations of its rows (`paged_kv_fork`);
  compact   the pages in use move to the front of the pool (`paged_kv_compact`).

Head layouts are those of the benchmark and the configuration: the 8B attention
(32/8 heads of 128), the 70B attention (64/8 of 128), the default configuration
(16/8 of 64) and the tiny model (8/2 of 32).
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = {"bf16": 2, "f16": 2, "f32": 4}
# query heads, kv heads, head_dim
HEADS = {"8b": (32, 8, 128), "70b": (64, 8, 128), "default": (16, 8, 64), "tiny": (8, 2, 32)}
# A residual that sums to less is rounding: the distributions agree.
AGREE = 2.0 ** -32


def listed():
    return [
        # Four drafted tokens of one short conversation: the smallest attention call.
        dict(name="extend_one", op="extend", heads="8b", dtype="bf16", batch=1, rows=5, ctx=1000,
             page=64, ragged=False),
        # A decode batch under verification, contexts and drafts of unequal length.
        dict(name="extend_batch", op="extend", heads="8b", dtype="bf16", batch=32, rows=5,
             ctx=4096, page=64, ragged=True),
        # Long documents: the long-context shape of the benchmark, four drafted tokens.
        dict(name="extend_long", op="extend", heads="70b", dtype="bf16", batch=8, rows=5,
             ctx=32768, page=64, ragged=False),
        # Chunks of prompts beside a cache, small pages, float16.
        dict(name="extend_chunk", op="extend", heads="8b", dtype="f16", batch=3, rows=160, ctx=4000,
             page=16, ragged=True),
        # One conversation, drafts without probabilities (taken from the text itself).
        dict(name="verify_one", op="verify", dtype="bf16", batch=1, drafts=4, vocab=32000,
             drawn=False, temperature=1.0, ragged=False),
        # A batch at the full vocabulary, drafts drawn from a draft model's float32 logits.
        dict(name="verify_batch", op="verify", dtype="f32", batch=64, drafts=5, vocab=128256,
             drawn=True, temperature=0.7, ragged=True),
        # A batch before its next step: four drafted tokens and one more, some rows shared.
        dict(name="resize_grow", op="resize", heads="8b", dtype="bf16", layers=16, batch=48,
             tokens=130, change=5, common=1, twins=4, page=64, spare=60),
        # Rejected tokens of a large batch given back, in a large pool of small pages.
        dict(name="resize_shrink", op="resize", heads="tiny", dtype="bf16", layers=4, batch=256,
             tokens=1200, change=-40, common=4, twins=0, page=16, spare=2000),
        # Prompts become the rows of their samples.
        dict(name="fork_samples", op="fork", heads="8b", dtype="bf16", layers=32, batch=4,
             tokens=700, children=32, keep=1.0, common=0, page=64, spare=40),
        # Finished rows leave a batch.
        dict(name="fork_drop", op="fork", heads="default", dtype="f16", layers=12, batch=64,
             tokens=400, children=48, keep=0.75, common=2, page=32, spare=20),
        # A small pool of the default configuration after half of its rows left.
        dict(name="compact_small", op="compact", heads="default", dtype="bf16", layers=12, batch=6,
             tokens=300, common=0, page=64, spare=8),
        # A server's pool after a busy hour.
        dict(name="compact_pool", op="compact", heads="8b", dtype="bf16", layers=16, batch=32,
             tokens=360, common=2, page=64, spare=30),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(["extend", "extend", "extend", "verify", "verify", "resize", "fork", "compact"])
    if op == "extend":
        heads = rng.choice(["8b", "8b", "70b", "default", "tiny"])
        dtype = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
        if dtype == "f32":
            heads = rng.choice(["default", "tiny"])
            batch, rows = _log(rng, 1, 16), _log(rng, 1, 32)
            ctx = _log(rng, rows + 16, 16384 // batch)
        else:
            rows = _log(rng, 1, 256)
            batch = _log(rng, 1, 64 if rows <= 16 else 4)
            ctx = _log(rng, rows + 16, min(16384, 131072 // batch, (1 << 20) // (batch * rows)))
        return dict(op=op, heads=heads, dtype=dtype, batch=batch, rows=rows, ctx=max(ctx, rows),
                    page=rng.choice([16, 32, 64, 64, 128]), ragged=rng.random() < 0.5)
    if op == "verify":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        batch = _log(rng, 1, 48)
        return dict(op=op, dtype=dtype, batch=batch, drafts=_log(rng, 1, min(15, 320 // batch)),
                    vocab=_log(rng, 1000, 128256), drawn=rng.random() < 0.6,
                    temperature=rng.choice([1.0, 0.7, 1.3, 0.0]), ragged=rng.random() < 0.5)
    heads = rng.choice(["8b", "70b", "default", "tiny"])
    dtype = rng.choice(["bf16", "f16", "f32"]) if heads in ("default", "tiny") else "bf16"
    page, layers = rng.choice([16, 32, 64, 128]), _log(rng, 1, 12)
    batch = _log(rng, 2, 24 if heads in ("8b", "70b") else 64)
    tokens = _log(rng, 4, 300 if heads in ("8b", "70b") else min(1000, 16000 // batch))
    common = rng.randint(0, tokens // page // 2)
    case = dict(op=op, heads=heads, dtype=dtype, layers=layers, batch=batch, tokens=tokens,
                common=common, page=page)
    if op == "resize":
        change = rng.choice([1, 5, 9, 64, -3, -30])
        case.update(change=change, twins=rng.choice([0, 0, 1, batch // 2]),
                    spare=batch * (max(change, 0) // page + 3))
    elif op == "fork":
        keep = rng.choice([1.0, 0.5, 0.8])
        children = rng.randint(1, 2 * batch)
        case.update(children=children, keep=keep, spare=children)
    else:
        case.update(spare=_log(rng, 1, 32))
    return case


# --------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _lengths(count, top, ragged, g, low=0):
    """`count` lengths: all `top`, or even from a quarter of it up (one holds it)."""
    lens = torch.full((count,), top, dtype=torch.int32)
    if ragged:
        lens = torch.randint(max(low, top // 4), top + 1, (count,), generator=g).to(torch.int32)
        lens[int(torch.randint(0, count, (1,), generator=g))] = top
    return lens


def _extend_lengths(case, seed):
    g = torch.Generator().manual_seed(seed)
    queries = _lengths(case["batch"], case["rows"], case["ragged"], g, 1)
    return _lengths(case["batch"], case["ctx"], case["ragged"], g, case["rows"]), queries


def _prepare_extend(case, seed):
    Hq, Hkv, D = HEADS[case["heads"]]
    B, P, dt = case["batch"], case["page"], DTYPES[case["dtype"]]
    pages = -(-case["ctx"] // P)
    lens, queries = _extend_lengths(case, seed)
    g = _gen(seed)
    table = torch.randperm(B * pages, generator=g, device=DEV).to(torch.int32).view(B, pages)
    return dict(op="extend",
                q=torch.randn(B, case["rows"], Hq, D, generator=g, device=DEV, dtype=dt).transpose(1, 2),
                key_pages=torch.randn(B * pages, Hkv, P, D, generator=g, device=DEV, dtype=dt),
                value_pages=torch.randn(B * pages, Hkv, P, D, generator=g, device=DEV, dtype=dt),
                block_table=table, seq_lens=lens.to(DEV), query_lens=queries.to(DEV))


def _prepare_verify(case, seed):
    B, K, V, dt = case["batch"], case["drafts"], case["vocab"], DTYPES[case["dtype"]]
    g = _gen(seed)
    x = torch.randn(B, K + 1, V, generator=g, device=DEV) * 2.0
    # a few likely tokens, as a language model's logits have
    hot = torch.randint(0, V, (B, K + 1, 24), generator=g, device=DEV)
    x.scatter_add_(2, hot, 9 * torch.rand(B, K + 1, 24, generator=g, device=DEV))
    logits = x.to(dt)
    u = torch.rand(B, K + 1, generator=g, device=DEV)
    if case["drawn"]:
        # the draft model is near the target, and its tokens are drawn from it
        y = (x[:, :K] + 0.7 * torch.randn(B, K, V, generator=g, device=DEV)).to(dt)
        z = y.float()
        if case["temperature"] > 0:
            noise = torch.rand(B, K, V, generator=g, device=DEV).clamp_(min=1e-30).log_().neg_().log_()
            z = z / case["temperature"] - noise
        drafts = z.argmax(-1)
    else:
        y = None
        drafts = logits[:, :K].float().argmax(-1)
        other = torch.rand(B, K, generator=g, device=DEV) < 0.2
        drafts = torch.where(other, torch.randint(0, V, (B, K), generator=g, device=DEV), drafts)
    lens = _lengths(B, K, case["ragged"], torch.Generator().manual_seed(seed))
    return dict(op="verify", logits=logits, draft_tokens=drafts, uniforms=u, draft_logits=y,
                draft_lens=lens.to(DEV), temperature=case["temperature"])


def _batch(case, seed):
    """Host side of a batch in a pool: lengths, table, references, pool size. The first
    `common` whole pages of every two neighbours are shared; the first `twins` pairs of
    neighbours are equal altogether."""
    g = torch.Generator().manual_seed(seed)
    B, P = case["batch"], case["page"]
    lens = _lengths(B, case["tokens"], True, g, 1)
    for i in range(case.get("twins", 0)):
        if 2 * i + 1 < B:
            lens[2 * i + 1] = lens[2 * i]
    longest = max(case["tokens"], case["tokens"] + case.get("change", 0))
    width = -(-longest // P) + 1
    table = torch.full((B, width), -1, dtype=torch.int64)
    used = 0
    for b in range(B):
        held = -(-int(lens[b]) // P)
        shared = 0
        if b % 2:
            shared = min(case["common"], int(lens[b]) // P, int(lens[b - 1]) // P)
            if b // 2 < case.get("twins", 0):
                shared = held
            table[b, :shared] = table[b - 1, :shared]
        table[b, shared:held] = torch.arange(used, used + held - shared)
        used += held - shared
    pool = B * -(-case["tokens"] // P) + case["spare"]  # (the same whatever the lengths)
    order = torch.randperm(pool, generator=g)
    table = torch.where(table >= 0, order[table.clamp(min=0)], -1)
    refs = torch.bincount(table[table >= 0], minlength=pool)
    return lens, table.to(torch.int32), refs.to(torch.int32), pool, g


def _prepare_pool(case, seed):
    _, Hkv, D = HEADS[case["heads"]]
    lens, table, refs, pool, g = _batch(case, seed)
    gpu, dt = _gen(seed), DTYPES[case["dtype"]]
    shape = (case["layers"], pool, Hkv, case["page"], D)
    s = dict(op=case["op"], key_pages=torch.randn(shape, generator=gpu, device=DEV, dtype=dt),
             value_pages=torch.randn(shape, generator=gpu, device=DEV, dtype=dt),
             block_table=table.to(DEV), seq_lens=lens.to(DEV), page_refs=refs.to(DEV))
    if case["op"] == "resize":
        s["new_lens"] = (lens + case["change"]).clamp(min=0).to(DEV)
    if case["op"] == "fork":
        kept = max(1, int(round(case["keep"] * case["batch"])))
        rows = torch.randperm(case["batch"], generator=g)[:kept]
        extra = rows[torch.randint(0, kept, (max(0, case["children"] - kept),), generator=g)]
        s["parents"] = torch.cat([rows, extra])[:case["children"]].sort().values.to(DEV)
    return s


def prepare(case, seed):
    return {"extend": _prepare_extend, "verify": _prepare_verify}.get(case["op"], _prepare_pool)(case, seed)


# --------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------
def _rows(pages, table):
    """The table's tokens in float32, [rows, kv heads, tokens, head_dim]."""
    R, M = table.shape
    _, H, P, D = pages.shape
    got = pages[table.long()].float()
    return got.permute(0, 2, 1, 3, 4).reshape(R, H, M * P, D)


def _plain_extend(s):
    q, table = s["q"].float(), s["block_table"]
    B, Hq, T, D = q.shape
    Hkv = s["key_pages"].shape[1]
    k, v = _rows(s["key_pages"], table), _rows(s["value_pages"], table)
    sc = torch.matmul(q.reshape(B, Hkv, -1, D), k.transpose(2, 3).contiguous()) / math.sqrt(D)
    sc = sc.view(B, Hq, T, -1)
    row = torch.arange(T, device=DEV).view(1, T, 1)
    n = s["query_lens"].view(B, 1, 1)
    at = s["seq_lens"].view(B, 1, 1) - n + row
    seen = (torch.arange(k.shape[2], device=DEV) <= at) & (row < n)
    sc = sc.masked_fill(~seen.unsqueeze(1), -math.inf)
    m = sc.amax(-1, keepdim=True)
    e = torch.exp(sc - torch.where(torch.isneginf(m), 0.0, m))
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e.view(B, Hkv, -1, k.shape[2]), v).view(B, Hq, T, D)
    out = out / torch.where(total == 0, 1.0, total)
    return out.to(s["q"].dtype), (m + torch.log(total)).squeeze(-1)


def _plain_distribution(x, temperature):
    """softmax(x / temperature) in 64 bits; one-hot at the first largest for 0."""
    x = x.double()
    if temperature <= 0:
        top = x.amax(-1, keepdim=True)
        first = torch.cumsum(x == top, -1) == 1
        return ((x == top) & first).double()
    e = torch.exp((x - x.amax(-1, keepdim=True)) / temperature)
    return e / e.sum(-1, keepdim=True)


def _plain_verify(s):
    d, u, n = s["draft_tokens"], s["uniforms"].double(), s["draft_lens"].long()
    B, K = d.shape
    V = s["logits"].shape[-1]
    p = _plain_distribution(s["logits"], s["temperature"])
    if s["draft_logits"] is None:
        q = (torch.arange(V, device=DEV) == d.unsqueeze(-1)).double()
    else:
        q = _plain_distribution(s["draft_logits"], s["temperature"])
    pd = torch.gather(p[:, :K], 2, d.unsqueeze(-1)).squeeze(-1)
    qd = torch.gather(q, 2, d.unsqueeze(-1)).squeeze(-1)
    stands = (u[:, :K] * qd < pd) & (torch.arange(K, device=DEV) < n.unsqueeze(1))
    a = torch.cumprod(stands.long(), 1).sum(1)
    at = torch.arange(B, device=DEV)
    w = p[at, a]
    refused = a < n
    rest = (w - q[at, a.clamp(max=K - 1)]).clamp(min=0)
    use = (refused & (rest.sum(-1) >= AGREE)).unsqueeze(-1)
    w = torch.where(use, rest, w)
    run_sum = torch.cumsum(w, -1)
    token = (run_sum <= (u[:, K] * run_sum[:, -1]).unsqueeze(-1)).sum(-1)
    out = torch.full((B, K + 1), -1, dtype=torch.int64, device=DEV)
    col = torch.arange(K + 1, device=DEV)
    out[:, :K] = torch.where(col[:K] < a.unsqueeze(1), d, -1)
    out = torch.where(col == a.unsqueeze(1), token.unsqueeze(1), out)
    return out, a.to(torch.int32)


def _copy_slots(pools, src, dst, fill):
    """Of page src[i] the first fill[i] slots to page dst[i], in every layer."""
    P = pools[0].shape[3]
    live = torch.arange(P, device=DEV).view(1, 1, 1, P, 1) < fill.view(1, -1, 1, 1, 1)
    for pages in pools:
        pages[:, dst] = torch.where(live, pages[:, src], pages[:, dst])


def _free_pages(refs):
    return torch.nonzero(refs == 0).view(-1)


def _plain_resize(s):
    table, refs, P = s["block_table"].long(), s["page_refs"].long(), s["key_pages"].shape[3]
    B, M = table.shape
    lens, new = s["seq_lens"].long(), s["new_lens"].long()
    col = torch.arange(M, device=DEV).view(1, M)
    held, want = ((lens + P - 1) // P).view(B, 1), ((new + P - 1) // P).view(B, 1)
    fill = (lens % P).view(B, 1)
    named = refs[table.clamp(min=0)]
    copied = ((new > lens).view(B, 1) & (fill > 0) & (col == (lens // P).view(B, 1)) & (named > 1))
    fresh = ((col >= held) & (col < want)) | copied
    rank = torch.cumsum(fresh.view(-1), 0).view(B, M) - 1
    free = _free_pages(refs)
    got = torch.where(rank < len(free), free[rank.clamp(0, max(len(free) - 1, 0))], -1)
    out = torch.where(fresh, got, torch.where(col < torch.minimum(held, want), table, -1))
    left = ((col >= want) & (col < held)) | copied
    after = refs.clone()
    after.index_add_(0, table[left], torch.full_like(table[left], -1))
    after.index_add_(0, out[fresh], torch.ones_like(out[fresh]))
    src, dst = table[copied], out[copied]
    _copy_slots((s["key_pages"], s["value_pages"]), src, dst, fill.expand(B, M)[copied])
    missing = (fresh.sum() - len(free)).clamp(min=0).view(1)
    return (out.to(torch.int32), after.to(torch.int32), missing.to(torch.int32), s["key_pages"],
            s["value_pages"])


def _plain_fork(s):
    table, refs, P = s["block_table"].long(), s["page_refs"].long(), s["key_pages"].shape[3]
    M, parents, lens = table.shape[1], s["parents"], s["seq_lens"].long()
    R = len(parents)
    col = torch.arange(M, device=DEV).view(1, M)
    n = lens[parents]
    whole, fill = (n // P).view(R, 1), (n % P).view(R, 1)
    same = parents.view(R, 1) == parents.view(1, R)
    later = (same & torch.ones(R, R, dtype=torch.bool, device=DEV).tril(-1)).any(1).view(R, 1)
    copied = (col == whole) & (fill > 0) & later
    rank = torch.cumsum(copied.view(-1), 0).view(R, M) - 1
    free = _free_pages(refs)
    out = torch.where(col < (n.view(R, 1) + P - 1) // P, table[parents], -1)
    src = out[copied]
    out = torch.where(copied, free[rank.clamp(0, len(free) - 1)], out)
    after = refs.clone()
    old = table[col < ((lens + P - 1) // P).view(-1, 1)]
    after.index_add_(0, old, torch.full_like(old, -1))
    live = out[out >= 0]
    after.index_add_(0, live, torch.ones_like(live))
    _copy_slots((s["key_pages"], s["value_pages"]), src, out[copied], fill.expand(R, M)[copied])
    missing = (copied.sum() - len(free)).clamp(min=0).view(1)
    return (out.to(torch.int32), n.to(torch.int32), after.to(torch.int32), missing.to(torch.int32),
            s["key_pages"], s["value_pages"])


def _plain_compact(s):
    table, refs, P = s["block_table"].long(), s["page_refs"], s["key_pages"].shape[3]
    N, M = len(refs), table.shape[1]
    page = torch.arange(N, device=DEV)
    n = (refs != 0).sum()
    src = page[(refs != 0) & (page >= n)]
    dst = page[(refs == 0) & (page < n)]
    new = torch.where(refs != 0, page, -1)
    new[src] = dst
    held = ((s["seq_lens"].long() + P - 1) // P).view(-1, 1)
    out = torch.where(torch.arange(M, device=DEV).view(1, M) < held, new[table.clamp(min=0)], -1)
    after = torch.zeros_like(refs)
    after[new[refs != 0]] = refs[refs != 0]
    for pages in (s["key_pages"], s["value_pages"]):
        pages[:, dst] = pages[:, src]
    return out.to(torch.int32), after, new.to(torch.int32), s["key_pages"], s["value_pages"]


def _own_modules():
    path = os.path.join(os.getcwd(), "llm-cuda_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from llm_cuda.kernels import page_pool, speculative
    from llm_cuda.kernels.triton import decode_attention

    return decode_attention, speculative, page_pool


def run(state):
    s = state
    if not own:
        return {"extend": _plain_extend, "verify": _plain_verify, "resize": _plain_resize,
                "fork": _plain_fork, "compact": _plain_compact}[s["op"]](s)
    decode_attention, speculative, page_pool = _own_modules()
    if s["op"] == "extend":
        return decode_attention.paged_extend_attention(
            s["q"], s["key_pages"], s["value_pages"], s["block_table"], s["seq_lens"],
            query_lens=s["query_lens"], return_lse=True)
    if s["op"] == "verify":
        return speculative.verify_draft_tokens(
            s["logits"], s["draft_tokens"], s["uniforms"], draft_logits=s["draft_logits"],
            draft_lens=s["draft_lens"], temperature=s["temperature"])
    pools = (s["key_pages"], s["value_pages"])
    if s["op"] == "resize":
        got = page_pool.paged_kv_resize(*pools, s["block_table"], s["seq_lens"], s["new_lens"],
                                        s["page_refs"])
    elif s["op"] == "fork":
        got = page_pool.paged_kv_fork(*pools, s["block_table"], s["seq_lens"], s["parents"],
                                      s["page_refs"])
    else:
        got = page_pool.paged_kv_compact(*pools, s["block_table"], s["seq_lens"], s["page_refs"])
    return (*got, *pools)


# --------------------------------------------------------------------------
# Work and 64-bit results
# --------------------------------------------------------------------------
def work(case):
    e = SIZES[case["dtype"]]
    # ragged lengths are even from a quarter up: five eighths of the longest on average
    part = lambda count, top: top * (1 + 0.625 * (count - 1)) if case["ragged"] else count * top  # noqa: E731
    if case["op"] == "extend":
        Hq, Hkv, D = HEADS[case["heads"]]
        B, T = case["batch"], case["rows"]
        tokens, rows = part(B, case["ctx"]), part(B, T)
        return {"bytes": 2 * Hkv * D * e * tokens + (rows + B * T) * Hq * D * e + 4 * B * Hq * T,
                "flops": 4 * Hq * D * tokens * rows / B}
    if case["op"] == "verify":
        B, K = case["batch"], case["drafts"]
        drafts = part(B, K)
        rows = drafts + B + (drafts if case["drawn"] else 0)
        return {"bytes": rows * case["vocab"] * e + 12 * B * (K + 1) + 8 * B * (K + 1),
                "flops": 4 * rows * case["vocab"]}
    lens, table, refs, pool, _ = _batch(case, 0)
    _, Hkv, D = HEADS[case["heads"]]
    slot = 2 * case["layers"] * Hkv * D * e
    P, B, M = case["page"], *table.shape
    slots, rows = 0, B
    if case["op"] == "resize" and case["change"] > 0:
        for b in range(B):
            n = int(lens[b])
            if n % P and int(refs[table[b, n // P]]) > 1:
                slots += n % P
    elif case["op"] == "fork":
        rows = case["children"]
        kept = max(1, int(round(case["keep"] * B)))
        slots = max(0, rows - kept) * P // 2
    elif case["op"] == "compact":
        live = refs != 0
        slots = int(live[int(live.sum()):].sum()) * P
    return {"bytes": 2 * slots * slot + 4 * (B + rows) * M + 8 * pool + 8 * (B + rows), "flops": 0}


def _exact_extend(case, seed):
    s = _prepare_extend(case, seed)
    Hq, Hkv, D = HEADS[case["heads"]]
    B, T, P = case["batch"], case["rows"], case["page"]
    lens, queries = _extend_lengths(case, seed)
    out = torch.zeros(B, Hq, T, D, dtype=torch.float64, device=DEV)
    lse = torch.full((B, Hq, T), -math.inf, dtype=torch.float64, device=DEV)
    for b in range(B):
        L, n = int(lens[b]), int(queries[b])
        pos = torch.arange(L, device=DEV)
        ids = s["block_table"][b, pos // P].long()
        k = s["key_pages"][ids, :, pos % P].double().permute(1, 2, 0).contiguous()
        v = s["value_pages"][ids, :, pos % P].double().permute(1, 0, 2).contiguous()
        q = s["q"][b, :, :n].double().reshape(Hkv, -1, D)
        sc = (torch.bmm(q, k) / math.sqrt(D)).view(Hkv, Hq // Hkv, n, L)
        ahead = pos.view(1, L) > (L - n + torch.arange(n, device=DEV)).view(n, 1)
        sc[:, :, ahead] = -math.inf
        peak = sc.max(-1, keepdim=True).values
        p = (sc - peak).exp()
        total = p.sum(-1, keepdim=True)
        o = torch.bmm((p / total).view(Hkv, -1, L), v)
        out[b, :, :n] = o.view(Hq, n, D)
        lse[b, :, :n] = (peak + total.log()).view(Hq, n)
    return out, lse


def _exact_verify(case, seed):
    s = _prepare_verify(case, seed)
    B, K, V = case["batch"], case["drafts"], case["vocab"]
    host = lambda t: t.double().cpu().numpy()  # noqa: E731
    x, d, u = host(s["logits"]), s["draft_tokens"].cpu().numpy(), host(s["uniforms"])
    y = None if s["draft_logits"] is None else host(s["draft_logits"])
    lens, temp = s["draft_lens"].cpu().numpy(), case["temperature"]

    def chances(row):
        if temp <= 0:
            return (np.arange(V) == row.argmax()).astype(np.float64)
        e = np.exp((row - row.max()) / temp)
        return e / e.sum()

    tokens = np.full((B, K + 1), -1, dtype=np.int64)
    accepted = np.zeros(B, dtype=np.int32)
    for b in range(B):
        i = 0
        while True:
            p = chances(x[b, i])
            if i == lens[b]:
                break
            q = chances(y[b, i]) if y is not None else (np.arange(V) == d[b, i]).astype(np.float64)
            if not u[b, i] * q[d[b, i]] < p[d[b, i]]:
                rest = np.maximum(p - q, 0)
                p = rest if rest.sum() >= AGREE else p
                break
            tokens[b, i] = d[b, i]
            i += 1
        accepted[b] = i
        total = np.cumsum(p)
        tokens[b, i] = np.searchsorted(total, u[b, K] * total[-1], side="right")
    return torch.from_numpy(tokens).to(DEV), torch.from_numpy(accepted).to(DEV)


def _exact_moves(s, moves):
    for src, dst, fill in moves:
        for pages in (s["key_pages"], s["value_pages"]):
            pages[:, dst, :, :fill] = pages[:, src, :, :fill]
    return s["key_pages"].double(), s["value_pages"].double()


def _exact_pool(case, seed):
    s, P = _prepare_pool(case, seed), case["page"]
    lens, table, refs, pool, _ = _batch(case, seed)
    lens, table, refs = lens.tolist(), table.tolist(), refs.tolist()
    B, M = case["batch"], len(table[0])
    free = [i for i in range(pool) if refs[i] == 0]
    after, moves, missing = list(refs), [], 0
    back = lambda rows: torch.tensor(rows, dtype=torch.int32, device=DEV)  # noqa: E731
    if case["op"] == "compact":
        n = pool - len(free)
        new = [-1 if refs[i] == 0 else i for i in range(pool)]
        holes = iter(free)
        for i in range(n, pool):
            if refs[i]:
                new[i] = next(holes)
                moves.append((i, new[i], P))
        after = [0] * pool
        for i in range(pool):
            if refs[i]:
                after[new[i]] = refs[i]
        rows = [[new[e] if c * P < lens[b] else -1 for c, e in enumerate(table[b])] for b in range(B)]
        return (back(rows), back(after), back(new), *_exact_moves(s, moves))

    def take():
        nonlocal missing
        if free:
            after[free[0]] = 1
            return free.pop(0)
        missing += 1
        return -1

    rows = []
    if case["op"] == "resize":
        for b in range(B):
            n, m, row = lens[b], max(0, lens[b] + case["change"]), list(table[b])
            held, want = -(-n // P), -(-m // P)
            if m > n and n % P and refs[row[n // P]] > 1:
                old = row[n // P]
                after[old] -= 1
                row[n // P] = take()
                moves.append((old, row[n // P], n % P))
            for c in range(M):
                if held <= c < want:
                    row[c] = take()
                elif c >= want:
                    if c < held:
                        after[row[c]] -= 1
                    row[c] = -1
            rows.append(row)
        return (back(rows), back(after), back([missing]), *_exact_moves(s, moves))
    parents = s["parents"].tolist()
    for b in range(B):
        for c in range(-(-lens[b] // P)):
            after[table[b][c]] -= 1
    first = set()
    for p in parents:
        n, row = lens[p], list(table[p])
        for c in range(M):
            if c * P >= n:
                row[c] = -1
            elif c == n // P and p in first:
                old = row[c]
                row[c] = take()
                moves.append((old, row[c], n % P))
            else:
                after[row[c]] += 1
        first.add(p)
        rows.append(row)
    return (back(rows), back([lens[p] for p in parents]), back(after), back([missing]),
            *_exact_moves(s, moves))


def exact(case, seed):
    return {"extend": _exact_extend, "verify": _exact_verify}.get(case["op"], _exact_pool)(case, seed)
