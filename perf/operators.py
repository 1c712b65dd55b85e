"""Performance cases of beam search over the paged KV cache: inputs, the plain
form, the framework's call, its work and its 64-bit result.

  prefix    one-token attention of a batch whose groups of sequences share a
            prefix (`shared_prefix_decode_attention`): the beams of a prompt, or
            the requests behind one system prompt;
  select    the best continuations over beams and vocabulary (`beam_select`);
  reorder   the caches follow the selected beams (`paged_kv_reorder`).

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


def listed():
    return [
        # Four beams of one question, a few tokens in: the smallest attention call.
        dict(name="prefix_beams4", op="prefix", heads="8b", dtype="bf16", groups=1, width=4,
             prefix=1000, ctx=30, page=64, ragged=False),
        # Beam search over a batch of prompts, small pages, float16, default configuration.
        dict(name="prefix_page16", op="prefix", heads="default", dtype="f16", groups=3, width=5,
             prefix=777, ctx=100, page=16, ragged=True),
        # Beam search over a batch of documents.
        dict(name="prefix_beams8", op="prefix", heads="8b", dtype="bf16", groups=4, width=8,
             prefix=4096, ctx=128, page=64, ragged=False),
        # A full decode batch of chats of unequal length behind one long system prompt.
        dict(name="prefix_system", op="prefix", heads="8b", dtype="bf16", groups=1, width=64,
             prefix=8192, ctx=1000, page=64, ragged=True),
        # Many samples of one long prompt: enough rows that the products bound it.
        dict(name="prefix_samples", op="prefix", heads="8b", dtype="bf16", groups=1, width=256,
             prefix=8192, ctx=200, page=128, ragged=False),
        # The default configuration in float32, as its tests run it.
        dict(name="prefix_f32", op="prefix", heads="default", dtype="f32", groups=2, width=4,
             prefix=1500, ctx=64, page=64, ragged=False),
        # One prompt's beams over a small vocabulary: the smallest selection.
        dict(name="select_beams4", op="select", dtype="bf16", groups=1, width=4, vocab=32000,
             count=4, finished=0, banned=0.0, first=False),
        # A batch of prompts over the full vocabulary, some beams finished.
        dict(name="select_batch", op="select", dtype="bf16", groups=8, width=8, vocab=128256,
             count=8, finished=1, banned=0.0, first=False),
        # Wide beams from float32 logits, twice as many candidates as beams.
        dict(name="select_wide", op="select", dtype="f32", groups=16, width=16, vocab=128256,
             count=32, finished=0, banned=0.5, first=False),
        # One prompt's beams in the default configuration (12 layers).
        dict(name="reorder_beams4", op="reorder", heads="default", dtype="bf16", layers=12,
             groups=1, width=4, tokens=37, pages=4, page=64, childless=1),
        # A batch of prompts in the 8B configuration (32 layers).
        dict(name="reorder_batch", op="reorder", heads="8b", dtype="bf16", layers=32, groups=4,
             width=8, tokens=300, pages=8, page=64, childless=3),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(["prefix", "prefix", "prefix", "select", "select", "reorder"])
    if op == "prefix":
        heads = rng.choice(["8b", "8b", "70b", "default", "tiny"])
        dtype = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
        if dtype == "f32":
            heads, groups, width = rng.choice(["default", "tiny"]), _log(rng, 1, 4), _log(rng, 1, 16)
            return dict(op=op, heads=heads, dtype=dtype, groups=groups, width=width,
                        prefix=_log(rng, 16, 4096 // groups), ctx=_log(rng, 1, 256),
                        page=rng.choice([16, 64, 128]), ragged=rng.random() < 0.5)
        width = _log(rng, 1, 128 if heads == "70b" else 256)
        groups = _log(rng, 1, min(8, 256 // width))
        return dict(op=op, heads=heads, dtype=dtype, groups=groups, width=width,
                    prefix=_log(rng, 16, 8192 // groups), ctx=_log(rng, 1, min(2048, 51200 // (groups * width))),
                    page=rng.choice([16, 32, 64, 64, 128]), ragged=rng.random() < 0.5)
    if op == "select":
        width = _log(rng, 1, 32)
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        vocab = _log(rng, 1000, 128256)
        return dict(op=op, dtype=dtype, groups=_log(rng, 1, 256 // width), width=width, vocab=vocab,
                    count=width * rng.choice([1, 1, 2]), finished=rng.choice([0, 0, width // 3]),
                    banned=rng.choice([0.0, 0.0, 0.3, 0.999]), first=rng.random() < 0.2)
    heads = rng.choice(["8b", "70b", "default", "tiny"])
    width = _log(rng, 1, 16)
    groups = _log(rng, 1, 32 // width)
    page = rng.choice([16, 32, 64, 128])
    tokens = _log(rng, 1, 512)
    childless = rng.randint(0, (width * 2) // 5)
    return dict(op=op, heads=heads, dtype=rng.choice(["bf16", "f16", "f32"]) if heads in ("default", "tiny") else "bf16",
                layers=_log(rng, 1, 32), groups=groups, width=width, tokens=tokens,
                pages=tokens // page + 1 + rng.randint(0, 3), page=page, childless=childless)


# --------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _lengths(count, top, ragged, g):
    """`count` lengths: all `top`, or even from a quarter of it up (one holds it)."""
    lens = torch.full((count,), top, dtype=torch.int32)
    if ragged:
        lens = torch.randint(max(0, top // 4), top + 1, (count,), generator=g).to(torch.int32)
        lens[int(torch.randint(0, count, (1,), generator=g))] = top
    return lens


def _prefix_shape(case):
    Hq, Hkv, D = HEADS[case["heads"]]
    N, W, P = case["groups"], case["width"], case["page"]
    return Hq, Hkv, D, N, W, N * W, P


def _prefix_lengths(case, seed):
    _, _, _, N, _, B, _ = _prefix_shape(case)
    g = torch.Generator().manual_seed(seed)
    return (_lengths(N, case["prefix"], case["ragged"], g),
            _lengths(B, case["ctx"], case["ragged"], g))


def _prepare_prefix(case, seed):
    Hq, Hkv, D, N, W, B, P = _prefix_shape(case)
    dt = DTYPES[case["dtype"]]
    plen, slen = _prefix_lengths(case, seed)
    pp, sp = -(-case["prefix"] // P), -(-case["ctx"] // P)
    pool = N * pp + B * sp
    g = _gen(seed)
    order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
    q = torch.randn(B, 1, Hq, D, generator=g, device=DEV, dtype=dt).transpose(1, 2)
    return dict(op="prefix", q=q, groups=N,
                key_pages=torch.randn(pool, Hkv, P, D, generator=g, device=DEV, dtype=dt),
                value_pages=torch.randn(pool, Hkv, P, D, generator=g, device=DEV, dtype=dt),
                prefix_table=order[:N * pp].view(N, pp), block_table=order[N * pp:].view(B, sp),
                prefix_lens=plen.to(DEV), seq_lens=slen.to(DEV))


def _prepare_select(case, seed):
    N, W, V = case["groups"], case["width"], case["vocab"]
    g = _gen(seed)
    x = torch.randn(N, W, V, generator=g, device=DEV) * 2.5
    # a few likely tokens per beam, as a language model's logits have
    hot = torch.randint(0, V, (N, W, 24), generator=g, device=DEV)
    x.scatter_add_(2, hot, 6 * torch.rand(N, W, 24, generator=g, device=DEV))
    if case["banned"]:
        x.masked_fill_(torch.rand(N, W, V, generator=g, device=DEV) < case["banned"], -math.inf)
    scores = (-20 - 5 * torch.rand(N, W, generator=g, device=DEV)).sort(1, descending=True).values
    done = torch.zeros(N, W, dtype=torch.bool, device=DEV)
    if case["first"]:
        # the first step: every beam is the prompt, and the first stands for all
        x[:, 1:] = x[:, :1]
        scores = torch.full((N, W), -math.inf, device=DEV)
        scores[:, 0] = 0.0
    elif case["finished"]:
        pick = torch.rand(N, W, generator=g, device=DEV).argsort(1)[:, :case["finished"]]
        done.scatter_(1, pick, True)
    return dict(op="select", logits=x.to(DTYPES[case["dtype"]]), scores=scores, finished=done,
                eos=V - 1, count=case["count"])


def _parents(case, seed):
    """Parents of a step in which exactly `childless` beams of each group have no child."""
    N, W, c = case["groups"], case["width"], case["childless"]
    g = torch.Generator().manual_seed(seed)
    rows = []
    for _ in range(N):
        order = torch.randperm(W, generator=g)
        live = order[c:]
        extra = live[torch.randint(0, W - c, (c,), generator=g)]
        both = torch.cat([live, extra])
        rows.append(both[torch.randperm(W, generator=g)])
    return torch.stack(rows)


def _prepare_reorder(case, seed):
    _, Hkv, D = HEADS[case["heads"]]
    L, N, W, P, M = case["layers"], case["groups"], case["width"], case["page"], case["pages"]
    B, dt, g = N * W, DTYPES[case["dtype"]], _gen(seed)
    order = torch.randperm(B * M, generator=g, device=DEV).to(torch.int32)
    return dict(op="reorder", parents=_parents(case, seed).to(DEV),
                key_pages=torch.randn(L, B * M, Hkv, P, D, generator=g, device=DEV, dtype=dt),
                value_pages=torch.randn(L, B * M, Hkv, P, D, generator=g, device=DEV, dtype=dt),
                block_table=order.view(B, M),
                seq_lens=torch.full((B,), case["tokens"], dtype=torch.int32, device=DEV))


def prepare(case, seed):
    return {"prefix": _prepare_prefix, "select": _prepare_select,
            "reorder": _prepare_reorder}[case["op"]](case, seed)


# --------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------
def _rows(pages, table):
    """The table's tokens in float32, [rows, kv heads, tokens, head_dim]."""
    R, M = table.shape
    _, H, P, D = pages.shape
    got = pages[table.long()].float()
    return got.permute(0, 2, 1, 3, 4).reshape(R, H, M * P, D)


def _plain_prefix(s):
    q, N = s["q"].squeeze(2).float(), s["groups"]
    B, Hq, D = q.shape
    Hkv = s["key_pages"].shape[1]
    W, G = B // N, Hq // Hkv
    scale = 1.0 / math.sqrt(D)
    kp, vp = _rows(s["key_pages"], s["prefix_table"]), _rows(s["value_pages"], s["prefix_table"])
    ko, vo = _rows(s["key_pages"], s["block_table"]), _rows(s["value_pages"], s["block_table"])
    # the prefix: all rows of a group against its tokens
    qg = q.view(N, W, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(N, Hkv, W * G, D)
    sp = torch.matmul(qg, kp.transpose(2, 3).contiguous()) * scale
    hidden = torch.arange(kp.shape[2], device=DEV) >= s["prefix_lens"].view(N, 1, 1, 1)
    sp = sp.masked_fill(hidden, -math.inf)
    # own tokens: each sequence against its own
    so = torch.matmul(q.view(B, Hkv, G, D), ko.transpose(2, 3).contiguous()) * scale
    hidden = torch.arange(ko.shape[2], device=DEV) >= s["seq_lens"].view(B, 1, 1, 1)
    so = so.masked_fill(hidden, -math.inf)
    so_g = so.view(N, W, Hkv, G, -1).permute(0, 2, 1, 3, 4).reshape(N, Hkv, W * G, -1)
    m = torch.maximum(sp.amax(-1, keepdim=True), so_g.amax(-1, keepdim=True))
    ep, eo = torch.exp(sp - m), torch.exp(so_g - m)
    total = ep.sum(-1, keepdim=True) + eo.sum(-1, keepdim=True)
    eo = eo.view(N, Hkv, W, G, -1).permute(0, 2, 1, 3, 4).reshape(B, Hkv, G, -1)
    out = torch.matmul(ep, vp).view(N, Hkv, W, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, G, D)
    out = out + torch.matmul(eo, vo)
    back = lambda t: t.view(N, Hkv, W, G, -1).permute(0, 2, 1, 3, 4).reshape(B, Hkv, G, -1)  # noqa: E731
    out = out / back(total)
    lse = (m + torch.log(total))
    return out.reshape(B, Hq, 1, D).to(s["q"].dtype), back(lse).reshape(B, Hq)


def _plain_select(s):
    # 64 bits: candidates of different beams are compared by sums that may differ in their last digits
    x, K = s["logits"].double(), s["count"]
    N, W, V = x.shape
    top = x.amax(-1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    value = s["scores"].double().unsqueeze(-1) + (x - lse)
    value = torch.where(torch.isneginf(top) | torch.isneginf(s["scores"]).unsqueeze(-1), -math.inf, value)
    alone = torch.where(torch.arange(V, device=DEV) == s["eos"],
                        s["scores"].double().unsqueeze(-1), -math.inf)
    value = torch.where(s["finished"].unsqueeze(-1), alone, value).view(N, W * V)
    best, at = torch.sort(value, dim=-1, descending=True, stable=True)
    best, at = best[:, :K], at[:, :K]
    parents, tokens = at // V, at % V
    done = torch.gather(s["finished"], 1, parents) | (tokens == s["eos"])
    return best.float(), tokens, parents, done


def _plain_reorder(s):
    kp, vp, table, parents = s["key_pages"], s["value_pages"], s["block_table"], s["parents"]
    N, W = parents.shape
    L, _, Hkv, P, D = kp.shape
    B, M = table.shape
    n = s["seq_lens"].view(N, W)[:, :1].long()
    col, fill = n // P, n % P  # of each group
    of = (parents + torch.arange(N, device=DEV).view(N, 1) * W).view(B)
    # a child is first if no earlier one has its parent; the rest take the childless rows in turn
    same = parents.unsqueeze(2) == parents.unsqueeze(1)
    earlier = torch.ones(W, W, dtype=torch.bool, device=DEV).tril(-1)
    later_child = (same & earlier).any(2)
    childless = ~(parents.unsqueeze(1) == torch.arange(W, device=DEV).view(1, W, 1)).any(2)
    rank = torch.cumsum(later_child, 1) - 1
    spare = torch.argsort(torch.where(childless, 0, 1) * W + torch.arange(W, device=DEV), dim=1)
    home = torch.where(later_child, torch.gather(spare, 1, rank.clamp(min=0)), parents)
    home = (home + torch.arange(N, device=DEV).view(N, 1) * W).view(B)
    c = torch.arange(M, device=DEV).view(1, M)
    col_b, fill_b = col.expand(N, W).reshape(B, 1), fill.expand(N, W).reshape(B, 1)
    new = torch.where(c < col_b, table[of], torch.where((c == col_b) & (fill_b > 0), table[home], table))
    at = torch.arange(B, device=DEV)
    src, dst = table[of, col_b[:, 0]].long(), table[home, col_b[:, 0]].long()
    dst = torch.where(fill_b[:, 0] > 0, dst, table[at, col_b[:, 0]].long())
    src = torch.where(fill_b[:, 0] > 0, src, dst)
    live = torch.arange(P, device=DEV).view(1, 1, 1, P, 1) < fill_b.view(1, B, 1, 1, 1)
    for pages in (kp, vp):
        pages[:, dst] = torch.where(live, pages[:, src], pages[:, dst])
    s["block_table"] = new
    return new, kp, vp


def _own_calls():
    path = os.path.join(os.getcwd(), "llm-cuda_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from llm_cuda.kernels import beam_search
    from llm_cuda.kernels.triton import decode_attention

    return decode_attention.shared_prefix_decode_attention, beam_search.beam_select, \
        beam_search.paged_kv_reorder


def run(state):
    s = state
    if own:
        attend, select, reorder = _own_calls()
        if s["op"] == "prefix":
            return attend(s["q"], s["key_pages"], s["value_pages"], s["prefix_table"],
                          s["prefix_lens"], s["block_table"], s["seq_lens"], return_lse=True)
        if s["op"] == "select":
            return select(s["logits"], s["scores"], num_candidates=s["count"],
                          finished=s["finished"], eos_token_id=s["eos"])
        s["block_table"] = reorder(s["key_pages"], s["value_pages"], s["block_table"],
                                   s["seq_lens"], s["parents"])
        return s["block_table"], s["key_pages"], s["value_pages"]
    return {"prefix": _plain_prefix, "select": _plain_select, "reorder": _plain_reorder}[s["op"]](s)


# --------------------------------------------------------------------------
# Work and 64-bit results
# --------------------------------------------------------------------------
def work(case):
    e = SIZES[case["dtype"]]
    if case["op"] == "prefix":
        Hq, Hkv, D, N, W, B, P = _prefix_shape(case)
        # ragged lengths are even from a quarter up: five eighths of the longest on average
        part = lambda count, top: top * (1 + 0.625 * (count - 1)) if case["ragged"] else count * top  # noqa: E731
        shared, mine = part(N, case["prefix"]), part(B, case["ctx"])
        return {"bytes": 2 * Hkv * D * e * (shared + mine) + 2 * B * Hq * D * e + 4 * B * Hq,
                "flops": 4 * Hq * D * (W * shared + mine)}
    if case["op"] == "select":
        rows = case["groups"] * (case["width"] - (0 if case["first"] else case["finished"]))
        return {"bytes": rows * case["vocab"] * e + case["groups"] * case["count"] * 21,
                "flops": 4 * rows * case["vocab"]}
    _, Hkv, D = HEADS[case["heads"]]
    fill, B = case["tokens"] % case["page"], case["groups"] * case["width"]
    copied = case["groups"] * case["childless"] * case["layers"] * 2 * Hkv * fill * D * e
    return {"bytes": 2 * copied + 2 * 4 * B * case["pages"] + 8 * B, "flops": 0}


def _exact_prefix(case, seed):
    s = _prepare_prefix(case, seed)
    Hq, Hkv, D, N, W, B, P = _prefix_shape(case)
    if 8.0 * B * Hq * (case["prefix"] + case["ctx"]) > 12e9:
        return None
    plen, slen = _prefix_lengths(case, seed)
    q, G = s["q"].double()[:, :, 0], Hq // Hkv
    out = torch.zeros(B, Hq, D, dtype=torch.float64, device=DEV)
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64, device=DEV)
    for b in range(B):
        n, lp, ls = b // W, int(plen[b // W]), int(slen[b])
        ids = torch.cat([s["prefix_table"][n, torch.arange(lp, device=DEV) // P],
                         s["block_table"][b, torch.arange(ls, device=DEV) // P]]).long()
        slot = torch.cat([torch.arange(lp, device=DEV) % P, torch.arange(ls, device=DEV) % P])
        if not len(ids):
            continue
        k = s["key_pages"][ids, :, slot].double().permute(1, 0, 2)
        v = s["value_pages"][ids, :, slot].double().permute(1, 0, 2)
        sc = torch.bmm(q[b].view(Hkv, G, D), k.transpose(1, 2).contiguous()) / math.sqrt(D)
        peak = sc.max(-1, keepdim=True).values
        p = (sc - peak).exp()
        out[b] = (torch.bmm(p, v) / p.sum(-1, keepdim=True)).reshape(Hq, D)
        lse[b] = (peak + p.sum(-1, keepdim=True).log()).reshape(Hq)
    return out.unsqueeze(2), lse


def _exact_select(case, seed):
    s = _prepare_select(case, seed)
    N, W, V = s["logits"].shape
    x = s["logits"].double().cpu().numpy()
    scores, done = s["scores"].double().cpu().numpy(), s["finished"].cpu().numpy()
    K = case["count"]
    best = np.empty((N, K))
    tokens, parents, ended = (np.empty((N, K), dtype=t) for t in (np.int64, np.int64, bool))
    for n in range(N):
        value = np.full((W, V), -np.inf)
        for w in range(W):
            if done[n, w]:
                value[w, s["eos"]] = scores[n, w]
                continue
            peak = x[n, w].max()
            if np.isfinite(peak) and np.isfinite(scores[n, w]):
                value[w] = x[n, w] - (peak + np.log(np.exp(x[n, w] - peak).sum())) + scores[n, w]
        value = value.ravel()
        kth = np.partition(value, value.size - K)[value.size - K]
        keep = np.flatnonzero(value > kth)
        keep = np.concatenate([keep, np.flatnonzero(value == kth)[:K - len(keep)]])
        keep = keep[np.lexsort((keep, -value[keep]))]
        best[n], tokens[n], parents[n] = value[keep], keep % V, keep // V
        ended[n] = done[n, parents[n]] | (tokens[n] == s["eos"])
    return best, tokens, parents, ended


def _exact_reorder(case, seed):
    s = _prepare_reorder(case, seed)
    table = s["block_table"].cpu().numpy()
    parents = s["parents"].cpu().numpy()
    N, W, P = case["groups"], case["width"], case["page"]
    col, fill = divmod(case["tokens"], P)
    new, moves = table.copy(), []
    for n in range(N):
        rows = range(n * W, (n + 1) * W)
        spare = [r for r in range(W) if r not in set(parents[n].tolist())]
        seen = set()
        for w, r in enumerate(rows):
            p = int(parents[n, w])
            new[r, :col] = table[n * W + p, :col]
            if fill:
                at = spare.pop(0) if p in seen else p
                new[r, col] = table[n * W + at, col]
                if at != p:
                    moves.append((int(table[n * W + p, col]), int(new[r, col])))
            seen.add(p)
    for pages in (s["key_pages"], s["value_pages"]):
        for a, b in moves:
            pages[:, b, :, :fill] = pages[:, a, :, :fill]
    return torch.from_numpy(new).to(DEV), s["key_pages"].double(), s["value_pages"].double()


def exact(case, seed):
    return {"prefix": _exact_prefix, "select": _exact_select,
            "reorder": _exact_reorder}[case["op"]](case, seed)
