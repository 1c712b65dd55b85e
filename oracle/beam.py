"""64-bit restatement of the beam-search operators: attention of sequences that
share a prefix, selection over beams and vocabulary, cache reordering."""
from __future__ import annotations

import math

import torch


def _tokens(pages: torch.Tensor, row: torch.Tensor, length: int) -> torch.Tensor:
    """The valid tokens of a table row, [kv heads, tokens, dim] in float64."""
    num_pages, _, P, _ = pages.shape
    got = [pages[int(row[t // P]), :, t % P] for t in range(min(length, row.numel() * P))
           if 0 <= int(row[t // P]) < num_pages]
    if not got:
        return pages.new_zeros((pages.shape[1], 0, pages.shape[3]), dtype=torch.float64)
    return torch.stack(got, dim=1).double()


def shared_prefix_decode(q, key_pages, value_pages, prefix_table, prefix_lens, block_table,
                         seq_lens, scale=None):
    """out [B, Hq, D] and lse [B, Hq], float64, on the CPU; sequence by sequence over
    the concatenation of its group's prefix and its own tokens."""
    B, Hq, D = q.shape[0], q.shape[1], q.shape[-1]
    N, Hkv = prefix_table.shape[0], key_pages.shape[1]
    G = Hq // Hkv
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(B, Hq, D, dtype=torch.float64)
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64)
    W = B // N if N else 0
    shared = [[_tokens(p, prefix_table[n], max(0, int(prefix_lens[n])))
               for p in (key_pages, value_pages)] for n in range(N)]
    for b in range(B):
        k, v = (torch.cat([shared[b // W][i], _tokens(p, block_table[b], max(0, int(seq_lens[b])))],
                          dim=1) for i, p in enumerate((key_pages, value_pages)))
        if k.shape[1] == 0:
            continue
        for h in range(Hq):
            s = (k[h // G] @ q[b].reshape(Hq, D)[h].double()) * scale
            lse[b, h] = torch.logsumexp(s, 0)
            out[b, h] = torch.exp(s - lse[b, h]) @ v[h // G]
    return out, lse


def beam_select(logits, scores, count, finished=None, eos=None):
    """(scores float64, tokens, parents, finished or None) by the definition, on the CPU."""
    N, W, V = logits.shape
    x, s = logits.double(), scores.double()
    bad = ~(x < math.inf).all(-1) | ~(s < math.inf)  # NaN or +inf
    empty = torch.isneginf(x).all(-1) | torch.isneginf(s)
    below = x - x.nan_to_num(0.0, 0.0, -math.inf).amax(-1, keepdim=True)
    lse = torch.logsumexp(below.nan_to_num(0.0, 0.0, -math.inf), -1, keepdim=True)
    value = s.unsqueeze(-1) + (below - lse)
    value = torch.where(empty.unsqueeze(-1), torch.full_like(value, -math.inf), value)
    value = torch.where(bad.unsqueeze(-1), torch.full_like(value, math.nan), value)
    if finished is not None:
        only = torch.full((V,), -math.inf, dtype=torch.float64)
        for n, w in finished.nonzero().tolist():
            value[n, w] = only
            value[n, w, eos] = s[n, w]
    flat = value.reshape(N, W * V)
    rank = flat.nan_to_num(math.inf, math.inf, -math.inf) + torch.zeros_like(flat)
    at = torch.stack([torch.tensor(sorted(range(W * V), key=lambda i: (-r[i], i))[:count],
                                   dtype=torch.int64) for r in rank.tolist()])
    parents, tokens = at // V, at % V
    done = None
    if finished is not None:
        done = torch.gather(finished, 1, parents) | (tokens == eos)
    return torch.gather(flat, 1, at), tokens, parents, done


def kv_reorder(key_pages, value_pages, block_table, seq_lens, parents):
    """(key_pages, value_pages, block_table) after the reordering, as new tensors."""
    kp, vp, new = key_pages.clone(), value_pages.clone(), block_table.clone()
    N, W = parents.shape
    P, M = key_pages.shape[-2], block_table.shape[1]
    for n in range(N):
        t = min(max(int(seq_lens[n * W]), 0), M * P)
        col, fill = divmod(t, P)
        par = [p if 0 <= p < W else w for w, p in enumerate(parents[n].tolist())]
        spare = [w for w in range(W) if w not in par]
        seen = set()
        for w, p in enumerate(par):
            row, old = new[n * W + w], block_table[n * W:(n + 1) * W]
            row[:col] = old[p, :col]
            if fill:
                home = spare.pop(0) if p in seen else p
                row[col] = old[home, col]
                src, dst = int(old[p, col]), int(old[home, col])
                N_pages = key_pages.shape[-4]
                if home != p and 0 <= src < N_pages and 0 <= dst < N_pages:
                    for new_pool, pool in ((kp, key_pages), (vp, value_pages)):
                        new_pool[..., dst, :, :fill, :] = pool[..., src, :, :fill, :]
            seen.add(p)
    return kp, vp, new


def beam_search(state, cfg, input_ids, width, max_new_tokens, eos=None):
    """(ids [N, width, S + n], scores [N, width] float64, smallest gap between a kept and a
    dropped candidate) by full recomputation of every beam at every step."""
    from .model import forward

    N, S = input_ids.shape
    ids = input_ids.cpu().unsqueeze(1)
    scores = torch.zeros(N, 1, dtype=torch.float64)
    done = None if eos is None else torch.zeros(N, 1, dtype=torch.bool)
    gap = math.inf
    for _ in range(max_new_tokens):
        n, w, length = ids.shape
        logits = forward(state, cfg, ids.reshape(n * w, length))[:, -1].view(n, w, -1)
        count = min(width + 1, w * logits.shape[-1])
        best, tokens, parents, fin = beam_select(logits, scores, count, done, eos)
        if count > width:
            gap = min(gap, (best[:, :-1] - best[:, 1:]).min().item())
        scores, tokens, parents = best[:, :width], tokens[:, :width], parents[:, :width]
        done = None if fin is None else fin[:, :width]
        ids = torch.cat([torch.gather(ids, 1, parents.unsqueeze(-1).expand(-1, -1, length)),
                         tokens.unsqueeze(-1)], dim=2)
    return ids, scores, gap
