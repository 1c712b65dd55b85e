"""64-bit restatement of the operators of speculative decoding over a pool of pages:
attention of the newest tokens, verification of drafts, page resizing, forking and
compaction. Plain loops on the CPU."""
from __future__ import annotations

import math

import torch

from .beam import _tokens

AGREE = 2.0 ** -32


def paged_extend(q, key_pages, value_pages, block_table, seq_lens, query_lens=None, scale=None):
    """(out [B, Hq, T, D], lse [B, Hq, T], mean absolute value [B, Hq, T, D]) in float64:
    the last is sum_t p_t |v_t|."""
    B, Hq, T, D = q.shape
    pages, Hkv, P, _ = key_pages.shape
    G = Hq // Hkv
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(B, Hq, T, D, dtype=torch.float64)
    size = torch.zeros(B, Hq, T, D, dtype=torch.float64)
    lse = torch.full((B, Hq, T), -math.inf, dtype=torch.float64)
    for b in range(B):
        L = min(max(0, int(seq_lens[b])), block_table.shape[1] * P)
        n = T if query_lens is None else min(max(0, int(query_lens[b])), T)
        for i in range(n):
            seen = L - n + i + 1
            if seen <= 0:
                continue
            k = _tokens(key_pages, block_table[b], seen)
            v = _tokens(value_pages, block_table[b], seen)
            if k.shape[1] == 0:
                continue
            x = torch.matmul(k, q[b, :, i].double().view(Hkv, G, D).transpose(1, 2)) * scale  # [Hkv, t, G]
            m = torch.logsumexp(x, 1)
            p = torch.exp(x - m.unsqueeze(1)).transpose(1, 2)
            out[b, :, i] = torch.matmul(p, v).view(Hq, D)
            size[b, :, i] = torch.matmul(p, v.abs()).view(Hq, D)
            lse[b, :, i] = m.view(Hq)
    return out, lse, size


def distribution(row, temperature):
    """softmax(row / temperature) in float64; all mass on the first largest (NaN largest)
    where that is not finite or the temperature no positive finite number."""
    row = row.double()
    rank = torch.where(row.isnan(), math.inf, row)
    top = rank.max()
    first = int((row.isnan() if row.isnan().any() else rank == top).nonzero()[0])
    if not (0 < temperature < math.inf) or not torch.isfinite(row[first]):
        one = torch.zeros_like(row)
        one[first] = 1
        return one
    e = torch.exp((row - top) / temperature)
    return e / e.sum()


def verify_draft(logits, draft_tokens, uniforms, draft_logits=None, draft_lens=None, temperature=1.0):
    """(tokens int64 [B, K + 1], accepted int32 [B], close, near): how far, relatively, the
    closest of the accepting comparisons was from its other outcome, and the random number
    from a border of the new token's running sum."""
    B, T, V = logits.shape
    K = T - 1
    tokens = torch.full((B, T), -1, dtype=torch.int64)
    accepted = torch.zeros(B, dtype=torch.int32)
    close = near = math.inf
    for b in range(B):
        t = float(temperature[b]) if isinstance(temperature, torch.Tensor) else float(temperature)
        n = K if draft_lens is None else min(max(0, int(draft_lens[b])), K)
        i = 0
        while True:
            p = w = distribution(logits[b, i], t)
            if i == n:
                break
            d = int(draft_tokens[b, i])
            inside = 0 <= d < V
            if draft_logits is None:
                q = torch.zeros(V, dtype=torch.float64)
                if inside:
                    q[d] = 1
            else:
                q = distribution(draft_logits[b, i], t)
            left = float(uniforms[b, i]) * (float(q[d]) if inside else (1.0 if draft_logits is None else 0.0))
            right = float(p[d]) if inside else 0.0
            if left != right:
                close = min(close, abs(left - right) / max(left, right))
            if not left < right:
                rest = (p - q).clamp(min=0)
                w = rest if rest.sum() >= AGREE else p
                break
            tokens[b, i] = d
            i += 1
        accepted[b] = i
        run = torch.cumsum(w, 0)
        at = float(uniforms[b, K]) * float(run[-1])
        v = min(int((run <= at).sum()), int(w.nonzero()[-1]))
        near = min(near, ((run[w > 0] - at).abs().min() / run[-1]).item())
        tokens[b, i] = v
    return tokens, accepted, close, near


def _length(n, table, P):
    return min(max(0, int(n)), table.shape[1] * P)


class _Pool:
    def __init__(self, key_pages, value_pages, page_refs):
        self.kp, self.vp, self.old = key_pages.clone(), value_pages.clone(), page_refs.tolist()
        self.refs = list(self.old)
        self.N = len(self.old)
        self.free = [p for p in range(self.N) if self.old[p] == 0]
        self.missing = 0

    def add(self, page, n):
        if 0 <= page < self.N:
            self.refs[page] += n

    def take(self):
        if not self.free:
            self.missing += 1
            return -1
        self.refs[self.free[0]] += 1
        return self.free.pop(0)

    def copy(self, src, dst, slots, kp, vp):
        if 0 <= src < self.N and 0 <= dst < self.N:
            for new, was in ((self.kp, kp), (self.vp, vp)):
                new[..., dst, :, :slots, :] = was[..., src, :, :slots, :]

    def counts(self):
        return torch.tensor(self.refs, dtype=torch.int32).view(self.N)


def kv_resize(key_pages, value_pages, block_table, seq_lens, new_lens, page_refs):
    """(block_table, page_refs, missing, key_pages, value_pages) after the resize."""
    P, (B, M) = key_pages.shape[-2], block_table.shape
    pool = _Pool(key_pages, value_pages, page_refs)
    new = torch.full((B, M), -1, dtype=torch.int32)
    for b in range(B):
        n, m = _length(seq_lens[b], block_table, P), _length(new_lens[b], block_table, P)
        held, want = -(-n // P), -(-m // P)
        for c in range(M):
            page = int(block_table[b, c])
            if held <= c < want:
                new[b, c] = pool.take()
            elif c < min(held, want):
                shared = m > n and n % P and c == held - 1 and 0 <= page < pool.N and pool.old[page] > 1
                if shared:
                    pool.add(page, -1)
                    new[b, c] = pool.take()
                    pool.copy(page, int(new[b, c]), n % P, key_pages, value_pages)
                else:
                    new[b, c] = page
            elif c < held:
                pool.add(page, -1)
    return new, pool.counts(), torch.tensor([pool.missing], dtype=torch.int32), pool.kp, pool.vp


def kv_fork(key_pages, value_pages, block_table, seq_lens, parents, page_refs):
    """(block_table, seq_lens, page_refs, missing, key_pages, value_pages) after the fork."""
    P, (B, M) = key_pages.shape[-2], block_table.shape
    pool = _Pool(key_pages, value_pages, page_refs)
    R = parents.shape[0]
    new = torch.full((R, M), -1, dtype=torch.int32)
    lens = torch.zeros(R, dtype=torch.int32)
    for b in range(B):
        for c in range(-(-_length(seq_lens[b], block_table, P) // P)):
            pool.add(int(block_table[b, c]), -1)
    seen = set()
    for r, p in enumerate(parents.tolist()):
        if not 0 <= p < B:
            continue
        n = _length(seq_lens[p], block_table, P)
        lens[r] = n
        for c in range(-(-n // P)):
            page = int(block_table[p, c])
            if c == n // P and p in seen and 0 <= page < pool.N:
                new[r, c] = pool.take()
                pool.copy(page, int(new[r, c]), n % P, key_pages, value_pages)
            else:
                new[r, c] = page
                pool.add(page, 1)
        seen.add(p)
    return new, lens, pool.counts(), torch.tensor([pool.missing], dtype=torch.int32), pool.kp, pool.vp


def kv_compact(key_pages, value_pages, block_table, seq_lens, page_refs):
    """(block_table, page_refs, page_map, key_pages, value_pages) after the compaction."""
    P, (B, M) = key_pages.shape[-2], block_table.shape
    pool = _Pool(key_pages, value_pages, page_refs)
    N, n = pool.N, pool.N - len(pool.free)
    where = [p if pool.old[p] else -1 for p in range(N)]
    for p in range(n, N):
        if pool.old[p]:
            where[p] = pool.free.pop(0)
            pool.copy(p, where[p], P, key_pages, value_pages)
    refs = [0] * N
    for p in range(N):
        if pool.old[p]:
            refs[where[p]] = pool.old[p]
    pool.refs = refs
    new = torch.full((B, M), -1, dtype=torch.int32)
    for b in range(B):
        for c in range(-(-_length(seq_lens[b], block_table, P) // P)):
            page = int(block_table[b, c])
            new[b, c] = where[page] if 0 <= page < N else page
    return new, pool.counts(), torch.tensor(where, dtype=torch.int32).view(N), pool.kp, pool.vp
