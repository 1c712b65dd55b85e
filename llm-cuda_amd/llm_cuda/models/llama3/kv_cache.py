"""Paged KV cache with a real block table (reference: models/llama3/kv_cache.py:1-125).

Layout (unchanged from the reference): per layer, `key_pages` and
`value_pages` are pools [num_pages, n_kv_heads, page_size, head_dim] in the
model dtype; token t of a sequence lives in page t // page_size, slot
t % page_size of that sequence's pages. What changes:
  * `block_table` (int32 [batch, max_pages]) maps each sequence's logical page
    to a physical page of the pool. The default table gives sequence b the
    pages b*max_pages .. (b+1)*max_pages - 1, so for batch 1 logical page i IS
    physical page i, the reference's identity mapping (kv_cache.py:55-57).
  * batch > 1 and per-sequence lengths (`seq_lens`, int32 [batch] on the
    device, mirrored on the host in `lengths`).
  * `append` is one HIP scatter launch (lc_paged_kv_append) instead of a Python
    loop of 2*seq slice copies; `get_kv` is one HIP gather (lc_paged_kv_gather)
    instead of a torch.cat of pages. The decode path does not call get_kv at
    all: it reads the pools in place (paged_decode_attention).

`BeamKVCache` is the cache of a beam search, `PooledKVCache` one whose sequences take,
share and give back pages of a pool (no counterparts in the reference).
"""
from __future__ import annotations

import math

import torch

from llm_cuda.kernels import _ops


class PagedKVLayerCache:
    def __init__(
        self,
        num_kv_heads: int,
        head_dim: int,
        max_seq_len: int,
        page_size: int,
        device: torch.device,
        dtype: torch.dtype,
        batch_size: int = 1,
        block_table: torch.Tensor | None = None,
        num_pages: int | None = None,
        seq_lens: torch.Tensor | None = None,
    ):
        if page_size <= 0:
            raise ValueError("page_size must be > 0")
        if max_seq_len <= 0:
            raise ValueError("max_seq_len must be > 0")
        if batch_size <= 0:
            raise ValueError("batch_size must be > 0")

        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.max_seq_len = max_seq_len
        self.page_size = page_size
        self.batch_size = batch_size
        self.max_pages = math.ceil(max_seq_len / page_size)
        device = torch.device(device)

        if block_table is None:
            pool = batch_size * self.max_pages if num_pages is None else num_pages
            if pool < batch_size * self.max_pages:
                raise ValueError("num_pages too small for the default block table")
            block_table = torch.arange(
                batch_size * self.max_pages, dtype=torch.int32, device=device
            ).view(batch_size, self.max_pages)
        else:
            if block_table.dtype != torch.int32 or block_table.shape != (batch_size, self.max_pages):
                raise ValueError(
                    f"block_table must be int32 [{batch_size}, {self.max_pages}]")
            block_table = block_table.to(device).contiguous()
            pool = int(block_table.max().item()) + 1 if num_pages is None else num_pages
        self.num_pages = pool
        self.block_table = block_table

        self.key_pages = torch.empty(
            pool, num_kv_heads, page_size, head_dim, device=device, dtype=dtype)
        self.value_pages = torch.empty_like(self.key_pages)
        if seq_lens is None:
            seq_lens = torch.zeros(batch_size, dtype=torch.int32, device=device)
        elif (seq_lens.dtype != torch.int32 or seq_lens.shape != (batch_size,)
              or seq_lens.device != device):
            raise ValueError(f"seq_lens must be int32 [{batch_size}] on {device}")
        else:
            seq_lens.zero_()
        self.seq_lens = seq_lens
        self.lengths = [0] * batch_size
        # Zeroed scratch of the fused decode step (it leaves the counters at zero).
        self.step_counters = torch.zeros(batch_size, dtype=torch.int32, device=device)

    @property
    def length(self) -> int:
        """Cached tokens per sequence (all sequences advance together in `append`)."""
        first = self.lengths[0]
        if any(n != first for n in self.lengths):
            raise ValueError("sequences have different lengths; use `lengths`")
        return first

    @property
    def uniform_length(self) -> int | None:
        """The common number of cached tokens when every sequence holds the
        same number (host mirror), else None."""
        first = self.lengths[0]
        return first if all(n == first for n in self.lengths) else None

    def append(self, k: torch.Tensor, v: torch.Tensor) -> None:
        if k.shape != v.shape:
            raise ValueError("k and v shapes must match")
        if k.dim() != 4:
            raise ValueError("Expected k/v shape [batch, kv_heads, seq, head_dim]")
        if k.shape[0] != self.batch_size:
            raise ValueError(
                f"batch {k.shape[0]} does not match the cache batch size {self.batch_size}")
        if k.shape[1] != self.num_kv_heads or k.shape[3] != self.head_dim:
            raise ValueError("k/v shapes do not match cache layout")
        seq = k.shape[2]
        if max(self.lengths) + seq > self.max_seq_len:
            raise ValueError("Appending would exceed max_seq_len")
        if seq == 0:
            return
        _ops.kv_append(k, v, self.key_pages, self.value_pages, self.block_table, self.seq_lens)
        self.seq_lens.add_(seq)
        self.lengths = [n + seq for n in self.lengths]

    def append_rotated(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                       cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
        """Decode-time fusion of RoPE and `append`: rotates q and k at the
        positions seq_lens[b] + s, appends the rotated k and v, and returns the
        rotated q. cos/sin are full tables indexed by position that cover
        max_pages * page_size positions."""
        if k.shape != v.shape or k.dim() != 4 or q.dim() != 4:
            raise ValueError("Expected q, k, v of shape [batch, heads, seq, head_dim]")
        if k.shape[0] != self.batch_size or q.shape[0] != self.batch_size:
            raise ValueError(
                f"batch {k.shape[0]} does not match the cache batch size {self.batch_size}")
        if k.shape[1] != self.num_kv_heads or k.shape[3] != self.head_dim:
            raise ValueError("k/v shapes do not match cache layout")
        seq = k.shape[2]
        if max(self.lengths) + seq > self.max_seq_len:
            raise ValueError("Appending would exceed max_seq_len")
        q_rot = _ops.rope_kv_append(q, k, v, cos, sin, self.key_pages, self.value_pages,
                                    self.block_table, self.seq_lens)
        self.lengths = [n + seq for n in self.lengths]
        return q_rot

    def can_fuse_decode_step(self, n_heads: int, dtype: torch.dtype) -> bool:
        """Whether `decode_step` takes this cache: equal lengths, a head layout
        whose (sequence, kv head, head group) units fill whole rounds of the
        CUs, and sizes the fused kernel supports (its single split must be
        the split the decode heuristic would choose)."""
        capacity = self.max_pages * self.page_size
        length = self.uniform_length
        if not (length is not None and self.key_pages.is_cuda
                and _ops.decode_step_supported(dtype, self.head_dim, self.page_size, capacity)):
            return False
        group = n_heads // self.num_kv_heads
        split = _ops.choose_split_tokens(
            self.batch_size, self.num_kv_heads, group, capacity, self.page_size, self.head_dim,
            length + 1, _ops._cu_count(self.key_pages.device))
        return split >= capacity

    def decode_step(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor,
                    sin: torch.Tensor, attention_mask: torch.Tensor | None = None,
                    return_lse: bool = False):
        """One decode step of attention in one launch: RoPE of q and k at the
        positions seq_lens[b], the append of the rotated k and v, and attention
        of the rotated q over the cache including the new token. Advances the
        lengths by one and returns out [B, Hq, 1, D] (and the fp32 lse [B, Hq]
        if return_lse). cos/sin are full tables indexed by position covering
        max_pages * page_size positions."""
        if k.shape != v.shape or k.dim() != 4 or q.dim() != 4 or k.shape[2] != 1:
            raise ValueError("Expected q [batch, heads, 1, head_dim] and k, v [batch, kv_heads, "
                             "1, head_dim]")
        if k.shape[0] != self.batch_size or q.shape[0] != self.batch_size:
            raise ValueError(
                f"batch {k.shape[0]} does not match the cache batch size {self.batch_size}")
        if k.shape[1] != self.num_kv_heads or k.shape[3] != self.head_dim:
            raise ValueError("k/v shapes do not match cache layout")
        if max(self.lengths) + 1 > self.max_seq_len:
            raise ValueError("Appending would exceed max_seq_len")
        res = _ops.paged_decode_step(q, k, v, cos, sin, self.key_pages, self.value_pages,
                                     self.block_table, self.seq_lens, self.step_counters,
                                     attention_mask=attention_mask, return_lse=return_lse)
        self.lengths = [n + 1 for n in self.lengths]
        return res

    def get_kv(self) -> tuple[torch.Tensor, torch.Tensor]:
        length = self.length
        if length == 0:
            empty = self.key_pages.new_empty(
                (self.batch_size, self.num_kv_heads, 0, self.head_dim))
            return empty, empty
        return _ops.kv_gather(self.key_pages, self.value_pages, self.block_table, length)

    def clear(self) -> None:
        self.lengths = [0] * self.batch_size
        self.seq_lens.zero_()


class PagedKVCache:
    def __init__(self, layer_caches: list[PagedKVLayerCache],
                 seq_lens_all: torch.Tensor | None = None):
        if not layer_caches:
            raise ValueError("layer_caches must not be empty")
        self.layer_caches = layer_caches
        # [num_layers, batch] int32 whose rows are the layers' seq_lens when the
        # cache was made by create(): one fill resets every layer's lengths.
        self.seq_lens_all = seq_lens_all

    @classmethod
    def create(
        cls,
        num_layers: int,
        num_kv_heads: int,
        head_dim: int,
        max_seq_len: int,
        page_size: int,
        device: torch.device,
        dtype: torch.dtype,
        batch_size: int = 1,
        block_table: torch.Tensor | None = None,
        num_pages: int | None = None,
    ) -> "PagedKVCache":
        device = torch.device(device)
        lens = torch.zeros(num_layers, batch_size, dtype=torch.int32, device=device)
        return cls(
            [
                PagedKVLayerCache(
                    num_kv_heads=num_kv_heads,
                    head_dim=head_dim,
                    max_seq_len=max_seq_len,
                    page_size=page_size,
                    device=device,
                    dtype=dtype,
                    batch_size=batch_size,
                    block_table=block_table,
                    num_pages=num_pages,
                    seq_lens=lens[i],
                )
                for i in range(num_layers)
            ],
            seq_lens_all=lens,
        )

    def get_layer(self, layer_idx: int) -> PagedKVLayerCache:
        return self.layer_caches[layer_idx]

    def clear(self) -> None:
        for layer in self.layer_caches:
            layer.clear()


class BeamKVLayerCache:
    """One layer of a BeamKVCache: views of its pools, tables and lengths."""

    def __init__(self, cache: "BeamKVCache", layer: int):
        self.cache = cache
        self.key_pages = cache.key_pages[layer]
        self.value_pages = cache.value_pages[layer]
        self.prefix_lens = cache.prefix_lens_all[layer]
        self.seq_lens = cache.seq_lens_all[layer]
        self.prefix_length = 0  # host mirrors of the (equal) lengths
        self.length = 0

    def append_prompt(self, k: torch.Tensor, v: torch.Tensor) -> None:
        """The prompts' (rotated) keys and values, [groups, kv_heads, seq, head_dim]."""
        c = self.cache
        if k.shape != v.shape or k.dim() != 4 or k.shape[0] != c.groups:
            raise ValueError(f"expected k and v of {c.groups} prompts, [groups, kv_heads, seq, "
                             f"head_dim]; got {tuple(k.shape)} and {tuple(v.shape)}")
        if self.prefix_length:
            raise ValueError("the cache already holds its prompts")
        if k.shape[2] > c.max_prefix_len:
            raise ValueError("the prompts exceed max_prefix_len")
        _ops.kv_append(k, v, self.key_pages, self.value_pages, c.prefix_table, self.prefix_lens)
        self.prefix_lens.add_(k.shape[2])
        self.prefix_length = k.shape[2]

    def append_rotated(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                       cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
        """Rotates every beam's q and k of one token, appends k and v to the beam's own
        tokens and returns the rotated q. cos/sin: tables by position."""
        c = self.cache
        if k.shape != v.shape or k.dim() != 4 or k.shape[0] != c.batch_size or k.shape[2] != 1:
            raise ValueError(f"expected one token of {c.batch_size} beams, [beams, kv_heads, 1, "
                             f"head_dim]; got {tuple(k.shape)} and {tuple(v.shape)}")
        if self.length + 1 > c.max_new_len:
            raise ValueError("Appending would exceed max_new_len")
        # The kernel places a token by its beam's own length; its position follows the
        # prompt's, so the tables start there.
        rows = c.block_table.shape[1] * c.page_size
        at = slice(self.prefix_length, self.prefix_length + rows)
        q = _ops.rope_kv_append(q, k, v, cos[at], sin[at], self.key_pages, self.value_pages,
                                c.block_table, self.seq_lens)
        self.length += 1
        return q

    def attend(self, q: torch.Tensor) -> torch.Tensor:
        """Attention of q [beams, heads, 1, head_dim] over prompt and own tokens."""
        c = self.cache
        return _ops.shared_prefix_decode(q, self.key_pages, self.value_pages, c.prefix_table,
                                         self.prefix_lens, c.block_table, self.seq_lens)


class BeamKVCache:
    """The paged cache of a beam search: `groups` prompts of equal length, `width` beams
    each. A prompt's pages are stored once for all of its beams (prefix_table); a beam's
    own tokens are in pages named by block_table, whole pages of which beams share after
    a `reorder`. The layers' pools are one tensor [layers, pages, kv_heads, page_size,
    head_dim], which share both tables."""

    def __init__(self, num_layers: int, num_kv_heads: int, head_dim: int, groups: int, width: int,
                 max_prefix_len: int, max_new_len: int, page_size: int, device: torch.device,
                 dtype: torch.dtype):
        if min(num_layers, groups, width, max_prefix_len, max_new_len, page_size) <= 0:
            raise ValueError("layers, groups, width, lengths and page_size must be > 0")
        device = torch.device(device)
        self.groups, self.width, self.batch_size = groups, width, groups * width
        self.max_prefix_len, self.max_new_len, self.page_size = (max_prefix_len, max_new_len,
                                                                 page_size)
        prefix_pages = math.ceil(max_prefix_len / page_size)
        own_pages = math.ceil(max_new_len / page_size)
        shared = groups * prefix_pages
        pool = shared + self.batch_size * own_pages
        pages = torch.arange(pool, dtype=torch.int32, device=device)
        self.prefix_table = pages[:shared].view(groups, prefix_pages)
        self.block_table = pages[shared:].view(self.batch_size, own_pages)
        self.key_pages = torch.empty(num_layers, pool, num_kv_heads, page_size, head_dim,
                                     device=device, dtype=dtype)
        self.value_pages = torch.empty_like(self.key_pages)
        self.prefix_lens_all = torch.zeros(num_layers, groups, dtype=torch.int32, device=device)
        self.seq_lens_all = torch.zeros(num_layers, self.batch_size, dtype=torch.int32,
                                        device=device)
        self.layer_caches = [BeamKVLayerCache(self, i) for i in range(num_layers)]

    def get_layer(self, layer_idx: int) -> BeamKVLayerCache:
        return self.layer_caches[layer_idx]

    def reorder(self, parents: torch.Tensor) -> None:
        """Beam w of prompt n continues what its beam parents[n, w] (int64) holds."""
        if tuple(parents.shape) != (self.groups, self.width):
            raise ValueError(f"parents must be {(self.groups, self.width)}, got "
                             f"{tuple(parents.shape)}")
        self.block_table.copy_(_ops.paged_kv_reorder(
            self.key_pages, self.value_pages, self.block_table, self.seq_lens_all[0], parents))


class PooledKVLayerCache:
    """One layer of a PooledKVCache: views of its pools and lengths."""

    def __init__(self, cache: "PooledKVCache", layer: int):
        self.cache = cache
        self.layer = layer
        self.key_pages = cache.key_pages[layer]
        self.value_pages = cache.value_pages[layer]

    @property
    def seq_lens(self) -> torch.Tensor:
        return self.cache.seq_lens_all[self.layer]

    @property
    def empty(self) -> bool:
        return self.cache.longest == 0

    def _check(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> None:
        c = self.cache
        if k.shape != v.shape or k.dim() != 4 or k.shape[0] != c.batch_size:
            raise ValueError(f"expected k and v of {c.batch_size} sequences, [batch, kv_heads, "
                             f"seq, head_dim]; got {tuple(k.shape)} and {tuple(v.shape)}")
        if k.shape[2] != c.reserved:
            raise ValueError(f"{k.shape[2]} tokens, {c.reserved} reserved")

    def append_prompt(self, k: torch.Tensor, v: torch.Tensor) -> None:
        """The prompts' (rotated) keys and values, into empty sequences."""
        self._check(k, k, v)
        _ops.kv_append(k, v, self.key_pages, self.value_pages, self.cache.block_table,
                       self.seq_lens)
        self.seq_lens.add_(k.shape[2])
        self.cache.appended(self.layer, k.shape[2])

    def append_rotated(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                       cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
        """Rotates q and k at the sequences' own next positions, appends k and v and returns
        the rotated q. cos/sin: tables by position that cover the capacity."""
        self._check(q, k, v)
        q = _ops.rope_kv_append(q, k, v, cos, sin, self.key_pages, self.value_pages,
                                self.cache.block_table, self.seq_lens)
        self.cache.appended(self.layer, k.shape[2])
        return q

    def attend(self, q: torch.Tensor) -> torch.Tensor:
        """Attention of the newest tokens' q [batch, heads, tokens, head_dim]."""
        return _ops.paged_extend(q, self.key_pages, self.value_pages, self.cache.block_table,
                                 self.seq_lens)


class PooledKVCache:
    """A paged cache whose sequences take pages of one pool as they grow, share them after
    a fork and give them back. Lengths are the sequences' own (on the device).

    A step is `reserve(n)`, then the layers append n tokens each; `truncate` gives the last
    ones back, `fork` makes the batch continuations of its sequences, `compact` moves the
    pages in use to the front. The pools are one tensor [layers, pages, kv_heads, page_size,
    head_dim] with one block table; page_refs counts the entries that name a page.

    num_pages: by default what `batch_size` sequences of max_seq_len tokens can ever ask for.
    With fewer, and while a fork has made more than `batch_size` sequences, `reserve` and `fork`
    wait for the GPU and raise where pages are missing (the cache stays as it was).
    """

    def __init__(self, num_layers: int, num_kv_heads: int, head_dim: int, max_seq_len: int,
                 page_size: int, device: torch.device, dtype: torch.dtype, batch_size: int = 1,
                 num_pages: int | None = None):
        if min(num_layers, max_seq_len, page_size, batch_size) <= 0:
            raise ValueError("layers, max_seq_len, page_size and batch_size must be > 0")
        if num_pages is not None and num_pages <= 0:
            raise ValueError("num_pages must be > 0")
        device = torch.device(device)
        self.max_seq_len, self.page_size = max_seq_len, page_size
        self.batch_size = batch_size
        self.max_pages = math.ceil(max_seq_len / page_size)
        # (a sequence that writes into a shared page holds that page and its own for a moment)
        self._enough = (self.max_pages + 1) * batch_size
        self.num_pages = self._enough if num_pages is None else num_pages
        self._rows = batch_size  # of which the pool is known to be large enough
        self.key_pages = torch.empty(num_layers, self.num_pages, num_kv_heads, page_size, head_dim,
                                     device=device, dtype=dtype)
        self.value_pages = torch.empty_like(self.key_pages)
        self.block_table = torch.full((batch_size, self.max_pages), -1, dtype=torch.int32,
                                      device=device)
        self.page_refs = torch.zeros(self.num_pages, dtype=torch.int32, device=device)
        self.seq_lens_all = torch.zeros(num_layers, batch_size, dtype=torch.int32, device=device)
        self.longest = 0  # host side: no sequence holds more tokens
        self.reserved = 0  # tokens of every sequence that pages are held for, not appended yet
        self.layer_caches = [PooledKVLayerCache(self, i) for i in range(num_layers)]

    def get_layer(self, layer_idx: int) -> PooledKVLayerCache:
        return self.layer_caches[layer_idx]

    @property
    def seq_lens(self) -> torch.Tensor:
        """Tokens of every sequence, int32 [batch]."""
        return self.seq_lens_all[0]

    def pages_in_use(self) -> int:
        return int((self.page_refs != 0).sum())

    def _check_missing(self, missing: torch.Tensor, rows: int) -> None:
        if self.num_pages < self._enough or rows > self._rows:
            short = int(missing)
            if short:
                raise RuntimeError(f"the pool of {self.num_pages} pages is {short} short")

    def reserve(self, tokens: int) -> None:
        """Pages for `tokens` more tokens of every sequence."""
        if self.reserved:
            raise ValueError(f"{self.reserved} reserved tokens are not appended yet")
        if tokens <= 0 or self.longest + tokens > self.max_seq_len:
            raise ValueError(f"{tokens} tokens beside up to {self.longest} exceed max_seq_len")
        table, refs, missing = _ops.paged_kv_resize(
            self.key_pages, self.value_pages, self.block_table, self.seq_lens,
            self.seq_lens + tokens, self.page_refs)
        self._check_missing(missing, self.batch_size)
        self.block_table, self.page_refs, self.reserved = table, refs, tokens

    def appended(self, layer: int, tokens: int) -> None:
        """A layer has appended the `tokens` reserved tokens."""
        if layer == len(self.layer_caches) - 1:
            self.longest += tokens
            self.reserved = 0

    def truncate(self, new_lens: torch.Tensor, longest: int) -> None:
        """Sequences keep their first new_lens (int32 [batch]) tokens at most; `longest`, known
        on the host: none is longer."""
        if self.reserved:
            raise ValueError(f"{self.reserved} reserved tokens are not appended yet")
        new_lens = torch.minimum(new_lens, self.seq_lens)
        self.block_table, self.page_refs, _ = _ops.paged_kv_resize(
            self.key_pages, self.value_pages, self.block_table, self.seq_lens, new_lens,
            self.page_refs)
        self.seq_lens_all.copy_(new_lens.clamp(min=0).expand_as(self.seq_lens_all))
        self.longest = min(self.longest, max(longest, 0))

    def fork(self, parents: torch.Tensor) -> None:
        """The batch becomes the continuations of sequences parents (int64 [rows])."""
        if self.reserved:
            raise ValueError(f"{self.reserved} reserved tokens are not appended yet")
        table, lens, refs, missing = _ops.paged_kv_fork(
            self.key_pages, self.value_pages, self.block_table, self.seq_lens, parents,
            self.page_refs)
        rows = parents.shape[0]
        # (the old rows hold their pages until the new ones have theirs)
        self._check_missing(missing, max(rows, self.batch_size))
        self.block_table, self.page_refs, self.batch_size = table, refs, rows
        self.seq_lens_all = lens.repeat(len(self.layer_caches), 1)

    def compact(self) -> torch.Tensor:
        """The pages in use move to the front of the pool; returns each page's new index (int32
        [num_pages], -1 for a free one)."""
        if self.reserved:
            raise ValueError(f"{self.reserved} reserved tokens are not appended yet")
        self.block_table, self.page_refs, page_map = _ops.paged_kv_compact(
            self.key_pages, self.value_pages, self.block_table, self.seq_lens, self.page_refs)
        return page_map
