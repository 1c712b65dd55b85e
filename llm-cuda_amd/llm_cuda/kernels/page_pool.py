"""Pages of a pool that sequences take, share and give back (no counterpart in the
reference, whose cache owns fixed pages: models/llama3/kv_cache.py:21-36).

page_refs counts the block-table entries that name each page; a page with 0 is free.

* `paged_kv_resize`: sequences grow (the lowest free pages) or shrink; a shared page
  that a sequence is about to write into is copied first.
* `paged_kv_fork`: the batch becomes continuations of its rows: samples of a prompt
  share its whole pages, rows that ended leave and give up theirs.
* `paged_kv_compact`: the pages in use move to the front of the pool.

Each returns a new table and new counts and changes nothing that the old ones name.
`llm_cuda.models.llama3.kv_cache.PooledKVCache` is a cache over such a pool.
"""
from __future__ import annotations

from llm_cuda.kernels._ops import paged_kv_compact, paged_kv_fork, paged_kv_resize

__all__ = ["paged_kv_compact", "paged_kv_fork", "paged_kv_resize"]
