"""Beam search over the paged KV cache (no counterpart in the reference, which
decodes greedily: models/llama3/model.py:200-218).

* `beam_select(logits, scores)`: the best continuations of each prompt's beams
  over beams and vocabulary, from one pass over the logits.
* `paged_kv_reorder(key_pages, value_pages, block_table, seq_lens, parents)`: the
  caches follow the selected beams; whole pages are shared through the block
  table, only the page being filled is copied, and only where a beam has several
  children.

The beams' attention is
`llm_cuda.kernels.triton.decode_attention.shared_prefix_decode_attention`: the
prompt's tokens are computed once for all of its beams.
`Llama3ForCausalLM.beam_search` runs the three for every token.
"""
from __future__ import annotations

from llm_cuda.kernels._ops import beam_select, paged_kv_reorder

__all__ = ["beam_select", "paged_kv_reorder"]
