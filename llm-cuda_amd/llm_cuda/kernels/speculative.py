"""Speculative decoding (no counterpart in the reference, which decodes greedily, a
token a step: models/llama3/model.py:200-218).

* `verify_draft_tokens(logits, draft_tokens, uniforms, draft_logits)`: which of every
  sequence's drafted tokens stand, and the token after them, distributed as the
  target's own, from given random numbers. Without drafts it samples.

The target's logits of all drafted places come from one step whose attention is
`llm_cuda.kernels.triton.decode_attention.paged_extend_attention`; the pages of sequences
whose lengths go up by the drafts and down by the refused ones are those of
`llm_cuda.kernels.page_pool`. `Llama3ForCausalLM.speculative_generate` runs them.
"""
from __future__ import annotations

from llm_cuda.kernels._ops import verify_draft_tokens

__all__ = ["verify_draft_tokens"]
