"""One attention layer's prefill on the paged KV cache.

Restates the prefill branch of the reference's ``Attention`` layer
(prism_infer/layers/attention.py:85-111 routing, :158-169 ``_store_current_kv``,
:180-208 prompts without a cached prefix, :448-459 ``_forward_prefill_paged``):
store the chunk's K/V into their slots, then attend.  Where no sequence has
cached tokens in front of its prompt the keys are the call's own K/V, packed
like the queries (:func:`prompt_attention`: 16-bit keys, also where the cache is
FP8); otherwise they are read from the pages (:func:`paged_prefill_attention`).

Bind the layer's caches as for :class:`PagedKVDecodeAttention`.  The metadata is a
:class:`StepMetadata`, or any object with ``slot_mapping``, ``cu_seqlens_q``,
``context_lens`` and ``block_tables``.
"""

from __future__ import annotations

import torch

from prism_infer.engine.decode_attention import PagedKVDecodeAttention
from prism_infer.ops.kv_cache_store import store_kvcache
from prism_infer.ops.paged_prefill import paged_prefill_attention
from prism_infer.ops.prompt_attention import prompt_attention


class PagedKVPrefillAttention(PagedKVDecodeAttention):
    """Prefill attention of one layer, over the same bound caches as its decode."""

    def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, metadata, *, cached_prefix: bool) -> torch.Tensor:
        """Store the chunk's K/V ([T, kv_heads, head_dim]) and attend; q is [T, num_heads, head_dim].

        ``cached_prefix`` says whether any sequence has stored tokens in front of
        this chunk, which the host knows.  With, every sequence has new tokens (as in
        the reference, one without is refused).  Without, the result has q's rows, zeros
        where they are padding; with, the sequences' rows, or under graph capture
        all of q's, of which padding is zeros over 16-bit caches and unspecified
        over FP8 ones.
        """

        self._validate_cache_bindings()
        if metadata.slot_mapping is None:
            raise RuntimeError("bound KV cache requires slot_mapping")
        store_kvcache(k, v, self.k_cache, self.v_cache, metadata.slot_mapping, self.k_scale_cache,
                      self.v_scale_cache)
        if not cached_prefix:
            return prompt_attention(q, k, v, metadata.cu_seqlens_q, num_heads=self.num_heads,
                                    num_kv_heads=self.num_kv_heads, scale=self.scale)
        return paged_prefill_attention(
            q, self.k_cache, self.v_cache, metadata, num_heads=self.num_heads, num_kv_heads=self.num_kv_heads,
            scale=self.scale, k_scale_cache=self.k_scale_cache, v_scale_cache=self.v_scale_cache,
        )

    __call__ = forward


__all__ = ["PagedKVPrefillAttention"]
