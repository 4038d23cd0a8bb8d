"""Fused sigmoid attention for AMD MI355X (gfx950), drop-in for triton-sigmoid.

    output = sigmoid(Q·Kᵀ·scale + bias + score_mod[k]) · V

Public API (same names and signatures as MSDLLCpapers/triton-sigmoid,
src/triton_sigmoid/__init__.py:68-78):
  * sigmoid_attention(query, key, value, is_causal, scale, sigmoid_bias, score_mod)
  * sigmoid_attention_padded(query, key, value, seq_lens_k, seq_lens_q,
                             is_causal, scale, sigmoid_bias, score_mod)
  * sigmoid_attention_ref(...)  eager PyTorch definition
plus additions with no counterpart in the reference's API:
  * sigmoid_attention_varlen(query, key, value, cu_seqlens_q, cu_seqlens_k,
                             max_seqlen_q, max_seqlen_k, is_causal, scale,
                             sigmoid_bias, score_mod)
    for packed [total_tokens, H, D] sequences (the packed layout of the
    reference's benchmark, benchmarks/benchmark_sigmoid.py:116-134), whose keys
    and values may have fewer heads than the queries.
and the paged key/value cache of a serving loop:
  * paged_plan(context_lens, new_lens, block_table, free_pages, page_size,
               num_tokens) pages and slots of a step's new tokens, on the GPU
  * paged_cache_write(key, value, key_cache, value_cache, slot_mapping)
  * sigmoid_attention_paged(query, key_cache, value_cache, block_table,
                            seq_lens_k, cu_seqlens_q, max_seqlen_q, is_causal,
                            scale, sigmoid_bias, score_mod)

The kernel entry points run hand-written HIP kernels for gfx950 (MFMA,
LDS-staged tiles) through the C ABI in libsigattn.so, registered as
torch.library custom ops `myops::sigmoid_attention_fwd/bwd`,
`myops::sigmoid_attn_padded_fwd/bwd`, `myops::sigmoid_attn_varlen_fwd/bwd`,
`myops::paged_plan`, `myops::paged_cache_write` and
`myops::sigmoid_attn_paged_fwd`.
Importing works anywhere (so graphs can be traced on the CPU); calling the
kernels needs a gfx950 GPU and raises RuntimeError otherwise.  There is no
CPU or eager fallback.
"""

__version__ = "0.1.2"

from .sigmoid_dense import sigmoid_attention
from .sigmoid_padded import sigmoid_attention_padded
from .sigmoid_paged import PagedPlan, paged_cache_write, paged_plan, sigmoid_attention_paged
from .sigmoid_reference import sigmoid_attention_ref
from .sigmoid_varlen import sigmoid_attention_varlen

__all__ = [
    "sigmoid_attention",
    "sigmoid_attention_padded",
    "sigmoid_attention_paged",
    "sigmoid_attention_ref",
    "sigmoid_attention_varlen",
    "PagedPlan",
    "paged_cache_write",
    "paged_plan",
]
