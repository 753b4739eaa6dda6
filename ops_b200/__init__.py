"""ops_b200 — B200-native (sm_100a) sparse flash attention.

Public surface:
  sparse_flash_attention(q, k, v, block_indices, ...) -> (o, lse)
  SparseFlashAttention.apply(q, kv, attn_sink, topk_idxs, sm_scale) -> out   # reference signature
  sparse_flash_attention_paged(q, k_cache, v_cache, block_indices, block_table, cache_seqlens, ...)
                                                      # forward over a paged kv cache (decode)
  lightning_indexer_topk(q_idx, k_idx, weights, topk) -> token indices for the op
  tree_attention_paged(q, k_cache, v_cache, block_table, cache_seqlens, parents, ...)
                                                      # drafted trees, chains or single tokens over the whole cache
  paged_cache_reserve / _trim / _fork / _accept / _compact / _copy   # pages of the cache, all on the device
  rotary_frequencies / rotary_embedding / qk_norm_rotary(q, k, positions, frequencies, ...)
                                                      # norm and rotary positions before the op, with gradients
  qk_norm_rotary_append(q, k, v, ..., k_cache, v_cache, block_table, cache_seqlens)   # the same into a paged cache
  sparse_flash_attention_fp8kv(q, kv_fp8, kv_scale, block_indices, d_v, ...)  # e4m3 latent kv cache
The kernels live in libsfa_b200.so (C ABI: include/sfa_b200.h).
"""
from ._lib import SfaError, SfaParams, load as load_library
from .sfa import (SparseFlashAttention, SparseFlashAttentionCompat, quantize_kv_fp8, reference_lse2,
                  sparse_flash_attention, sparse_flash_attention_fp8kv, sparse_flash_attention_paged)
from . import tiling
from .cache import (paged_cache_accept, paged_cache_compact, paged_cache_copy, paged_cache_fork, paged_cache_reserve,
                    paged_cache_trim)
from .indexer import lightning_indexer_topk
from .tree import tree_attention_paged
from .rotary import qk_norm_rotary, qk_norm_rotary_append, rotary_embedding, rotary_frequencies

__all__ = ["sparse_flash_attention", "sparse_flash_attention_paged", "SparseFlashAttention",
           "SparseFlashAttentionCompat", "SfaError", "SfaParams", "load_library", "reference_lse2", "tiling",
           "lightning_indexer_topk", "sparse_flash_attention_fp8kv", "quantize_kv_fp8", "rotary_frequencies",
           "rotary_embedding", "tree_attention_paged", "paged_cache_reserve", "paged_cache_trim", "paged_cache_fork",
           "paged_cache_accept", "paged_cache_compact", "paged_cache_copy", "qk_norm_rotary", "qk_norm_rotary_append"]
