"""Attention of drafted tokens over a paged kv cache: the verification step of
speculative decoding, plain decoding (one token a sequence) and short chunks of
a prompt.  It stands beside ``sparse_flash_attention_paged`` (which attends to
the blocks that indices select) and reads the same caches, tables and lengths.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import SfaTreeParams
from .rotary import _check_pool, _check_table

_pack = _lib.packer(SfaTreeParams)
_DTYPE = {torch.bfloat16: _lib.SFA_DTYPE_BF16, torch.float16: _lib.SFA_DTYPE_F16}


def _tma_ready(q: torch.Tensor) -> bool:
    """16-byte aligned rows and heads (a size-1 axis has no stride to speak of)."""
    (rows, heads, _), (st, sh, sd) = q.shape, q.stride()
    return (sd == 1 and q.data_ptr() % 16 == 0 and (rows == 1 or (st > 0 and st % 8 == 0))
            and (heads == 1 or (sh > 0 and sh % 8 == 0)))


def tree_attention_paged(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                         cache_seqlens: torch.Tensor, parents: Optional[torch.Tensor] = None,
                         scale: Optional[float] = None, cu_seqlens: Optional[torch.Tensor] = None,
                         attn_sink: Optional[torch.Tensor] = None, max_seqlen_q: Optional[int] = None,
                         max_seqlen_k: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention of each sequence's drafted rows to its whole cached prefix and to
    their ancestors; returns ``(o [total, Hq, Dv], lse [total, Hq])``, no autograd.

    ``q [total, Hq, Dqk]`` (bf16 or fp16) holds the drafted rows of all
    sequences, ``cu_seqlens [n + 1]`` (int32) their offsets (default: one row
    per sequence, plain decoding).  The rows are already in the cache:
    ``cache_seqlens [n]`` are the lengths with them, row j of a sequence with m
    rows being cache position ``cache_seqlens - m + j``.  ``parents [total]``
    (int32) gives each row's parent as a row number within its sequence, below
    its own; -1 (or any number that is not below its own) hangs the row on the
    prefix.  Without ``parents`` the rows form a chain (causal).  A tree has at
    most 256 rows a sequence, a chain any number.

    ``k_cache [num_pages, page_size, Hk, Dqk]``, ``v_cache [num_pages,
    page_size, Hk, Dv]``, ``block_table [n, max_pages]`` (int32) as in
    ``sparse_flash_attention_paged``; any page size; head dims are multiples of
    8 up to 256 (latent caches of more dims go through the sparse surface,
    where a drafted row's ancestors are token indices).  A table entry outside
    the pool holds no keys.  Cache rows that a row does not see have no effect
    on it, whatever they hold.  A row that sees nothing gives ``o = 0`` and
    ``lse = -inf`` (or its sink); so do rows outside all sequences.

    ``max_seqlen_q`` must cover the longest sequence of drafted rows; left unset
    with ``cu_seqlens`` it is read back with a host sync.  It also decides how the
    GPU is shared out: where it is many times what most sequences have (a chunk of
    a prompt among single tokens), those run on a part of the GPU, so give such
    sequences calls of their own.  ``max_seqlen_k`` is an
    estimate of the longest cache that sizes the split of the work (default:
    what the table covers)."""
    if q.dtype not in _DTYPE:
        raise ValueError(f"q must be bfloat16 or float16, got {q.dtype}")
    if q.dim() != 3:
        raise ValueError("q must be [total, Hq, Dqk]")
    device, (total, hq, dqk) = q.device, q.shape
    pools = []
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        pools.append(_check_pool(name, c, q))
        if c.dtype != q.dtype:
            raise ValueError(f"{name} must have q's type")
    ((pages, page, hk, dk), ks), ((v_pages, v_page, v_hk, dv), vs) = pools
    if v_pages != pages or v_page != page or v_hk != hk or dk != dqk:
        raise ValueError("k_cache and v_cache must have the same pages and heads, and k_cache q's head size")
    n, width = _check_table(block_table, cache_seqlens, q)
    if cu_seqlens is None:
        if total != n:
            raise ValueError("without cu_seqlens, q must hold one row per sequence")
        max_seqlen_q = 1
    elif cu_seqlens.dtype != torch.int32 or cu_seqlens.shape != (n + 1,) or cu_seqlens.device != device:
        raise ValueError("cu_seqlens must be int32 [n + 1] on q's device")
    if parents is not None and (parents.dtype != torch.int32 or parents.shape != (total,) or parents.device != device):
        raise ValueError("parents must be int32 [total] on q's device")
    if attn_sink is not None and (attn_sink.shape != (hq,) or attn_sink.device != device):
        raise ValueError("attn_sink must be [Hq] on q's device")
    if scale is None:
        scale = 1.0 / math.sqrt(max(1, dqk))
    if not q.is_cuda:
        raise ValueError("the inputs must be CUDA tensors (tree attention has no CPU implementation)")
    if max_seqlen_q is None:
        max_seqlen_q = int((cu_seqlens[1:] - cu_seqlens[:-1]).max().item()) if n else 0
    max_seqlen_q = min(int(max_seqlen_q), max(1, total))            # no sequence has more rows
    q = q if _tma_ready(q) else q.detach().clone(memory_format=torch.contiguous_format)
    table = block_table if width < 2 or block_table.stride(1) == 1 else block_table.contiguous()
    lens = cache_seqlens.contiguous()
    cu = None if cu_seqlens is None else cu_seqlens.contiguous()
    par = None if parents is None else parents.contiguous()
    sink = None if attn_sink is None else attn_sink.detach().float().contiguous()
    o = q.new_empty((total, hq, dv))
    lse = q.new_empty((total, hq), dtype=torch.float32)
    qs = q.stride()
    max_seqlen_k = min(2**31 - 1, width * page if max_seqlen_k is None else int(max_seqlen_k))
    P = _pack(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), table.data_ptr(), lens.data_ptr(),
              0 if cu is None else cu.data_ptr(), 0 if par is None else par.data_ptr(),
              0 if sink is None else sink.data_ptr(), o.data_ptr(), lse.data_ptr(), qs[0], qs[1], ks[1], ks[2],
              vs[1], vs[2], hq * dv, dv, hq, 1, table.stride(0), n, total, max_seqlen_q, max_seqlen_k, hq, hk,
              dqk, dv, pages, page, width, _DTYPE[q.dtype], float(scale), 0)
    lib, at = _lib.load(), ctypes.byref(P)
    with _lib.on(device):
        nbytes = lib.sfa_tree_workspace_bytes(at)                       # 0 also when the call is refused
        ws = q.new_empty(max(nbytes, 1), dtype=torch.uint8)
        _lib.check(lib.sfa_tree_attention(at, ws.data_ptr(), nbytes, _lib.stream_of(device)), "sfa_tree_attention")
    return o, lse
