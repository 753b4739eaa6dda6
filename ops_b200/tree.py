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
    return (q.stride(2) == 1 and q.data_ptr() % 16 == 0
            and all(q.shape[i] == 1 or (q.stride(i) > 0 and q.stride(i) % 8 == 0) for i in (0, 1)))


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
    with ``cu_seqlens`` it is read back with a host sync.  ``max_seqlen_k`` is an
    estimate of the longest cache that sizes the split of the work (default:
    what the table covers)."""
    if q.dtype not in _DTYPE:
        raise ValueError(f"q must be bfloat16 or float16, got {q.dtype}")
    if q.dim() != 3:
        raise ValueError("q must be [total, Hq, Dqk]")
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        _check_pool(name, c, q)
        if c.dtype != q.dtype:
            raise ValueError(f"{name} must have q's type")
    if k_cache.shape[:3] != v_cache.shape[:3] or k_cache.shape[3] != q.shape[2]:
        raise ValueError("k_cache and v_cache must have the same pages and heads, and k_cache q's head size")
    _check_table(block_table, cache_seqlens, q)
    n, total = block_table.shape[0], q.shape[0]
    if cu_seqlens is None:
        if total != n:
            raise ValueError("without cu_seqlens, q must hold one row per sequence")
        max_seqlen_q = 1
    elif cu_seqlens.dtype != torch.int32 or tuple(cu_seqlens.shape) != (n + 1,) or cu_seqlens.device != q.device:
        raise ValueError("cu_seqlens must be int32 [n + 1] on q's device")
    if parents is not None and (parents.dtype != torch.int32 or tuple(parents.shape) != (total,)
                                or parents.device != q.device):
        raise ValueError("parents must be int32 [total] on q's device")
    if attn_sink is not None and (tuple(attn_sink.shape) != (q.shape[1],) or attn_sink.device != q.device):
        raise ValueError("attn_sink must be [Hq] on q's device")
    if scale is None:
        scale = 1.0 / math.sqrt(max(1, q.shape[2]))
    if not q.is_cuda:
        raise ValueError("the inputs must be CUDA tensors (tree attention has no CPU implementation)")
    if max_seqlen_q is None:
        max_seqlen_q = int((cu_seqlens[1:] - cu_seqlens[:-1]).max().item()) if n else 0
    max_seqlen_q = min(int(max_seqlen_q), max(1, total))            # no sequence has more rows
    device = q.device
    q = q if _tma_ready(q) else q.detach().clone(memory_format=torch.contiguous_format)
    table = block_table if block_table.stride(-1) == 1 or block_table.shape[1] < 2 else block_table.contiguous()
    lens = cache_seqlens.contiguous()
    cu = None if cu_seqlens is None else cu_seqlens.contiguous()
    par = None if parents is None else parents.contiguous()
    sink = None if attn_sink is None else attn_sink.detach().float().contiguous()
    hq, dv = q.shape[1], v_cache.shape[3]
    o = q.new_empty((total, hq, dv))
    lse = q.new_empty((total, hq), dtype=torch.float32)
    pages, page, hk = k_cache.shape[:3]
    ks, vs = k_cache.stride(), v_cache.stride()
    width = table.shape[1]
    max_seqlen_k = min(2**31 - 1, width * page if max_seqlen_k is None else int(max_seqlen_k))
    P = _pack(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), table.data_ptr(), lens.data_ptr(),
              0 if cu is None else cu.data_ptr(), 0 if par is None else par.data_ptr(),
              0 if sink is None else sink.data_ptr(), o.data_ptr(), lse.data_ptr(), q.stride(0), q.stride(1), ks[1], ks[2],
              vs[1], vs[2], hq * dv, dv, hq, 1, table.stride(0), n, total, max_seqlen_q, max_seqlen_k, hq, hk,
              q.shape[2], dv, pages, page, width, _DTYPE[q.dtype], float(scale), 0)
    lib, at = _lib.load(), ctypes.byref(P)
    with _lib.on(device):
        nbytes = lib.sfa_tree_workspace_bytes(at)                       # 0 also when the call is refused
        ws = q.new_empty(max(nbytes, 1), dtype=torch.uint8)
        _lib.check(lib.sfa_tree_attention(at, ws.data_ptr(), nbytes, _lib.stream_of(device)), "sfa_tree_attention")
    return o, lse
