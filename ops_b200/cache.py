"""Pages of a kv cache, between the steps that attend to it: room for new rows,
forks that share pages, the accepted path of a drafted tree moved together,
pages given back, and a pool compacted.

The state is three int32 tensors on the device, changed in place and never read
back to the host: ``refcounts [num_pages]`` (how many table entries hold a page;
0 is free, and a fresh pool is ``torch.zeros``), ``block_table [n, max_pages]``
(the pages of each sequence, -1 behind them) and ``cache_seqlens [n]`` (a free
sequence has length 0) — the table and the lengths that
``sparse_flash_attention_paged`` and ``tree_attention_paged`` take.  New pages
are the free ones of lowest number, in the order of the rows that ask, so a run
repeats.  ``pools`` are the tensors that the pages index, ``[num_pages,
page_size, ...]`` with contiguous pages: K and V of every layer, any type.
"""
from __future__ import annotations

import ctypes
import struct
from operator import sub
from typing import Optional, Sequence

import torch

from . import _lib
from ._lib import SfaCacheParams, SfaCachePool


def _ints(name: str, t: torch.Tensor, dim: int, like: torch.Tensor, size: Optional[int] = None) -> None:
    """An int32 tensor changed or read in place."""
    if t.dtype != torch.int32 or t.dim() != dim or t.device != like.device:
        raise ValueError(f"{name} must be a {dim}-D int32 tensor on the device of the others")
    if size is not None and t.shape[0] != size:
        raise ValueError(f"{name} must have {size} entries, got {t.shape[0]}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must be contiguous in its last dim (it is used in place)")


def _pools_meet(values, num_pages: int) -> bool:
    """Whether pools share memory; values: (address, page stride, page bytes) of each, one after another."""
    bases, strides, sizes = values[::3], values[1::3], values[2::3]
    stride, size = strides[0], sizes[0]
    if strides.count(stride) == len(strides) and sizes.count(size) == len(sizes):
        at = sorted(bases)                             # pools alike, one behind the other or side by side in a page
        gap = min(map(sub, at[1:], at), default=stride)
        if gap >= (num_pages - 1) * stride + size or gap >= size and at[-1] + size - at[0] <= stride:
            return False
    spans = sorted(p for p in zip(bases, strides, sizes) if p[2] and num_pages > 0)
    for i, (base, stride, size) in enumerate(spans):
        last = base + (num_pages - 1) * stride + size
        for base2, stride2, size2 in spans[i + 1:]:
            if base2 >= last:
                break
            # pages of one stride lie in one another's gaps, or they meet
            r = base2 - base
            if num_pages > 1:
                if stride2 != stride:
                    return True
                r %= stride
            if r < size or num_pages > 1 and r + size2 > stride:
                return True
    return False


def _pool_array(pools: Sequence[torch.Tensor], like: torch.Tensor, num_pages: Optional[int]):
    if len(pools) == 0:
        raise ValueError("pools must hold at least one tensor")
    lead, device = pools[0].shape[:2], like.device
    bad = len(lead) < 2 or lead[1] < 1 or num_pages not in (None, lead[0])
    values = []
    first, same = pools[0], None                       # same: page bytes of contiguous pools like the first
    if not bad and first.is_contiguous():
        shape, dtype = first.shape, first.dtype
        same = first.numel() // max(lead[0], 1) * first.element_size()
    for t in pools:
        if same is not None and t.shape == shape and t.dtype is dtype and t.device == device and t.is_contiguous():
            values += (t.data_ptr(), same, same)
            continue
        if bad or t.device != device or t.shape[:2] != lead:
            raise ValueError("every pool must be [num_pages, page_size, ...] with the same pages, on the device of the table")
        size = t.element_size()
        if t.is_contiguous():
            inner = expect = t.numel() // max(lead[0], 1)
        else:
            inner = t.stride(0) if t.shape[0] > 1 else 0
            expect = 1
            for extent, stride in zip(reversed(t.shape[1:]), reversed(t.stride()[1:])):
                if extent > 1 and stride != expect:
                    raise ValueError("a pool's pages must be contiguous")
                expect *= extent
            if t.shape[0] > 1 and inner < expect:
                raise ValueError("a pool's pages must not overlap")
        values += (t.data_ptr(), (inner or expect) * size, expect * size)
    held = [ptr for ptr in values[::3] if ptr]
    if len(set(held)) < len(held):
        raise ValueError("a pool is named twice")
    if _pools_meet(values, lead[0]):
        raise ValueError("pools must not share memory")
    arr = (SfaCachePool * len(pools)).from_buffer_copy(struct.pack("@" + "Pqq" * len(pools), *values))
    return arr, lead[0], lead[1]


_pack = _lib.packer(SfaCacheParams)


def _params(refcounts, table, lens, page_size, num_pages, a=None, b=None, out=None, pools=None, count=0) -> SfaCacheParams:
    def ptr(t):
        return 0 if t is None else t.data_ptr()

    n, width, bt = (0, 0, 0) if table is None else (*table.shape, table.stride(0))
    a_stride = a.stride(0) if a is not None and a.dim() == 2 else 0
    P = _pack(ptr(refcounts), ptr(table), ptr(lens), ptr(a), ptr(b), ptr(out), 0 if pools is None else ctypes.addressof(pools),
              bt, a_stride, 0 if pools is None else len(pools), n, num_pages, int(page_size), width, count)
    P.held = pools                       # the array lives as long as the struct
    return P


def _call(name: str, P: SfaCacheParams, like: torch.Tensor, workspace: bool = True) -> None:
    if not like.is_cuda:
        raise ValueError("the cache's state must be CUDA tensors (there is no CPU implementation)")
    lib = _lib.load()
    with _lib.on(like.device):
        if workspace:
            nbytes = lib.sfa_cache_workspace_bytes(ctypes.byref(P))
            ws = like.new_empty(max(nbytes, 1), dtype=torch.uint8)
            rc = getattr(lib, name)(ctypes.byref(P), ws.data_ptr(), nbytes, _lib.stream_of(like.device))
        else:
            rc = getattr(lib, name)(ctypes.byref(P), _lib.stream_of(like.device))
        _lib.check(rc, name)


def _state(refcounts, block_table, cache_seqlens, page_size=None) -> None:
    _ints("refcounts", refcounts, 1, refcounts)
    _ints("block_table", block_table, 2, refcounts)
    if block_table.shape[0] > 1 and block_table.stride(0) < block_table.shape[1]:
        raise ValueError("block_table's rows must not overlap")
    if cache_seqlens is not None:
        _ints("cache_seqlens", cache_seqlens, 1, refcounts, block_table.shape[0])
    if page_size is not None and int(page_size) < 1:
        raise ValueError("page_size must be positive")


def paged_cache_reserve(refcounts: torch.Tensor, block_table: torch.Tensor, cache_seqlens: torch.Tensor,
                        add: torch.Tensor, page_size: int) -> torch.Tensor:
    """Room for ``add [n]`` (int32) more rows of each sequence: the pages they need
    go into the table and ``cache_seqlens`` grows.  Returns ``granted [n]``
    (int32): 1, or 0 where nothing was changed — a negative count, a table too
    narrow, a partly filled last page that other sequences share, or free pages
    too few for the sequences up to this one together.  The length of a sequence
    that was refused does not include its new rows, so they would be stored over
    its last ones: pass ``cache_seqlens * granted`` to ``qk_norm_rotary_append``
    and ``tree_attention_paged`` (at length 0 the rows have no place and are not
    stored, and see nothing) and ``drafted * granted`` to
    ``paged_cache_accept``."""
    _state(refcounts, block_table, cache_seqlens, page_size)
    _ints("add", add, 1, refcounts, block_table.shape[0])
    granted = torch.empty_like(add)
    P = _params(refcounts, block_table, cache_seqlens, page_size, refcounts.shape[0], add, None, granted)
    _call("sfa_cache_reserve", P, refcounts)
    return granted


def paged_cache_trim(refcounts: torch.Tensor, block_table: torch.Tensor, cache_seqlens: torch.Tensor,
                     keep: torch.Tensor, page_size: int) -> None:
    """Every sequence keeps its first ``keep [n]`` (int32) rows — 0 frees it, a
    negative number leaves it alone — and the pages behind them are given back:
    a page is free once no sequence holds it."""
    _state(refcounts, block_table, cache_seqlens, page_size)
    _ints("keep", keep, 1, refcounts, block_table.shape[0])
    P = _params(refcounts, block_table, cache_seqlens, page_size, refcounts.shape[0], keep)
    _call("sfa_cache_trim", P, refcounts, workspace=False)


def paged_cache_fork(refcounts: torch.Tensor, block_table: torch.Tensor, cache_seqlens: torch.Tensor,
                     src: torch.Tensor, dst: torch.Tensor, pools: Sequence[torch.Tensor]) -> torch.Tensor:
    """Sequence ``dst[i]`` becomes a copy of sequence ``src[i]`` (int32 ``[f]``
    each): whole pages are shared, a partly filled last page is copied into a new
    page in every pool.  Returns ``forked [f]`` (int32): 1, or 0 where nothing was
    changed — a number outside the table, a target that still holds rows or that
    an earlier fork of the call names, a last page outside the pool, or no free
    page.  Sources are taken as they were before the call, and may repeat.  Rows
    that were reserved but not stored yet are part of a source's whole pages: store
    them before the fork, or both sequences would store into one page."""
    _state(refcounts, block_table, cache_seqlens)
    _ints("src", src, 1, refcounts)
    _ints("dst", dst, 1, refcounts, src.shape[0])
    arr, num_pages, page = _pool_array(pools, refcounts, refcounts.shape[0])
    forked = torch.empty_like(src)
    P = _params(refcounts, block_table, cache_seqlens, page, num_pages, src, dst, forked, arr, src.shape[0])
    _call("sfa_cache_fork", P, refcounts)
    return forked


def paged_cache_accept(pools: Sequence[torch.Tensor], block_table: torch.Tensor, cache_seqlens: torch.Tensor,
                       accepted: torch.Tensor, drafted: torch.Tensor, refcounts: Optional[torch.Tensor] = None) -> torch.Tensor:
    """After the verification of drafted trees: of the last ``drafted [n]`` rows of
    each sequence, those named by ``accepted [n, m]`` (int32: ascending row
    numbers of the tree, ended by -1 or the width; an entry that is not above the
    one before or not below ``drafted`` ends it too) are moved together behind
    the prefix, in every pool.  Returns ``keep [n]`` (int32), the rows that each
    sequence should keep, for ``paged_cache_trim``; -1 where nothing was moved:
    ``drafted`` is negative or above the length, or a row would go into a page
    that another sequence holds too (a fork after the drafted rows were stored
    shares their whole pages: free one of the two, or fork after the
    acceptance).  ``refcounts [num_pages]`` says which pages are shared; without
    it the entries of this table are counted, in a launch of its own, and pages
    that only another table holds count as unshared."""
    _ints("block_table", block_table, 2, block_table)
    _ints("cache_seqlens", cache_seqlens, 1, block_table, block_table.shape[0])
    _ints("accepted", accepted, 2, block_table, block_table.shape[0])
    _ints("drafted", drafted, 1, block_table, block_table.shape[0])
    arr, num_pages, page = _pool_array(pools, block_table, None)
    name = "sfa_cache_accept"
    if refcounts is not None:
        _ints("refcounts", refcounts, 1, block_table, num_pages)
    else:
        name, refcounts = "sfa_cache_accept_table", block_table.new_empty(num_pages)
    keep = torch.empty_like(cache_seqlens)
    P = _params(refcounts, block_table, cache_seqlens, page, num_pages, accepted if accepted.numel() else drafted, drafted, keep,
                arr, accepted.shape[1])
    _call(name, P, block_table, workspace=False)
    return keep


def paged_cache_compact(refcounts: torch.Tensor, block_table: torch.Tensor, pools: Sequence[torch.Tensor]) -> torch.Tensor:
    """The pages in use move to the lowest numbers (each page above their count to
    the next free one below it), with the table and the counts.  Returns their
    number (int32 ``[1]``, on the device): every page from there on is free."""
    _state(refcounts, block_table, None)
    arr, num_pages, page = _pool_array(pools, refcounts, refcounts.shape[0])
    live = torch.empty(1, dtype=torch.int32, device=refcounts.device)
    P = _params(refcounts, block_table, None, page, num_pages, None, None, live, arr)
    _call("sfa_cache_compact", P, refcounts)
    return live


def paged_cache_copy(pools: Sequence[torch.Tensor], src: torch.Tensor, dst: torch.Tensor) -> torch.Tensor:
    """Page ``src[i]`` is copied to page ``dst[i]`` (int32 ``[m]`` each) in every
    pool.  Returns ``copied [m]`` (int32): 1, or 0 for a page outside the pool, a
    target that an earlier pair names, or a source that another pair writes."""
    _ints("src", src, 1, src)
    _ints("dst", dst, 1, src, src.shape[0])
    arr, num_pages, page = _pool_array(pools, src, None)
    copied = torch.empty_like(src)
    P = _params(None, None, None, page, num_pages, src, dst, copied, arr, src.shape[0])
    _call("sfa_cache_copy", P, src)
    return copied
