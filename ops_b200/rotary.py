"""Norm and rotary positions of queries and keys, the step before the sparse
attention op (the reference takes q and kv as they are, SFA.py:87-90).

``qk_norm_rotary`` normalises every head of q and k (RMS norm with a weight per
dim) and turns the pairs of the rotated part by ``position * frequency``, in one
pass, with gradients for q, k and both weights; ``rotary_embedding`` is the
rotation of one tensor alone; ``qk_norm_rotary_append`` is the serving form,
which stores k and v straight into the pages of a kv cache.  Everything is
computed in fp32 and rounded once; angles are reduced exactly, so positions far
into a long context are as accurate as the first ones.
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import SfaRotaryParams

_DTYPE = {torch.bfloat16: _lib.SFA_DTYPE_BF16, torch.float16: _lib.SFA_DTYPE_F16, torch.float32: _lib.SFA_DTYPE_F32}


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                       original_length: int = 8192, beta_fast: float = 32.0, beta_slow: float = 1.0,
                       device: Optional[torch.device] = None) -> Tuple[torch.Tensor, float]:
    """``(frequencies, amplitude)`` for the rotary functions: ``[rotary_dim / 2]``
    float64 radians per position, ``base ** (-2 i / rotary_dim)``, and the factor
    on the turned dims.  ``scaling`` stretches them for contexts ``factor``
    times longer:

    * ``"linear"``: every frequency divided by ``factor``;
    * ``"ntk"``: the base raised so that the slowest pair turns ``factor`` times
      slower and the fastest as before;
    * ``"yarn"``: pairs that turn more than ``beta_fast`` times in
      ``original_length`` positions stay, those that turn less than
      ``beta_slow`` times are divided by ``factor``, those between are blended
      linearly in their number of turns; the amplitude is ``0.1 ln(factor) + 1``.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be a positive even number")
    if not (base > 0 and math.isfinite(base)) or not (factor > 0 and math.isfinite(factor)):
        raise ValueError("base and factor must be positive and finite")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    amplitude = 1.0
    if scaling == "ntk" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    f = torch.tensor(float(base), dtype=torch.float64) ** (-i / rotary_dim)
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        if not beta_fast > beta_slow:
            raise ValueError("beta_fast must be above beta_slow")
        turns = original_length * f / (2 * math.pi)
        keep = ((turns - beta_slow) / (beta_fast - beta_slow)).clamp(0.0, 1.0)
        f = f * keep + f / factor * (1.0 - keep)
        amplitude = 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0
    elif scaling not in (None, "ntk"):
        raise ValueError(f"unknown scaling {scaling!r}: expected None, 'linear', 'ntk' or 'yarn'")
    return f.to(device) if device is not None else f, amplitude


@dataclass(frozen=True)
class _Cfg:
    rot: int
    start: int
    interleaved: bool
    eps: float
    amplitude: float


def _rows(x: torch.Tensor) -> torch.Tensor:
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _strides(x: torch.Tensor):
    """(batch, token, head) element strides of [B, T, H, D] or [T, H, D]."""
    s = x.stride()
    return s[:3] if len(s) == 4 else (0, s[0], s[1])


def _check(name: str, x: torch.Tensor, like: Optional[torch.Tensor] = None) -> None:
    if x.dtype not in _DTYPE:
        raise ValueError(f"{name} must be bfloat16, float16 or float32, got {x.dtype}")
    if x.dim() not in (3, 4) or x.shape[-2] < 1 or x.shape[-1] < 1:
        raise ValueError(f"{name} must be [B, T, H, D] or [T, H, D] with at least one head and dim")
    if like is not None and (x.dtype != like.dtype or x.device != like.device or x.shape[:-2] != like.shape[:-2]
                             or x.shape[-1] != like.shape[-1]):
        raise ValueError(f"{name} must have q's type, device, tokens and head size")


def _need_cuda(x: torch.Tensor) -> None:
    if not x.is_cuda:
        raise ValueError("the inputs must be CUDA tensors (the rotary ops have no CPU implementation)")


def _check_turn(x: torch.Tensor, positions, frequencies, interleaved, start, eps, amplitude):
    """The config and the positions broadcast to x's tokens."""
    if (positions is None) != (frequencies is None):
        raise ValueError("positions and frequencies go together")
    rot = 0
    if frequencies is not None:
        if frequencies.dim() != 1 or frequencies.dtype != torch.float64 or frequencies.device != x.device:
            raise ValueError("frequencies must be a 1-D float64 tensor on the inputs' device")
        if positions.dtype not in (torch.int32, torch.int64) or positions.device != x.device:
            raise ValueError("positions must be int32 or int64 on the inputs' device")
        if frequencies.requires_grad:
            raise ValueError("frequencies have no gradient: detach them")
        rot = 2 * frequencies.numel()
        frequencies = frequencies.contiguous()
        tokens = x.shape[:-2]
        if positions.shape != tokens:
            try:
                positions = positions.expand(tokens)
            except RuntimeError:
                raise ValueError(f"positions {tuple(positions.shape)} do not broadcast to tokens {tuple(tokens)}")
    if start < 0 or start + rot > x.shape[-1]:
        raise ValueError("the rotated dims [start, start + rotary_dim) must lie within the head")
    if not eps >= 0:
        raise ValueError("eps must be >= 0")
    return _Cfg(rot, int(start), bool(interleaved), float(eps), float(amplitude)), positions, frequencies


def _weight(name: str, w: Optional[torch.Tensor], x: torch.Tensor) -> Optional[torch.Tensor]:
    if w is None:
        return None
    if w.dim() != 1 or w.shape[0] != x.shape[-1] or w.device != x.device or not w.is_floating_point():
        raise ValueError(f"{name} must be a floating-point vector of the head size on the inputs' device")
    return w if w.dtype == torch.float32 and w.is_contiguous() else w.float().contiguous()


_pack = _lib.packer(SfaRotaryParams)
_TURN, _PAGED = _lib.SFA_ROTARY_TURN, _lib.SFA_ROTARY_PAGED
_NO_TENSOR = (0,) * 20
_NO_CACHE = (0, 0, 0, 0)


def _tensor(x, w, y=None, dy=None, dx=None, dw=None, turned=_TURN):
    """The values of one SfaRotaryTensor."""
    return (x.data_ptr(), 0 if y is None else y.data_ptr(), 0 if dy is None else dy.data_ptr(),
            0 if dx is None else dx.data_ptr(), 0 if w is None else w.data_ptr(), 0 if dw is None else dw.data_ptr(),
            *_strides(x), *(_strides(y) if y is not None else (0, 0, 0)), *(_strides(dy) if dy is not None else (0, 0, 0)),
            *(_strides(dx) if dx is not None else (0, 0, 0)), x.shape[-2], turned)


def _paged(x, w, pool, turned):
    """The values of one SfaRotaryTensor that goes into a page pool."""
    return (x.data_ptr(), pool.data_ptr(), 0, 0, 0 if w is None else w.data_ptr(), 0, *_strides(x), 0, pool.stride(1),
            pool.stride(2), 0, 0, 0, 0, 0, 0, x.shape[-2], turned | _PAGED)


def _params(x: torch.Tensor, tensors, cfg: _Cfg, positions, frequencies, cache=_NO_CACHE, sizes=_NO_CACHE) -> SfaRotaryParams:
    batch, length = (x.shape[0], x.shape[1]) if x.dim() == 4 else (1, x.shape[0])
    if positions is None:
        pos, freq, sb, st, p64 = 0, 0, 0, 0, 0
    else:
        pos, freq, p64 = positions.data_ptr(), frequencies.data_ptr(), int(positions.dtype == torch.int64)
        sb, st = positions.stride() if positions.dim() == 2 else (0, positions.stride(0))
    n = len(tensors)
    return _pack(*tensors[0], *(tensors[1] if n > 1 else _NO_TENSOR), *(tensors[2] if n > 2 else _NO_TENSOR), pos, freq,
                 *cache, sb, st, n, batch, length, x.shape[-1], cfg.rot, cfg.start, int(cfg.interleaved), _DTYPE[x.dtype],
                 p64, *sizes, cfg.eps, cfg.amplitude, 0)


class _NormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, positions, frequencies, cfg: _Cfg):
        oq = torch.empty_like(q, memory_format=torch.contiguous_format)
        tensors = [_tensor(q, wq, oq)]
        if k is not None:
            ok = torch.empty_like(k, memory_format=torch.contiguous_format)
            tensors.append(_tensor(k, wk, ok))
        P = _params(q, tensors, cfg, positions, frequencies)
        with _lib.on(q.device):
            _lib.check(_lib.load().sfa_rotary_fwd(ctypes.byref(P), _lib.stream_of(q.device)), "sfa_rotary_fwd")
        ctx.save_for_backward(q, k, wq, wk, positions, frequencies)
        ctx.cfg = cfg
        return (oq, ok) if k is not None else oq

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        q, k, wq, wk, positions, frequencies = ctx.saved_tensors
        need = ctx.needs_input_grad
        out = [None] * 7
        tensors, held = [], []
        sums = False
        for i, (x, w) in enumerate(((q, wq), (k, wk))):
            if x is None or not (need[i] or need[2 + i]):
                continue
            dy = _rows(grads[i])
            dx = torch.empty_like(x, memory_format=torch.contiguous_format)
            dw = torch.empty_like(w) if w is not None and need[2 + i] else None
            tensors.append(_tensor(x, w, None, dy, dx, dw))
            out[i], out[2 + i] = dx, dw
            held.append(dy)
            sums = sums or dw is not None
        if tensors:
            lib, P, device = _lib.load(), _params(q, tensors, ctx.cfg, positions, frequencies), q.device
            with _lib.on(device):
                nbytes = lib.sfa_rotary_bwd_workspace_bytes(ctypes.byref(P)) if sums else 0
                ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
                _lib.check(lib.sfa_rotary_bwd(ctypes.byref(P), None if ws is None else ws.data_ptr(), nbytes,
                                              _lib.stream_of(device)), "sfa_rotary_bwd")
        return tuple(out)


def rotary_embedding(x: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor, interleaved: bool = False,
                     start: int = 0, amplitude: float = 1.0) -> torch.Tensor:
    """Rotary positions of one tensor ``[B, T, H, D]`` or ``[T, H, D]`` (bf16,
    fp16 or fp32; any strides with the head dims contiguous): dims ``[start,
    start + 2 * len(frequencies))`` of every head are turned pair by pair by
    ``position * frequency`` and scaled by ``amplitude``, the others are copied.
    Pairs are ``(i, i + rotary_dim / 2)``, or neighbours when ``interleaved``.
    ``positions`` (int32 or int64) broadcast to the tokens.  Differentiable in x."""
    _check("x", x)
    if frequencies is None or positions is None:
        raise ValueError("rotary_embedding needs positions and frequencies")
    cfg, positions, frequencies = _check_turn(x, positions, frequencies, interleaved, start, 0.0, amplitude)
    _need_cuda(x)
    return _NormRotary.apply(_rows(x), None, None, None, positions, frequencies, cfg)


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, positions: Optional[torch.Tensor],
                   frequencies: Optional[torch.Tensor], q_weight: Optional[torch.Tensor] = None,
                   k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False,
                   start: int = 0, amplitude: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(q, k)`` with every head RMS-normalised (where its weight ``[D]`` is
    given) and rotated, in one launch: ``q [B, T, Hq, D]``, ``k [B, T, Hk, D]``
    (varlen: no B), layouts and rotation as in ``rotary_embedding``.  Pass None
    for positions and frequencies to norm only.  Gradients flow to q, k and the
    weights (the weights' sums are in fp32 in a fixed order, so runs repeat bit
    for bit)."""
    _check("q", q)
    _check("k", k, q)
    cfg, positions, frequencies = _check_turn(q, positions, frequencies, interleaved, start, eps, amplitude)
    wq, wk = _weight("q_weight", q_weight, q), _weight("k_weight", k_weight, k)
    _need_cuda(q)
    return _NormRotary.apply(_rows(q), _rows(k), wq, wk, positions, frequencies, cfg)


def _check_pool(name: str, c: torch.Tensor, like: torch.Tensor) -> None:
    if c.dim() != 4 or c.device != like.device:
        raise ValueError(f"{name} must be a [num_pages, page_size, H, D] page pool on the inputs' device")
    if c.shape[3] > 1 and c.stride(-1) != 1 or c.shape[0] > 1 and c.stride(0) != c.shape[1] * c.stride(1):
        raise ValueError(f"{name}: pages must be [page_size, H, D] row ranges of one pool, innermost dim contiguous")


def _check_table(block_table: torch.Tensor, cache_seqlens: torch.Tensor, like: torch.Tensor) -> None:
    for name, t, d in (("block_table", block_table, 2), ("cache_seqlens", cache_seqlens, 1)):
        if t.dtype != torch.int32 or t.dim() != d or t.device != like.device:
            raise ValueError(f"{name} must be a {d}-D int32 tensor on the inputs' device")
    if cache_seqlens.shape[0] != block_table.shape[0]:
        raise ValueError("block_table and cache_seqlens must name the same number of sequences")


def qk_norm_rotary_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: Optional[torch.Tensor],
                          frequencies: Optional[torch.Tensor], k_cache: torch.Tensor, v_cache: torch.Tensor,
                          block_table: torch.Tensor, cache_seqlens: torch.Tensor,
                          cu_seqlens: Optional[torch.Tensor] = None, q_weight: Optional[torch.Tensor] = None,
                          k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False,
                          start: int = 0, amplitude: float = 1.0) -> torch.Tensor:
    """The serving form of ``qk_norm_rotary``: one launch norms and rotates q
    (returned) and k, and stores k and v into the pages of a kv cache (forward
    only, no autograd).

    ``q [total, Hq, D]``, ``k [total, Hk, D]`` and ``v [total, Hk, Dv]`` hold
    the new rows of all sequences; ``cu_seqlens [n + 1]`` (int32) are their
    offsets (default: one row per sequence, the decode step).  ``cache_seqlens
    [n]`` are the cache lengths *with* the new rows, as the paged attention
    takes them: row i of sequence s goes to cache position ``cache_seqlens[s] -
    rows(s) + i`` in ``k_cache [num_pages, page_size, Hk, D]`` and ``v_cache
    [num_pages, page_size, Hk, Dv]`` through ``block_table [n, max_pages]``.
    ``positions`` are the rotary positions, which may differ from the cache
    positions (the depth of a drafted node).  Rows behind the last sequence,
    negative cache positions, positions behind the table and page ids outside
    the pool are not stored.  ``v`` may have another head size than k."""
    for name, x in (("q", q), ("k", k), ("v", v)):
        _check(name, x)
        if x.dim() != 3 or x.dtype != q.dtype or x.device != q.device or x.shape[0] != q.shape[0]:
            raise ValueError(f"{name} must be [total, H, D] with q's type, device and rows")
    if k.shape[-1] != q.shape[-1] or v.shape[1] != k.shape[1]:
        raise ValueError("k must have q's head size and v must have k's heads")
    for name, c, x in (("k_cache", k_cache, k), ("v_cache", v_cache, v)):
        _check_pool(name, c, q)
        if c.dtype != q.dtype or tuple(c.shape[2:]) != tuple(x.shape[1:]):
            raise ValueError(f"{name} must have the type, heads and head size of the rows stored into it")
    if v_cache.shape[:2] != k_cache.shape[:2]:
        raise ValueError("k_cache and v_cache must have the same pages")
    if k_cache.data_ptr() == v_cache.data_ptr() != 0:
        raise ValueError("k_cache and v_cache must not be the same memory")
    _check_table(block_table, cache_seqlens, q)
    n = block_table.shape[0]
    if cu_seqlens is None:
        if q.shape[0] != n:
            raise ValueError("without cu_seqlens, q must hold one row per sequence")
    elif cu_seqlens.dtype != torch.int32 or tuple(cu_seqlens.shape) != (n + 1,) or cu_seqlens.device != q.device:
        raise ValueError("cu_seqlens must be int32 [n + 1] on the inputs' device")
    cfg, positions, frequencies = _check_turn(q, positions, frequencies, interleaved, start, eps, amplitude)
    wq, wk = _weight("q_weight", q_weight, q), _weight("k_weight", k_weight, k)
    _need_cuda(q)
    q, k, v = _rows(q), _rows(k), _rows(v)
    table = block_table if block_table.stride(-1) == 1 or block_table.shape[1] < 2 else block_table.contiguous()
    lens = cache_seqlens.contiguous()
    cu = None if cu_seqlens is None else cu_seqlens.contiguous()
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    cache = (table.data_ptr(), lens.data_ptr(), 0 if cu is None else cu.data_ptr(), table.stride(0))
    sizes = (n, k_cache.shape[0], k_cache.shape[1], table.shape[1])
    tensors = [_tensor(q, wq, out), _paged(k, wk, k_cache, _TURN), _paged(v, None, v_cache, 0)]
    lib, stream = _lib.load(), _lib.stream_of(q.device)
    with _lib.on(q.device):
        if v.shape[-1] != q.shape[-1]:             # v's rows alone: their head size is another
            V = _params(v, tensors[2:], _Cfg(0, 0, False, 0.0, 1.0), None, None, cache, sizes)
            _lib.check(lib.sfa_rotary_fwd(ctypes.byref(V), stream), "sfa_rotary_fwd (append)")
            tensors = tensors[:2]
        P = _params(q, tensors, cfg, positions, frequencies, cache, sizes)
        _lib.check(lib.sfa_rotary_fwd(ctypes.byref(P), stream), "sfa_rotary_fwd (append)")
    return out
