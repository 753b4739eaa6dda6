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
from typing import NamedTuple, Optional, Tuple

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
      linearly in their number of turns, as the method was published; the
      amplitude is ``0.1 ln(factor) + 1``.  Checkpoints made with the public
      implementation blend linearly in the pair's index between the two pairs
      that turn ``beta_fast`` and ``beta_slow`` times instead, which gives the
      pairs between other frequencies: pass theirs as ``frequencies``.
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


class _Cfg(NamedTuple):
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
    shape = x.shape
    if not 3 <= len(shape) <= 4 or shape[-2] < 1 or shape[-1] < 1:
        raise ValueError(f"{name} must be [B, T, H, D] or [T, H, D] with at least one head and dim")
    if like is not None and (x.dtype != like.dtype or x.device != like.device or shape[:-2] != like.shape[:-2]
                             or shape[-1] != like.shape[-1]):
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
    return w if w.dtype is torch.float32 and w.is_contiguous() else w.float().contiguous()


_pack = _lib.packer(SfaRotaryParams)
_TURN, _PAGED = _lib.SFA_ROTARY_TURN, _lib.SFA_ROTARY_PAGED
_NO_TENSOR = (0,) * 20
_NO_CACHE = (0, 0, 0, 0)


def _tensor(x, w, y=None, dy=None, dx=None, dw=None):
    """The values of one SfaRotaryTensor: y forward, dy and dx backward."""
    head = (x.data_ptr(), 0 if y is None else y.data_ptr(), 0 if dy is None else dy.data_ptr(),
            0 if dx is None else dx.data_ptr(), 0 if w is None else w.data_ptr(), 0 if dw is None else dw.data_ptr())
    if y is not None:
        return head + _strides(x) + _strides(y) + (0, 0, 0, 0, 0, 0, x.shape[-2], _TURN)
    return head + _strides(x) + (0, 0, 0) + _strides(dy) + _strides(dx) + (x.shape[-2], _TURN)


def _paged(x, w, pool, stride, turned):
    """The values of one SfaRotaryTensor that goes into a page pool."""
    xs = x.stride()
    return (x.data_ptr(), pool.data_ptr(), 0, 0, 0 if w is None else w.data_ptr(), 0, 0, xs[0], xs[1], 0, stride[1],
            stride[2], 0, 0, 0, 0, 0, 0, x.shape[1], turned | _PAGED)


def _params(x: torch.Tensor, tensors, cfg: _Cfg, positions, frequencies, cache=_NO_CACHE, sizes=_NO_CACHE) -> SfaRotaryParams:
    shape = x.shape
    batch, length = (shape[0], shape[1]) if len(shape) == 4 else (1, shape[0])
    if positions is None:
        pos, freq, sb, st, p64 = 0, 0, 0, 0, 0
    else:
        pos, freq, p64 = positions.data_ptr(), frequencies.data_ptr(), int(positions.dtype == torch.int64)
        ps = positions.stride()
        sb, st = ps if len(ps) == 2 else (0, ps[0])
    n = len(tensors)
    return _pack(*tensors[0], *(tensors[1] if n > 1 else _NO_TENSOR), *(tensors[2] if n > 2 else _NO_TENSOR), pos, freq,
                 *cache, sb, st, n, batch, length, shape[-1], cfg.rot, cfg.start, int(cfg.interleaved), _DTYPE[x.dtype],
                 p64, *sizes, cfg.eps, cfg.amplitude, 0)


class _NormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, positions, frequencies, cfg: _Cfg):
        oq = torch.empty_like(q, memory_format=torch.contiguous_format)
        tensors = [_tensor(q, wq, oq)]
        if k is not None:
            ok = torch.empty_like(k, memory_format=torch.contiguous_format)
            tensors.append(_tensor(k, wk, ok))
        P, device = _params(q, tensors, cfg, positions, frequencies), q.device
        with _lib.on(device):
            _lib.check(_lib.load().sfa_rotary_fwd(ctypes.byref(P), _lib.stream_of(device)), "sfa_rotary_fwd")
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
    ``positions`` (int32 or int64) broadcast to the tokens.  Differentiable in x.
    Head sizes, rotated parts and starts that are not multiples of 8, and rows
    that are not aligned to 8 bytes (fp32: 16), take a kernel about five times slower."""
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


def _check_pool(name: str, c: torch.Tensor, like: torch.Tensor):
    """A page pool's shape and strides."""
    if c.dim() != 4 or c.device != like.device:
        raise ValueError(f"{name} must be a [num_pages, page_size, H, D] page pool on the inputs' device")
    shape, stride = c.shape, c.stride()
    pages, page, _, d = shape
    if d > 1 and stride[3] != 1 or pages > 1 and stride[0] != page * stride[1]:
        raise ValueError(f"{name}: pages must be [page_size, H, D] row ranges of one pool, innermost dim contiguous")
    return shape, stride


def _rows_meet(rows: int, heads: int, d: int, st: int, sh: int) -> bool:
    """Whether different rows or heads of a pool share elements."""
    if rows > 1 and st < d or heads > 1 and sh < d:
        return True
    if rows < 2 or heads < 2 or st >= (heads - 1) * sh + d or sh >= (rows - 1) * st + d:
        return False                       # heads inside a row, or rows inside a head
    for j in range(1, heads):              # a head j further on, and the rows around it
        i, r = divmod(j * sh, st)
        if i < rows and r < d or i + 1 < rows and st - r < d:
            return True
    return False


def _pools_meet(rows: int, heads: int, k, v) -> bool:
    """Whether two pools share elements; k and v: (first element, row stride, head
    stride, head size), all in elements."""
    (k0, kst, ksh, dk), (v0, vst, vsh, dv) = k, v
    if rows < 1 or v0 >= k0 + (rows - 1) * kst + (heads - 1) * ksh + dk or k0 >= v0 + (rows - 1) * vst + (heads - 1) * vsh + dv:
        return False
    if rows > 1 and kst != vst:
        return True                        # one inside the other with rows of its own: not a layout of two pools
    st, at = kst if rows > 1 else max(kst, vst, 1), v0 - k0
    r = at % st
    if (heads - 1) * ksh + dk <= r and r + (heads - 1) * vsh + dv <= st:
        return False                       # [rows, 2, heads, D]
    if ksh == vsh and ksh > 0 and st % ksh == 0 and dk <= r % ksh and r % ksh + dv <= ksh:
        return False                       # [rows, heads, 2, D]
    for a in range(heads):
        for b in range(heads):
            x = at + b * vsh - a * ksh     # head b of v behind head a of k; rows i apart move it by i * st
            for i in range(-((x + dv - 1) // st), (dk - 1 - x) // st + 1):
                if -rows < i < rows:
                    return True
    return False


def _check_table(block_table: torch.Tensor, cache_seqlens: torch.Tensor, like: torch.Tensor):
    """(sequences, pages of a row of the table)."""
    for name, t, d in (("block_table", block_table, 2), ("cache_seqlens", cache_seqlens, 1)):
        if t.dtype != torch.int32 or t.dim() != d or t.device != like.device:
            raise ValueError(f"{name} must be a {d}-D int32 tensor on the inputs' device")
    n, width = block_table.shape
    if cache_seqlens.shape[0] != n:
        raise ValueError("block_table and cache_seqlens must name the same number of sequences")
    return n, width


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
    qs, ks, vs, dtype, device = q.shape, k.shape, v.shape, q.dtype, q.device
    for name, x, shape in (("q", q, qs), ("k", k, ks), ("v", v, vs)):
        _check(name, x)
        if len(shape) != 3 or x.dtype != dtype or x.device != device or shape[0] != qs[0]:
            raise ValueError(f"{name} must be [total, H, D] with q's type, device and rows")
    if ks[2] != qs[2] or vs[1] != ks[1]:
        raise ValueError("k must have q's head size and v must have k's heads")
    pools = []
    for name, c, rows in (("k_cache", k_cache, ks), ("v_cache", v_cache, vs)):
        pools.append(_check_pool(name, c, q))
        (n, m, h, d), (_, st, sh, _) = pools[-1]
        if c.dtype != dtype or h != rows[1] or d != rows[2]:
            raise ValueError(f"{name} must have the type, heads and head size of the rows stored into it")
        if _rows_meet(n * m, h, d, st, sh):
            raise ValueError(f"{name}: rows and heads must not overlap, they are stored into")
    (num_pages, page, _, _), kst = pools[0]
    (v_pages, v_page, _, _), vst = pools[1]
    if v_pages != num_pages or v_page != page:
        raise ValueError("k_cache and v_cache must have the same pages")
    if k_cache.data_ptr() == v_cache.data_ptr() != 0:
        raise ValueError("k_cache and v_cache must not be the same memory")
    size = dtype.itemsize
    if _pools_meet(num_pages * page, ks[1], (k_cache.data_ptr() // size, kst[1], kst[2], ks[2]),
                   (v_cache.data_ptr() // size, vst[1], vst[2], vs[2])):
        raise ValueError("k_cache and v_cache must not share elements")
    n, width = _check_table(block_table, cache_seqlens, q)
    if cu_seqlens is None:
        if qs[0] != n:
            raise ValueError("without cu_seqlens, q must hold one row per sequence")
    elif cu_seqlens.dtype != torch.int32 or cu_seqlens.shape != (n + 1,) or cu_seqlens.device != device:
        raise ValueError("cu_seqlens must be int32 [n + 1] on the inputs' device")
    cfg, positions, frequencies = _check_turn(q, positions, frequencies, interleaved, start, eps, amplitude)
    wq, wk = _weight("q_weight", q_weight, q), _weight("k_weight", k_weight, k)
    _need_cuda(q)
    q, k, v = _rows(q), _rows(k), _rows(v)
    table = block_table if width < 2 or block_table.stride(1) == 1 else block_table.contiguous()
    lens = cache_seqlens.contiguous()
    cu = None if cu_seqlens is None else cu_seqlens.contiguous()
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    cache = (table.data_ptr(), lens.data_ptr(), 0 if cu is None else cu.data_ptr(), table.stride(0))
    sizes = (n, num_pages, page, width)
    tensors = [_tensor(q, wq, out), _paged(k, wk, k_cache, kst, _TURN), _paged(v, None, v_cache, vst, 0)]
    lib, stream = _lib.load(), _lib.stream_of(device)
    with _lib.on(device):
        if vs[2] != qs[2]:             # v's rows alone: their head size is another
            V = _params(v, tensors[2:], _Cfg(0, 0, False, 0.0, 1.0), None, None, cache, sizes)
            _lib.check(lib.sfa_rotary_fwd(ctypes.byref(V), stream), "sfa_rotary_fwd (append)")
            tensors = tensors[:2]
        P = _params(q, tensors, cfg, positions, frequencies, cache, sizes)
        _lib.check(lib.sfa_rotary_fwd(ctypes.byref(P), stream), "sfa_rotary_fwd (append)")
    return out
