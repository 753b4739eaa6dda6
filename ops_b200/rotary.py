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
    return (x.stride(0), x.stride(1), x.stride(2)) if x.dim() == 4 else (0, x.stride(0), x.stride(1))


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
        rot = 2 * frequencies.numel()
        frequencies = frequencies.contiguous()
        try:
            positions = positions.expand(x.shape[:-2])
        except RuntimeError:
            raise ValueError(f"positions {tuple(positions.shape)} do not broadcast to tokens {tuple(x.shape[:-2])}")
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
    return w.float().contiguous()


def _params(x: torch.Tensor, cfg: _Cfg, positions, frequencies) -> SfaRotaryParams:
    P = SfaRotaryParams()
    P.batch, P.len = (x.shape[0], x.shape[1]) if x.dim() == 4 else (1, x.shape[0])
    P.dim, P.dtype = x.shape[-1], _DTYPE[x.dtype]
    P.rot, P.start, P.interleaved = cfg.rot, cfg.start, 1 if cfg.interleaved else 0
    P.eps, P.amplitude = cfg.eps, cfg.amplitude
    if positions is not None:
        P.positions, P.frequencies = positions.data_ptr(), frequencies.data_ptr()
        P.pos64 = 1 if positions.dtype == torch.int64 else 0
        P.p_sb, P.p_st = (positions.stride(0), positions.stride(1)) if positions.dim() == 2 else (0, positions.stride(0))
    return P


def _fill(t, x, w, turned: bool = True) -> None:
    t.x, t.heads = x.data_ptr(), x.shape[-2]
    t.x_sb, t.x_st, t.x_sh = _strides(x)
    t.weight = None if w is None else w.data_ptr()
    t.flags = _lib.SFA_ROTARY_TURN if turned else 0


def _stream(x: torch.Tensor) -> int:
    return torch.cuda.current_stream(x.device).cuda_stream


class _NormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, positions, frequencies, cfg: _Cfg):
        lib = _lib.load()
        P = _params(q, cfg, positions, frequencies)
        outs = []
        for i, (x, w) in enumerate(((q, wq), (k, wk))):
            if x is None:
                break
            y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            _fill(P.t[i], x, w)
            P.t[i].y = y.data_ptr()
            P.t[i].y_sb, P.t[i].y_st, P.t[i].y_sh = _strides(y)
            outs.append(y)
        P.num_tensors = len(outs)
        with torch.cuda.device(q.device):
            _lib.check(lib.sfa_rotary_fwd(ctypes.byref(P), _stream(q)), "sfa_rotary_fwd")
        ctx.save_for_backward(q, k, wq, wk, positions, frequencies)
        ctx.cfg = cfg
        return tuple(outs) if k is not None else outs[0]

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        q, k, wq, wk, positions, frequencies = ctx.saved_tensors
        lib = _lib.load()
        P = _params(q, ctx.cfg, positions, frequencies)
        need = ctx.needs_input_grad
        out = [None] * 7
        held = []
        n = 0
        for i, (x, w) in enumerate(((q, wq), (k, wk))):
            if x is None or not (need[i] or need[2 + i]):
                continue
            dy = _rows(grads[i])
            dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            dw = torch.empty_like(w) if w is not None and need[2 + i] else None
            t = P.t[n]
            _fill(t, x, w)
            t.dy, t.dx, t.dweight = dy.data_ptr(), dx.data_ptr(), None if dw is None else dw.data_ptr()
            t.dy_sb, t.dy_st, t.dy_sh = _strides(dy)
            t.dx_sb, t.dx_st, t.dx_sh = _strides(dx)
            out[i], out[2 + i] = dx, dw
            held.append(dy)
            n += 1
        P.num_tensors = n
        if n:
            with torch.cuda.device(q.device):
                nbytes = lib.sfa_rotary_bwd_workspace_bytes(ctypes.byref(P))
                ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=q.device)
                _lib.check(lib.sfa_rotary_bwd(ctypes.byref(P), ws.data_ptr(), nbytes, _stream(q)), "sfa_rotary_bwd")
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
    with torch.no_grad():
        q, k, v = _rows(q), _rows(k), _rows(v)
        table = block_table if block_table.stride(-1) == 1 or block_table.shape[1] < 2 else block_table.contiguous()
        lens = cache_seqlens.contiguous()
        cu = None if cu_seqlens is None else cu_seqlens.contiguous()
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        P = _params(q, cfg, positions, frequencies)
        same = v.shape[-1] == q.shape[-1]
        pools = ((P.t[1], k, wk, k_cache, True), (P.t[2], v, None, v_cache, False))
        _fill(P.t[0], q, wq)
        P.t[0].y = out.data_ptr()
        P.t[0].y_sb, P.t[0].y_st, P.t[0].y_sh = _strides(out)
        for t, x, w, c, turned in pools:
            _fill(t, x, w, turned)
            t.flags |= _lib.SFA_ROTARY_PAGED
            t.y, t.y_sb, t.y_st, t.y_sh = c.data_ptr(), 0, c.stride(1), c.stride(2)
        P.block_table, P.bt_stride, P.table_width = table.data_ptr(), table.stride(0), table.shape[1]
        P.cache_seqlens, P.cu_seqlens = lens.data_ptr(), None if cu is None else cu.data_ptr()
        P.num_seqs, P.num_pages, P.page_size = n, k_cache.shape[0], k_cache.shape[1]
        P.num_tensors = 3 if same else 2
        lib = _lib.load()
        with torch.cuda.device(q.device):
            if not same:                       # v's rows alone: its head size is another
                V = SfaRotaryParams.from_buffer_copy(P)
                V.t[0], V.num_tensors, V.dim, V.rot, V.start = P.t[2], 1, v.shape[-1], 0, 0
                _lib.check(lib.sfa_rotary_fwd(ctypes.byref(V), _stream(q)), "sfa_rotary_fwd (append)")
            _lib.check(lib.sfa_rotary_fwd(ctypes.byref(P), _stream(q)), "sfa_rotary_fwd (append)")
    return out
