"""Append refuses caches whose rows, heads or pools share elements, and takes
every layout in which none do; checked against the addresses themselves."""
import random

import pytest
import torch

import ops_b200
from ops_b200.rotary import _pools_meet, _rows_meet
from test_rotary_host import append_args


def addresses(first, rows, heads, d, st, sh):
    return [first + i * st + j * sh + e for i in range(rows) for j in range(heads) for e in range(d)]


def test_rows_and_heads_against_addresses():
    r, seen = random.Random(1), {True: 0, False: 0}
    for _ in range(6000):
        rows, heads, d, st, sh = r.randint(1, 7), r.randint(1, 5), r.randint(1, 4), r.randint(0, 24), r.randint(0, 24)
        a = addresses(0, rows, heads, d, st, sh)
        want = len(set(a)) < len(a)
        assert _rows_meet(rows, heads, d, st, sh) == want, (rows, heads, d, st, sh)
        seen[want] += 1
    assert min(seen.values()) > 500


def test_pools_against_addresses():
    r, seen = random.Random(2), {True: 0, False: 0}
    for _ in range(20000):
        rows, heads, dk, dv, st = r.randint(1, 6), r.randint(1, 4), r.randint(1, 4), r.randint(1, 4), r.randint(1, 30)
        ksh = r.randint(0, 30)
        vsh = ksh if r.random() < 0.6 else r.randint(0, 30)
        k, v = (100, st, ksh, dk), (100 + r.randint(-60, 60), st, vsh, dv)
        ak, av = (set(addresses(p[0], rows, heads, p[3], p[1], p[2])) for p in (k, v))
        if any(_rows_meet(rows, heads, p[3], p[1], p[2]) for p in (k, v)):
            continue                              # refused before
        want = bool(ak & av)
        assert _pools_meet(rows, heads, k, v) == want, (rows, heads, k, v)
        seen[want] += 1
    assert min(seen.values()) > 500


N, PAGE, H, D = 5, 8, 2, 64
BUF = torch.zeros(4 * N * PAGE * H * D)


def pool(st, sh, at=0):
    return BUF.as_strided((N, PAGE, H, D), (PAGE * st, st, sh, 1), at)


BOTH = torch.zeros(N, PAGE, H, 2, D)
PAIR = torch.zeros(N, PAGE, 2, H, D)
WIDE = torch.zeros(N, PAGE, H * D + H * 32)
OUTER = torch.zeros(H, 2, N * PAGE, D)


@pytest.mark.parametrize("k,v,msg", [
    (pool(D, D), None, "rows and heads must not overlap"),             # row 1 of a head is row 0 of the next
    (None, pool(D, D), "rows and heads must not overlap"),
    (pool(D, 7 * D), None, "rows and heads must not overlap"),
    (pool(H * D, D), pool(H * D, D, H * D), "share elements"),         # v one row further on
    (pool(H * D, D, D), pool(H * D, D), "share elements"),
    (pool(2 * H * D, D), pool(2 * H * D, D, D), "share elements"),
    (pool(H * D, D), pool(2 * H * D, D, H * D), "share elements"),
    (BOTH[:, :, :, 0], BOTH[:, :, :, 1], "CUDA"), (BOTH[:, :, :, 1], BOTH[:, :, :, 0], "CUDA"),
    (PAIR[:, :, 0], PAIR[:, :, 1], "CUDA"), (PAIR[:, :, 1], PAIR[:, :, 0], "CUDA"),
    (OUTER[:, 0].view(H, N, PAGE, D).permute(1, 2, 0, 3), OUTER[:, 1].view(H, N, PAGE, D).permute(1, 2, 0, 3), "CUDA"),
    (pool(H * D, D), pool(H * D, D, N * PAGE * H * D), "CUDA"),
])
def test_layouts(k, v, msg):
    bad = {n: c for n, c in (("k_cache", k), ("v_cache", v)) if c is not None}
    with pytest.raises(ValueError, match=msg):
        ops_b200.qk_norm_rotary_append(**{**append_args(), **bad})


def test_values_of_another_size_in_one_buffer():
    k, v = WIDE[..., :H * D].unflatten(-1, (H, D)), WIDE[..., H * D:].unflatten(-1, (H, 32))
    with pytest.raises(ValueError, match="CUDA"):
        ops_b200.qk_norm_rotary_append(**{**append_args(), "v": torch.zeros(3, H, 32), "k_cache": k, "v_cache": v})
    with pytest.raises(ValueError, match="share elements"):
        late = WIDE[..., H * D - 8:-8].unflatten(-1, (H, 32))
        ops_b200.qk_norm_rotary_append(**{**append_args(), "v": torch.zeros(3, H, 32), "k_cache": k, "v_cache": late})
