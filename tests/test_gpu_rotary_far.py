"""GPU: rotary positions of any size, against angles reduced in whole numbers.

Tolerance: that of a forward near the origin (tests/test_gpu_rotary.py): the
angle's fraction of a turn is exact, so an element is off by 64 units of 2^-24
of the pair's size, at most twice the row's largest element."""
import math
from fractions import Fraction

import pytest
import torch

import ops_b200
from oracle.rotary_oracle import pair_columns

pytestmark = pytest.mark.gpu

BITS = 320


def turns_per_radian():
    """1 / (2 pi) as a whole number of 2^-BITS, from Machin's formula."""
    one = 1 << (BITS + 64)

    def arctan_inverse(n):
        total, term, k = 0, one // n, 0
        while term:
            total += (-1) ** k * (term // (2 * k + 1))
            term //= n * n
            k += 1
        return total

    pi = 4 * (4 * arctan_inverse(5) - arctan_inverse(239))
    return (one << BITS) // (2 * pi)


def angles(positions, frequencies):
    """Position times frequency modulo 2 pi, reduced exactly and rounded to 64 bits."""
    inv = turns_per_radian()
    out = torch.empty(len(positions), len(frequencies), dtype=torch.float64)
    for j, f in enumerate(frequencies):
        f = Fraction(f)                          # a double is a fraction of whole numbers
        for i, p in enumerate(positions):
            turns = f.numerator * p * inv // f.denominator % (1 << BITS)
            out[i, j] = 2 * math.pi * ((turns >> (BITS - 62)) / 2.0 ** 62)
    return out


FAR = [0, 1, -1, 2 ** 31 - 1, -2 ** 31, 2 ** 40 + 12345, -(2 ** 41) - 7, 2 ** 50 + 3, 10 ** 17 + 1, 2 ** 62 + 999, 2 ** 63 - 1, -2 ** 63]


@pytest.mark.parametrize("dim,rot,start,inter", [(64, 64, 0, False), (64, 32, 32, True), (576, 64, 512, False), (30, 10, 3, True)])
def test_far_positions(dim, rot, start, inter):
    f = ops_b200.rotary_frequencies(rot)[0]
    f[1], f[2], f[3] = 1.0, -0.7, 123.456        # a whole radian, a backward turn, many turns a position
    x = torch.randn(len(FAR), 3, dim, generator=torch.Generator().manual_seed(2))
    gx = x.cuda().requires_grad_()
    y = ops_b200.rotary_embedding(gx, torch.tensor(FAR).cuda(), f.cuda(), interleaved=inter, start=start)
    dx, = torch.autograd.grad(y, gx, x.cuda())
    angle = angles(FAR, f.tolist())[:, None]
    a, b = pair_columns(rot, start, inter)
    for got, sign in ((y, 1.0), (dx, -1.0)):
        ref = x.double().clone()
        c, s = torch.cos(angle), sign * torch.sin(angle)
        ref[..., a] = x.double()[..., a] * c - x.double()[..., b] * s
        ref[..., b] = x.double()[..., b] * c + x.double()[..., a] * s
        u = 2.0 ** -24
        tol = u * ref.abs() + 64 * u * 2 * ref.abs().amax(-1, keepdim=True) * (1 + u)
        off = ((got.detach().double().cpu() - ref).abs() / tol).amax((1, 2))
        assert float(off.max()) <= 1.0, [f"{p}: {float(v):.3g}" for p, v in zip(FAR, off)]


def test_int32_positions_agree_with_int64():
    pos = torch.tensor([p for p in FAR if -2 ** 31 <= p < 2 ** 31], dtype=torch.int32, device="cuda")
    f = ops_b200.rotary_frequencies(64, device="cuda")[0]
    x = torch.randn(len(pos), 2, 64, generator=torch.Generator().manual_seed(3)).cuda()
    a, b = (ops_b200.rotary_embedding(x, p, f).double() for p in (pos, pos.long()))
    # 2^31 positions of at most half a step of 2^-64 turns each: 2^-34 turns, far below the angle's own rounding,
    # which may fall the other way: pi 2^-24 of a pair's size
    assert ((a - b).abs() <= 4 * 2.0 ** -24 * 2 * x.double().abs().amax(-1, keepdim=True)).all()
