"""The several-axes rotary at positions of any size, against exact angles: whole
numbers times the frequencies' rational values, reduced by pi to 400 bits."""
import math
from fractions import Fraction

import pytest
import torch

pytestmark = pytest.mark.gpu
F32 = torch.float32


def pi():
    """Machin's formula in whole numbers, to 400 bits."""
    one = 1 << 420

    def arctan(n):   # of 1 / n
        x, s, k = one // n, 0, 1
        while x:
            s += -(x // k) if k & 2 else x // k
            x //= n * n
            k += 2
        return s

    return Fraction(4 * (4 * arctan(5) - arctan(239)), one)


PI = pi()


def turn(p, f):
    """cos and sin of p * f, p a whole number and f fp32."""
    half = Fraction(p) * Fraction(f) / PI
    half -= 2 * round(half / 2)
    return math.cos(float(half) * math.pi), math.sin(float(half) * math.pi)


FAR = [0, 1, -1, 1000, 100_003, 2 ** 24 + 1, -(2 ** 28) - 3, 2 ** 31 - 1, -2 ** 31]
FARTHER = [2 ** 31, 2 ** 32 - 1, 2 ** 32, -2 ** 32 - 1, 10 ** 12 + 7, -(10 ** 15) - 1, 2 ** 53 + 1, -(2 ** 53) - 3,
           2 ** 62 + 12345, 2 ** 63 - 1, 2 ** 63 - 600, -2 ** 63]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("pos_type", [torch.int32, torch.int64])
def test_exact_angles(pos_type, interleaved):
    """Per element 8 * 2^-24 of the pair's length: the angle's rounding to fp32
    half turns (pi 2^-24), sine and cosine (2 * 2^-24) and three operations."""
    from uttt_amd.positions import axis_frequencies, rotary_axes
    where = FAR + (FARTHER if pos_type == torch.int64 else [])
    sections = [20, 12]
    freq = torch.cat([axis_frequencies([20], base=500000.0), torch.tensor([1.0, 0.1, 3.0, 7.77, 1e-8, 1e3, 0.5, 2.0 ** -20,
                                                                         math.pi, math.pi / 2, 1 / math.pi, 100.0])])
    R, L = 32, len(where)
    pos = torch.tensor([[where[i], where[-1 - i]] for i in range(L)]).to(pos_type)
    x = torch.randn(1, L, 3, 64, generator=torch.Generator().manual_seed(0))
    angles = torch.tensor([[turn(where[i] if j < 20 else where[-1 - i], float(f)) for j, f in enumerate(freq.tolist())]
                           for i in range(L)], dtype=torch.float64)
    cos, sin = angles[..., 0][:, None], angles[..., 1][:, None]
    a, b = (slice(0, 2 * R, 2), slice(1, 2 * R, 2)) if interleaved else (slice(0, R), slice(R, 2 * R))
    y = rotary_axes(x.cuda(), pos.cuda(), freq.cuda(), sections, interleaved=interleaved).cpu().double()[0]
    u, w = x[0, ..., a].double(), x[0, ..., b].double()
    size = 8 * 2.0 ** -24 * (u.square() + w.square()).sqrt()
    for got, ref in ((y[..., a], u * cos - w * sin), (y[..., b], u * sin + w * cos)):
        off = (got - ref).abs()
        assert (off <= size + 2.0 ** -24 * ref.abs()).all(), [
            (where[i], (off / size)[i].max().item()) for i in (off > size).flatten(1).any(1).nonzero().flatten().tolist()]
