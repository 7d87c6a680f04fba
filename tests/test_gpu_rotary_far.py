"""Angles of any size: positions to the end of int32, frequencies above one, without the norms, whose roundings would hide an angle's.  The definition takes the float64 product position * frequency, reduced
here by the whole turns in it with a hundred digits of pi.

Bound: as for the rotation elsewhere, 2^-21 of a pair's length (sine and cosine in float32, two products, a sum) and one rounding at the end; nothing of it grows with the angle."""
from fractions import Fraction
from math import cos, sin

import pytest
import torch

from dinoml_v2_b200 import kernels
from oracle import decoder as D

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
TURN = 2 * Fraction(31415926535897932384626433832795028841971693993751058209749445923078164062862089986280348253421170679, 10 ** 100)


def _reduced(angle):
    exact = Fraction(angle)
    return float(exact - round(exact / TURN) * TURN)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("scale", [1.0, 0.37, 50.0, 1e6])
def test_far_positions(scale, interleaved, dtype):
    positions = [0, 1, 131071, (1 << 20) + 7, (1 << 24) + 1, 1234567891, (1 << 31) - 1]
    f = kernels.rotary_frequencies(64, 500000.0, scale=scale)
    g = torch.Generator(device=DEV)
    g.manual_seed(2)
    x = torch.randn(len(positions), 3, 64, device=DEV, generator=g).to(getattr(torch, dtype))
    got, _ = kernels.rotary(x, None, torch.tensor(positions, dtype=torch.int32, device=DEV), f, interleaved=interleaved)
    angles = [[_reduced(float(p) * v) for v in f.tolist()] for p in positions]
    c, s = (torch.tensor([[turn(a) for a in row] for row in angles], dtype=torch.float64)[:, None] for turn in (cos, sin))
    y = x.cpu().double()
    a, b = (y[..., ::2], y[..., 1::2]) if interleaved else (y[..., :32], y[..., 32:])
    want = torch.stack((a * c - b * s, b * c + a * s), -1 if interleaved else -2).flatten(-2)
    size = torch.stack((torch.hypot(a, b),) * 2, -1 if interleaved else -2).flatten(-2)
    inside = 2.0 ** -21
    assert ((got.cpu().double() - want).abs() <= D.UNIT[dtype] * (want.abs() + inside * size) + inside * size + D.SMALLEST[dtype]).all()
    assert torch.equal(got[0], x[0])
