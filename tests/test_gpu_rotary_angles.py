"""Angles of rotary positions against position * frequency in whole numbers, apart from how the kernel holds a frequency."""
import math
from fractions import Fraction

import numpy as np
import pytest
import torch

from sddmm_gpu_b200 import api

pytestmark = pytest.mark.gpu


def _pi(bits):
    """pi 2^bits, by Machin's formula."""
    def arctan(k):
        term, total, i, sign = (1 << bits + 32) // k, 0, 1, 1
        while term:
            total += sign * (term // i)
            term //= k * k
            i, sign = i + 2, -sign
        return total
    return 4 * (4 * arctan(5) - arctan(239)) >> 32


TWO_PI = Fraction(2 * _pi(512), 1 << 512)
FREQUENCIES = [1.0, 100.0, 6.2, 6.4, 1e6, 12345.678, 2.0 ** 40 + 0.5, 2.0 ** 63 * 1.1, -3.7, -1e-3, 2.0 ** -20, 1e-9, 5e-324, 0.0]
POSITIONS = [0, 1, -1, 4095, 1 << 20, (1 << 31) + 5, -(1 << 31) - 7, 10 ** 10, (1 << 38) - 1, 10 ** 12, -(10 ** 12)]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("inverse", [False, True])
def test_near_and_far(engine, layout, inverse):
    n = len(FREQUENCIES)
    g = torch.Generator("cuda").manual_seed(7)
    x = torch.randn((len(POSITIONS), 2, 2 * n), device="cuda", generator=g)
    y = torch.empty_like(x)
    engine.rotary([api.RotaryPart(x, y)], torch.tensor(POSITIONS, device="cuda"), np.array(FREQUENCIES), layout, inverse)
    turn = [[Fraction(t) * Fraction(f) / TWO_PI % 1 for f in FREQUENCIES] for t in POSITIONS]
    angle = torch.tensor([[float(v) * 2 * math.pi for v in row] for row in turn], dtype=torch.float64, device="cuda")[:, None]
    c, s = angle.cos(), angle.sin() * (-1 if inverse else 1)
    a, b = (x[..., 0::2], x[..., 1::2]) if layout == "interleaved" else (x[..., :n], x[..., n:])
    u, w = (y[..., 0::2], y[..., 1::2]) if layout == "interleaved" else (y[..., :n], y[..., n:])
    a, b = a.double(), b.double()
    # the angle: |t| 2^-64 turns, 2^-25 of half a turn and 2^-31 below its argument's bits, 2^-51 here; sine and cosine 2 units, two products, a sum: 5 x 2^-24
    off = torch.tensor(POSITIONS, dtype=torch.float64, device="cuda").abs()[:, None, None] * 2.0 ** -64 * 2 * math.pi
    tol = (a.abs() + b.abs()) * (off + math.pi * (2.0 ** -25 + 2.0 ** -31) + 2.0 ** -48 + 5 * 2.0 ** -24)
    assert bool(((u.double() - (a * c - b * s)).abs() <= tol).all())
    assert bool(((w.double() - (b * c + a * s)).abs() <= tol).all())


@pytest.mark.parametrize("f", [2.0 ** 64, -2.0 ** 64, 1e300, math.inf, math.nan])
def test_frequencies_that_are_refused(engine, f):
    x = torch.zeros((3, 1, 4), device="cuda")
    with pytest.raises(api.SddmmError) as e:
        engine.rotary([api.RotaryPart(x)], 0, np.array([1.0, f]))
    assert e.value.status == api.INVALID_ARG
