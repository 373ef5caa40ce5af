"""Edges of the operators that serve many requests, on the GPU."""
import math
from fractions import Fraction

import pytest
import torch

from flyai_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _two_pi(bits):
    """2 pi as a Fraction, good to 2^-bits: pi = 16 atan(1/5) - 4 atan(1/239) in integers."""
    one = 1 << (bits + 16)

    def atan_inverse(n):
        total, term, k = 0, one // n, 1
        while term:
            total += term // k if k % 4 == 1 else -(term // k)
            term //= n * n
            k += 2
        return total

    return 2 * Fraction(16 * atan_inverse(5) - 4 * atan_inverse(239), one)


def _exact_cos_sin(position, frequency, two_pi):
    """cos and sin of position * frequency, the product and its remainder by 2 pi exact: off by the 2^-51 or so of a double's
    remainder and its cos and sin."""
    angle = Fraction(position) * Fraction(frequency)
    rest = float(angle - round(angle / two_pi) * two_pi)
    return math.cos(rest), math.sin(rest)


def test_rope_angles_are_exact_at_far_positions():
    """cos and sin of the exact angle, read off the pair (1, 0), at frequencies and positions where the product's own rounding to 64
    bits is up to 2^-23.

    Tolerance, in units of u = 2^-25 (half an fp32 step in [0.5, 1)): the reduced angle's rounding u, times at most 0.88 in sin and
    0.71 in cos; the last fma's rounding u; in cos the rounding of z = r^2 under 0.62, u / 2 of the result, and its polynomial's,
    u / 2 times 0.62; in sin that of r^3's polynomial, u / 4 times 0.49 and what r z < 0.49 loses, u / 2 / 6.  The Taylor rest
    is 2e-9 = 0.07 u.  Below 2.6 u; 3 u is asked for."""
    g = torch.Generator().manual_seed(3)
    freq = torch.rand(64, generator=g, dtype=torch.float64) * 0.5 + 0.5
    pos = torch.randint(2 ** 31 - 10 ** 6, 2 ** 31, (24,), generator=g, dtype=torch.int64)
    pos[:4] = torch.tensor([2 ** 31 - 1, -2 ** 31, 2 ** 30 + 1, 10 ** 9 + 7])
    two_pi = _two_pi(160)
    want = torch.tensor([[_exact_cos_sin(int(p), float(f), two_pi) for f in freq] for p in pos], dtype=torch.float64)
    x = torch.zeros(len(pos), 1, 128, device=DEV)
    x[..., 0::2] = 1.0
    y = ops.rope(x, pos.to(torch.int32).to(DEV), freq.to(DEV), layout="interleaved").double().cpu()
    err = (y.view(len(pos), 64, 2) - want).abs()
    assert float(err.max()) <= 3 * 2.0 ** -25, float(err.max()) * 2 ** 25
