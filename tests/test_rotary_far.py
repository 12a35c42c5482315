"""Angles of far positions: the stated bound, and positions beyond 32 bits."""
from __future__ import annotations

import math
import random
from fractions import Fraction

import numpy as np
import pytest
import torch

from cache_util import BF16_HALF_STEP, randn
from min_fa3_demo_b200 import min_fa3_op as op, rotary

PI = Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")
FREQ = [1e6 ** (-i / 64) for i in range(64)]


def turn_left_over(position, freq):
    """Exact fraction of a turn, in [-1/2, 1/2)."""
    t = Fraction(position) * Fraction(freq) / (2 * PI)
    t -= math.floor(t)
    return t - 1 if t >= Fraction(1, 2) else t


def bound(position):
    """In turns: 32 of 64 bits are used (2^-32) and rounded to the 24 of a float (2^-26); the frequency's fraction is off by half of 2^-64."""
    return Fraction(1, 2**26) + Fraction(1, 2**32) + abs(position) * Fraction(1, 2**65)


def test_the_angle_is_within_its_bound():
    rng = random.Random(0)
    worst = 0.0
    for _ in range(20000):
        position = rng.choice([-1, 1]) * rng.randrange(1 << rng.randrange(1, 50))
        freq = rng.choice(FREQ)
        turns = (position * rotary._turn(freq)) % 2**64
        high = turns >> 32
        # What the kernel does: the upper half as a signed number, in float, times 2^-31 half turns.
        ours = Fraction(float(np.float32(np.int32(high - 2**32 if high >= 2**31 else high)))) / 2**32
        off = abs(ours - turn_left_over(position, freq))
        off = min(off, 1 - off)
        assert off <= bound(position), (position, freq)
        if abs(position) <= 2**36:
            worst = max(worst, float(2 * PI * off))
    assert 8e-8 < worst < 1.1e-7                            # in radians: the figure that the documents name


@pytest.mark.gpu
@pytest.mark.parametrize("adjacent", [False, True])
def test_positions_beyond_32_bits(adjacent):
    """One rounding to bf16, 2^-20 of the pair's length for sine, cosine, products and sum in 32 bits, and the angle's bound."""
    positions = [2**31, 2**31 + 1, -2**31 - 1, 2**33 + 12345, -2**35 + 7, 2**40 + 3, 10**12, -10**13, 2**45 + 1]
    gen = torch.Generator().manual_seed(0)
    q = randn(gen, len(positions), 3, 128)
    axes = op.RotaryAxes(FREQ, adjacent=adjacent)
    for inverse in (False, True):
        ours = op.rotary(q.cuda(), None, torch.tensor([positions]).cuda(), axes, inverse=inverse)[0].double().cpu()
        x = q.double()
        for t, position in enumerate(positions):
            slack = 2**-20 + float(2 * PI * bound(position))
            for i, freq in enumerate(FREQ):
                a, b = (2 * i, 2 * i + 1) if adjacent else (i, i + 64)
                angle = float(2 * PI * turn_left_over(position, freq)) * (-1 if inverse else 1)
                first = x[t, :, a] * math.cos(angle) - x[t, :, b] * math.sin(angle)
                second = x[t, :, b] * math.cos(angle) + x[t, :, a] * math.sin(angle)
                length = (x[t, :, a] ** 2 + x[t, :, b] ** 2).sqrt()
                for got, want in ((ours[t, :, a], first), (ours[t, :, b], second)):
                    assert ((got - want).abs() <= BF16_HALF_STEP * (1 + 2**-10) * want.abs() + slack * length).all(), (position, i)
