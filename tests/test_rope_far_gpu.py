"""Rotary positions from frequencies far from the origin, against turns counted in whole numbers.

The reference takes n f / 2 pi as a fraction of integers (f and n are what they are, pi to 60 digits) and only its rest of a
turn as a float.  Tolerance: sines off by 2^-23 and a few fp32 roundings, 2^-21 of the largest element (test_rope_scaled_gpu.py),
and the turn of a position, held to 2^-64 and its own rounding: |n| 2^-64 turns, under |n| 2^-61 of the largest element.
"""

from __future__ import annotations

import math
from fractions import Fraction

import pytest
import torch

from helpers import announce

pytestmark = pytest.mark.gpu
DEV = "cuda"
PI = Fraction(3141592653589793238462643383279502884197169399375105820974944592, 10 ** 63)


def turned(x, positions, freq, interleaved):
    """x (T, H, D) float64 with its pairs turned, one by one."""
    T, H, D = x.shape
    out = x.clone()
    for t, n in enumerate(positions):
        for i, f in enumerate(freq):
            a = 2 * math.pi * float((n * Fraction(f) / (2 * PI)) % 1)
            c, s = math.cos(a), math.sin(a)
            p, q = (2 * i, 2 * i + 1) if interleaved else (i, i + D // 2)
            out[t, :, p], out[t, :, q] = x[t, :, p] * c - x[t, :, q] * s, x[t, :, q] * c + x[t, :, p] * s
    return out


@pytest.mark.parametrize("first", [0, 10 ** 6, 2 ** 31, 2 ** 40, 2 ** 40 + 12345, 2 ** 45 + 1, -2 ** 40])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float64, torch.float32])
def test_far_positions(gpu_pkg, first, interleaved, dtype):
    D = 64
    freq = torch.cat([10000.0 ** (-torch.arange(0, D - 8, 2, dtype=torch.float64) / D),
                      torch.tensor([3.0, -1.0, 100.0, 6.25], dtype=torch.float64)]).to(dtype)
    pos = [first + i for i in range(9)]
    q = torch.randn(1, 9, 2, D, device=DEV)
    announce(f"positions from {first} {dtype}")
    got, _ = gpu_pkg.rope_scaled(q, None, torch.tensor(pos, device=DEV), freq.to(DEV), interleaved=interleaved)
    want = turned(q[0].double().cpu(), pos, freq.tolist(), interleaved)
    top = float(q.abs().max())
    worst = float((got[0].double().cpu() - want).abs().max())
    assert worst <= top * (2.0 ** -21 + abs(first) * 2.0 ** -61), worst


def test_frequencies_past_every_turn(gpu_pkg):
    """Large frequencies turn by what is left of whole turns, and none of them spoils another pair."""
    freq = torch.tensor([2.0 ** 20 + 0.7, 2.0 ** 40 * 1.1, 1e15, -1e15, 1e300, -1e300, 5e-324, -5e-324], dtype=torch.float64)
    pos = list(range(9))
    q = torch.randn(1, 9, 2, 16, device=DEV)
    announce("large frequencies")
    got, _ = gpu_pkg.rope_scaled(q, None, torch.tensor(pos, device=DEV), freq.to(DEV))
    assert torch.isfinite(got).all()
    fits = freq.abs() < 1e14                               # (f / 2 pi is held to 2^-106 of it)
    want = turned(q[0].double().cpu(), pos, freq.tolist(), False)
    cols = [i for i in range(8) if fits[i]]
    cols += [i + 8 for i in cols]
    worst = float((got[0].double().cpu() - want)[..., cols].abs().max())
    assert worst <= float(q.abs().max()) * 2.0 ** -21, worst
