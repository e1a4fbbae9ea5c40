"""Angles of rotary up to 2^51 on the GPU: the exact product of position and frequency, reduced by pi in whole numbers.

Bound of a value, whatever its angle: its cosine and sine are off by at most 2^-23 each; the fp32 rotation rounds a product and the
result (2^-24 of each); then comes the output's own rounding."""
from __future__ import annotations

import math
import random
from fractions import Fraction

import pytest
import torch

import gtx16_fp16 as g

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32

ONE = 1 << 256


def _arctan(n):
    """arctan(1 / n) in units of 1 / ONE, by its series."""
    term, total, k = ONE // n, 0, 1
    while term:
        total += term // k if k % 4 == 1 else -(term // k)
        term //= n * n
        k += 2
    return total


PI = 4 * (4 * _arctan(5) - _arctan(239))  # (Machin's sum), within some tens of units


def reduced(position, freq):
    """position * freq less its whole turns, as a double: the product exact, off by at most 2^60 units of 2^-256 before that."""
    units = Fraction(freq) * position * ONE  # (a frequency has at most 149 digits behind the point)
    assert units.denominator == 1
    turn = 2 * PI
    return math.ldexp((int(units) + PI) % turn - PI, -256)


def angles_of(positions, freqs):
    return torch.tensor([[reduced(p, f) for f in freqs.tolist()] for p in positions.tolist()], dtype=torch.float64)


def check(x, positions, freqs, angles):
    y, half = g.rotary(x, positions, freqs), x.dtype == F16
    assert y.dtype == x.dtype
    x, y = x.cpu().double(), y.cpu().double()
    pairs = freqs.shape[0]
    a, b = x[..., :pairs], x[..., pairs:]
    cos, sin = angles.cos()[:, None], angles.sin()[:, None]
    want = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    off = ((2.0 ** -23 + 2.0 ** -24) * (a.abs() + b.abs())).repeat(1, 1, 2)
    u, least = (2.0 ** -11, 2.0 ** -25) if half else (2.0 ** -24, 1e-37)
    over = ((y - want).abs() / (off * (1 + u) + u * want.abs() + least)).max().item()
    assert over <= 1.0, f"{over:.3g} times the bound"


@pytest.mark.parametrize("seed", range(3))
def test_angles_up_to_the_limit(cuda, seed):
    # every size from 2^20 to 2^50.5, both signs
    rng = random.Random(seed)
    freqs = torch.tensor([2.0 ** (rng.random() * 19.5) for _ in range(64)], dtype=F32)
    positions = torch.tensor([rng.choice((-1, 1)) * int(2.0 ** (20 + 11 * rng.random())) for _ in range(40)] + [(1 << 31) - 1, -(1 << 31)],
                             dtype=torch.int32)
    x = torch.randn(42, 2, 128, generator=torch.Generator().manual_seed(seed))
    check(x.to(cuda), positions.to(cuda), freqs.to(cuda), angles_of(positions, freqs))


@pytest.mark.parametrize("dtype", [F16, F32])
def test_positions_of_32_bits(cuda, dtype):
    # the usual frequencies, none above 1, at positions all the way to the type's ends
    rng = random.Random(5)
    freqs = torch.tensor([10000.0 ** (-i / 32) for i in range(32)], dtype=F32)
    positions = torch.tensor([rng.randrange(-(1 << 31), 1 << 31) for _ in range(100)], dtype=torch.int32)
    x = torch.randn(100, 1, 64, generator=torch.Generator().manual_seed(1)).to(dtype)
    check(x.to(cuda), positions.to(cuda), freqs.to(cuda), angles_of(positions, freqs))
