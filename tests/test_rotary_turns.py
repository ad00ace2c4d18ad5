"""The rotation's table of turns per position is right to its last bit, so that far positions are too."""

import math
from fractions import Fraction

import pytest
import torch

import splash_attention_mgpu as sa

DEV = "cuda:0"
# Pi to 110 digits (A000796).
PI = Fraction(int("31415926535897932384626433832795028841971693993751058209749445923078164062862089986280348253421170679821480865"), 10 ** 109)
PLANS = [dict(), dict(base=500000.0), dict(inv_freq=[(-1) ** i * 0.7 ** i * 9.0 for i in range(64)]), dict(inv_freq=[1e30 / 7 ** i for i in range(64)]),
         dict(inv_freq=[0.0, 2 * math.pi, 1e-300, 5e-324] * 16)]


@pytest.mark.parametrize("plan", PLANS, ids=range(len(PLANS)))
def test_table(plan):
  plan = sa.make_rotary(128, **plan)
  for f, stored in zip(plan.inv_freq, plan._turns.tolist()):
    off = (Fraction(f) / (2 * PI) * 2 ** 64 - stored) % 2 ** 64
    assert min(off, 2 ** 64 - off) <= Fraction(1, 2) + Fraction(1, 10 ** 6)


@pytest.mark.gpu
def test_gpu_far_positions():
  """An angle is off by |pos| 2^-65 turns and 2^-25 half turns, a result by as much of |a| + |b|; 2^-20 and half a rounding step as
  in test_gpu_rotary.py."""
  far = [2 ** e + 12345 for e in range(30, 47)] + [-2 ** 41, -2 ** 45 - 7]
  plan = sa.make_rotary(128)
  g = torch.Generator().manual_seed(0)
  x = torch.randn(2, len(far), 128, generator=g).to(torch.float16)
  got = plan(x.to(DEV), None, torch.tensor(far, device=DEV)).double().cpu()
  for i, position in enumerate(far):
    turns = [float(Fraction(f) * position / (2 * PI) % 1) for f in plan.inv_freq]
    angle = 2 * math.pi * torch.tensor(turns, dtype=torch.float64)
    a, b = x[:, i, :64].double(), x[:, i, 64:].double()
    want = torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1)
    size = (a.abs() + b.abs()).repeat(1, 2)
    off = 2.0 ** -20 + 2 * math.pi * (abs(position) * 2.0 ** -65 + 2.0 ** -26)
    assert ((got[:, i] - want).abs() <= 2.0 ** -11 * want.abs() + off * size + 2.0 ** -24).all(), position
