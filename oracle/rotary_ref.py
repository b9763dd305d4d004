"""CPU oracle of rotary positions, in 64 bits.  TEST INFRASTRUCTURE ONLY.

From the definition: pairs as complex numbers, turned by ``position * frequency``.  Angles are reduced as rational numbers, so that
far positions lose nothing.
"""
from __future__ import annotations

import math
from fractions import Fraction

import torch

TWO_PI = Fraction("6.28318530717958647692528676655900576839433879875")


def angles(positions, freq):
  """``positions [..]`` (whole numbers) times ``freq [pairs]`` modulo a turn, float64 ``[.., pairs]``."""
  flat = []
  for position in positions.flatten().tolist():
    for f in freq:
      turns = Fraction(float(f)) * position / TWO_PI
      flat.append(float(turns - math.floor(turns)) * 2 * math.pi)
  return torch.tensor(flat, dtype=torch.float64).view(*positions.shape, len(freq))


def rotate(x, positions, freq, *, interleaved=False, factor=1.0, inverse=False):
  """x [B, H, T, D], positions [B, T].  Returns the rotated rows in float64, and |x0| + |x1| of each channel's pair (0 for channels that
  are copied), which is what rounding on the way scales with."""
  dim = 2 * len(freq)
  angle = angles(positions, freq)[:, None]
  turn = torch.polar(torch.full_like(angle, factor), -angle if inverse else angle)
  y, size = x.detach().cpu().double().clone(), torch.zeros(x.shape, dtype=torch.float64)
  pairs = torch.arange(dim // 2)
  one, two = (2 * pairs, 2 * pairs + 1) if interleaved else (pairs, pairs + dim // 2)
  z = torch.complex(y[..., one], y[..., two])
  size[..., one] = size[..., two] = z.real.abs() + z.imag.abs()
  z = z * turn
  y[..., one], y[..., two] = z.real, z.imag
  return y, size * abs(factor)
