"""Rotary positions of queries and keys, with their gradient.

The reference's splash path takes queries and keys that have their positions already
(`tokamax/_src/ops/experimental/tpu/splash_attention/splash_attention_kernel.py`); here :func:`rotate` gives them theirs, for the
splash kernels and for the cache of :mod:`tokamax_b200.kv_cache`:

  rot = rotary.make_rotary(128, base=500000.0, scaling=rotary.Scaling("bands", factor=8.0, original=8192))
  q, k = rotary.rotate(rot, positions, q, k)

A pair of channels is turned by its position times a frequency.  Angles are fractions of a whole turn in 64 bits, which wrap
as turns do: a pair's frequency is held to 2^-65 of a turn a token, and its product with a position of 10^9 to 3e-11 of a turn.  Sine and
cosine are taken of the upper 32 bits in 24 bits: up to 1.5e-8 of a turn off, at any position, for rows of 16 bits, 4e-9 for
float32 rows.
"""
from __future__ import annotations

import dataclasses
import math
from fractions import Fraction

import numpy as np
import torch

from tokamax_b200 import _native

_TWO_PI = Fraction("6.28318530717958647692528676655900576839433879875")
SCALINGS = ("linear", "base", "by_parts", "bands")


@dataclasses.dataclass(frozen=True)
class Scaling:
  """How frequencies are changed for contexts ``factor`` times as long as those that a model was trained on.

  ``"linear"``    all of them divided by ``factor``
  ``"base"``      another base, so that the last pair turns ``factor`` times slower and the first as before
  ``"by_parts"``  pairs that make ``fast`` turns and more over the ``original`` length as before, those that make ``slow`` and fewer
                  divided by ``factor``, a ramp over the pairs between; rotated channels times ``attention`` (default ``0.1 ln(factor) + 1``)
  ``"bands"``     pairs that make ``high`` turns and more over the ``original`` length as before, those that make fewer than ``low``
                  divided by ``factor``, between by their turns"""
  kind: str
  factor: float = 1.0
  original: int | None = None
  fast: float = 32.0
  slow: float = 1.0
  low: float = 1.0
  high: float = 4.0
  attention: float | None = None

  def __post_init__(self):
    if self.kind not in SCALINGS:
      raise ValueError(f"scaling must be one of {SCALINGS}, got {self.kind!r}")
    if not (math.isfinite(self.factor) and self.factor >= 1.0):
      raise ValueError(f"factor must be 1 at least, got {self.factor}")
    if self.kind in ("by_parts", "bands") and not (self.original is not None and self.original > 0):
      raise ValueError(f"{self.kind!r} needs the original length, got {self.original}")
    if self.kind == "by_parts" and not self.fast > self.slow > 0:
      raise ValueError(f"expected fast > slow > 0, got {self.fast} and {self.slow}")
    if self.kind == "bands" and not self.high > self.low > 0:
      raise ValueError(f"expected high > low > 0, got {self.high} and {self.low}")


def frequencies(dim: int, *, base: float = 10000.0, scaling: Scaling | None = None) -> tuple[np.ndarray, float]:
  """Radians a token of each of ``dim / 2`` pairs, in 64 bits, and what rotated channels are multiplied by."""
  if dim < 2 or dim % 2:
    raise ValueError(f"dim must be even, 2 at least, got {dim}")
  if not (math.isfinite(base) and base > 1.0):
    raise ValueError(f"base must be above 1, got {base}")
  pairs = dim // 2
  pair = np.arange(pairs, dtype=np.float64)
  factor = 1.0 if scaling is None else scaling.factor
  if scaling is not None and scaling.kind == "base":
    if pairs == 1:
      raise ValueError("a single pair cannot turn as before and slower")
    base = base * factor ** (pairs / (pairs - 1))
  freq = base ** (-pair / pairs)
  if scaling is None or scaling.kind == "base":
    return freq, 1.0
  if scaling.kind == "linear":
    return freq / factor, 1.0
  if scaling.kind == "by_parts":
    # the pair (a real number) that makes so many turns over the original length
    pair_of = lambda turns: pairs * math.log(scaling.original / (turns * 2 * math.pi)) / math.log(base)  # noqa: E731
    lo, hi = max(math.floor(pair_of(scaling.fast)), 0), min(math.ceil(pair_of(scaling.slow)), dim - 1)
    slower = np.clip((pair - lo) / max(hi - lo, 0.001), 0.0, 1.0)
    attention = 0.1 * math.log(factor) + 1.0 if scaling.attention is None else scaling.attention
    return freq * (1.0 - slower) + freq / factor * slower, attention
  turns = scaling.original * freq / (2 * math.pi)
  keep = np.clip((turns - scaling.low) / (scaling.high - scaling.low), 0.0, 1.0)
  return freq * keep + freq / factor * (1.0 - keep), 1.0


@dataclasses.dataclass(frozen=True, eq=False)
class Rotary:
  """What the layers of a model share; made by :func:`make_rotary`.  ``turns`` int64 ``[dim / 2]``: of each pair the part of a
  whole turn that a token is, in units of 2^-64 (the bits of an unsigned number)."""
  dim: int
  interleaved: bool
  factor: float
  turns: torch.Tensor
  native: object = dataclasses.field(repr=False)

  def __reduce__(self):  # (a module that holds one can be copied and pickled)
    return _of_turns, (self.dim, self.interleaved, self.factor, self.turns)


def _of_turns(dim: int, interleaved: bool, factor: float, turns: torch.Tensor) -> Rotary:
  return Rotary(dim, interleaved, factor, turns, _native.host().RotaryTable(turns, dim, interleaved, factor))


def make_rotary(dim: int, *, base: float = 10000.0, scaling: Scaling | None = None, frequency=None, factor: float | None = None,
                interleaved: bool = False, device="cuda") -> Rotary:
  """Rotary positions for the first ``dim`` channels of rows (even; the others are left as they are).

  Pair i is ``(x[i], x[i + dim / 2])``, or ``(x[2 i], x[2 i + 1])`` if ``interleaved``.  ``frequency [dim / 2]`` (radians a token) takes
  the place of those that ``base`` and ``scaling`` make, ``factor`` of what the scaling multiplies rotated channels by."""
  freq, attention = frequencies(dim, base=base, scaling=scaling)
  if frequency is not None:
    if scaling is not None:
      raise ValueError("frequencies that are given are not scaled")
    freq = np.asarray(frequency.detach().cpu() if isinstance(frequency, torch.Tensor) else frequency, dtype=np.float64)
    if freq.shape != (dim // 2,) or not np.isfinite(freq).all():
      raise ValueError(f"expected {dim // 2} finite frequencies, got {freq.shape}")
  factor = attention if factor is None else float(factor)
  if not abs(factor) <= torch.finfo(torch.float32).max:
    raise ValueError(f"factor must be finite in 32 bits, got {factor}")
  parts = [round(Fraction(f) / _TWO_PI * 2 ** 64) % 2 ** 64 for f in freq.tolist()]  # (whole turns are none)
  turns = torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in parts], dtype=torch.int64, device=device)
  return _of_turns(dim, interleaved, factor, turns)


def rotate(rotary: Rotary, positions: torch.Tensor, q: torch.Tensor, k: torch.Tensor | None = None):
  """``q [B, heads, T, D]`` and ``k [B, other heads, T, D]`` (one type of bf16, f16 and f32) turned by their positions; without k
  the rotated q alone.

  ``positions [B, T]`` or ``[T]`` (int32 or int64), any numbers.  Rows are read through their strides, the ``[B, T, H, D]`` of a projection,
  transposed, is not copied, and results lie as the inputs do.  (Strides that are no multiples of eight, or rows that begin between
  two boundaries of 16 bytes: a contiguous copy is turned.)  Products are of 32 bits, rounded to the type once.

  Gradients go to q and k: the rotation back, which keeps nothing of a call but its positions.  Tangents of forward mode,
  the transforms of ``torch.func``, ``torch.jit.trace`` and ``make_fx`` are refused; ``torch.compile`` runs the call as it is."""
  out_q, out_k = _native.host().rotate(rotary.native, positions, q, k)
  return out_q if k is None else (out_q, out_k)
