"""What rotary positions decide without a GPU: frequencies, refusals, the checks of the C entry point."""
import ctypes as C
import math
import re
from fractions import Fraction

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from oracle import rotary_ref
from tokamax_b200 import _native
from tokamax_b200 import rotary


def test_frequencies():
  freq, factor = rotary.frequencies(8, base=10000.0)
  assert np.allclose(freq, [1.0, 0.1, 0.01, 0.001], rtol=1e-14) and factor == 1.0
  linear, _ = rotary.frequencies(8, scaling=rotary.Scaling("linear", factor=4.0))
  assert np.allclose(linear, freq / 4, rtol=1e-14)
  other, _ = rotary.frequencies(8, scaling=rotary.Scaling("base", factor=8.0))
  assert other[0] == 1.0 and math.isclose(other[-1], freq[-1] / 8, rel_tol=1e-12)


def test_frequencies_by_parts():
  spec = rotary.Scaling("by_parts", factor=16.0, original=4096)
  freq, _ = rotary.frequencies(128)
  got, factor = rotary.frequencies(128, scaling=spec)
  turns = 4096 * freq / (2 * math.pi)
  assert np.allclose(got[turns > 40], freq[turns > 40]) and np.allclose(got[turns < 0.9], freq[turns < 0.9] / 16)
  assert (np.diff(got) < 0).all() and math.isclose(factor, 1 + 0.1 * math.log(16))
  assert rotary.frequencies(128, scaling=rotary.Scaling("by_parts", factor=16.0, original=4096, attention=2.0))[1] == 2.0


def test_frequencies_in_bands():
  freq, _ = rotary.frequencies(128, base=500000.0)
  got, factor = rotary.frequencies(128, base=500000.0, scaling=rotary.Scaling("bands", factor=8.0, original=8192))
  wave = 2 * math.pi / freq
  assert factor == 1.0 and np.allclose(got[wave <= 2048], freq[wave <= 2048]) and np.allclose(got[wave >= 8192], freq[wave >= 8192] / 8)
  between = (wave > 2048) & (wave < 8192)
  part = (8192 / wave[between] - 1) / 3
  assert between.any() and np.allclose(got[between], (1 - part) * freq[between] / 8 + part * freq[between])


@pytest.mark.parametrize("kw", [dict(kind="other"), dict(kind="linear", factor=0.5), dict(kind="linear", factor=math.nan), dict(kind="bands", factor=2.0),
                                dict(kind="by_parts", factor=2.0, original=0), dict(kind="by_parts", original=9, fast=1.0),
                                dict(kind="bands", original=9, low=4.0)])
def test_scalings_that_cannot_be(kw):
  with pytest.raises(ValueError):
    rotary.Scaling(**kw)


@pytest.mark.parametrize("kw", [dict(dim=0), dict(dim=3), dict(dim=-2), dict(base=1.0), dict(base=math.inf), dict(factor=math.nan),
                                dict(frequency=[1.0]), dict(frequency=[1.0, math.nan, 1.0, 1.0]),
                                dict(frequency=[1.0] * 4, scaling=rotary.Scaling("linear")), dict(dim=2, scaling=rotary.Scaling("base", factor=2.0))])
def test_tables_that_cannot_be_made(kw):
  with pytest.raises(ValueError):
    rotary.make_rotary(**dict(dict(dim=8, device="cpu"), **kw))


@pytest.mark.parametrize("kw", [dict(factor=1e39), dict(factor=-math.inf), dict(scaling=rotary.Scaling("by_parts", original=9, attention=1e300))])
def test_factors_that_32_bits_do_not_hold_are_refused(kw):
  """The kernels' factor is one: infinity times a sine of 0 would be NaN."""
  with pytest.raises(ValueError, match="finite in 32 bits"):
    rotary.make_rotary(8, device="cpu", **kw)
  assert rotary.make_rotary(8, device="cpu", factor=3e38).factor == 3e38


def test_turns():
  """The part of a turn that a token is, to 2^-65, whole turns left out."""
  freq = [1.0, 2 * math.pi + 0.25, -0.125, 0.0]
  turns = rotary.make_rotary(8, frequency=freq, device="cpu").turns.tolist()
  for f, got in zip(freq, turns):
    off = (Fraction(f) / rotary_ref.TWO_PI - Fraction(got, 2 ** 64)) % 1
    assert min(off, 1 - off) <= Fraction(1, 2 ** 65)


def _call(rot=None, positions=None, q=None, k=None):
  rot = rotary.make_rotary(8, device="cpu") if rot is None else rot
  return rotary.rotate(rot, torch.zeros(1, 3, dtype=torch.int64) if positions is None else positions, torch.zeros(1, 2, 3, 16) if q is None else q, k)


@pytest.mark.parametrize("kw,error", [
    (dict(), RuntimeError),  # no CUDA device
    (dict(positions=torch.zeros(1, 3)), ValueError), (dict(positions=torch.zeros(1, 4, dtype=torch.int64)), ValueError),
    (dict(positions=torch.zeros(2, 3, dtype=torch.int64)), ValueError), (dict(positions=torch.zeros(1, 1, 3, dtype=torch.int64)), ValueError),
    (dict(q=torch.zeros(2, 3, 16)), ValueError), (dict(k=torch.zeros(1, 2, 4, 16)), ValueError), (dict(k=torch.zeros(2, 2, 3, 16)), ValueError),
    (dict(k=torch.zeros(1, 2, 3, 8)), ValueError), (dict(k=torch.zeros(1, 2, 3, 16, dtype=torch.float16)), ValueError)])
def test_operands_that_do_not_match_are_refused(kw, error):
  with pytest.raises(error):
    _call(**kw)


def test_calls_are_not_recorded_and_tangents_refused():
  q = torch.zeros(1, 2, 3, 16)
  with pytest.raises(NotImplementedError, match="recorded"):
    torch.jit.trace(lambda x: _call(q=x), q, check_trace=False)
  with pytest.raises(RuntimeError, match="CUDA"):
    _call(q=q)
  with forward_ad.dual_level():
    dual = forward_ad.make_dual(q, torch.ones_like(q))
    for kw in (dict(q=dual), dict(k=dual)):
      with pytest.raises(NotImplementedError, match="tangent"):
        _call(**kw)
  for dtype in (torch.float64, torch.int32, torch.complex64):
    with pytest.raises(NotImplementedError, match="not built"):
      _call(q=q.to(dtype))


def test_calls_are_not_recorded_by_make_fx():
  """A graph of it would give back what this call's rows became, whatever it is given."""
  with pytest.raises(NotImplementedError, match="recorded by make_fx"):
    make_fx(lambda x: _call(q=x))(torch.zeros(1, 2, 3, 16))


def _args():
  """Arguments that pass every check up to the missing device; addresses that nobody reads."""
  a = _native.SplashRotateArgs()
  for t in (*a.x, *a.y):
    t.data, t.dtype = 4096, 0
    for i, (n, s) in enumerate(zip((1, 2, 3, 64), (384, 192, 64, 1))):
      t.size[i], t.stride[i] = n, s
  a.positions = a.turns = 4096
  a.position_stride, a.dim, a.factor = 3, 64, 1.0
  return a


def _spoil(a, path, value):
  at = a
  *way, last = re.findall(r"\w+", path)
  for step in way:
    at = getattr(at, step) if not step.isdigit() else at[int(step)]
  if last.isdigit():
    at[int(last)] = value
  else:
    setattr(at, last, value)


@pytest.mark.parametrize("path,value,status", [
    ("x.0.data", 4100, -1), ("y.1.data", 4100, -1), ("x.0.dtype", 2, -2), ("x.0.dtype", 3, -1), ("x.1.dtype", 1, -1), ("x.0.size.1", 3, -1),
    ("x.1.size.2", 4, -1), ("x.0.stride.2", 60, -1), ("y.0.stride.3", 2, -1), ("positions", None, -1), ("turns", None, -1), ("dim", 0, -1),
    ("dim", 3, -1), ("dim", 66, -1), ("position_stride", -1, -1), ("factor", math.nan, -1), ("x.0.data", None, -1)])
def test_the_c_entry_point_refuses_before_it_touches_the_gpu(path, value, status):
  a = _args()
  _spoil(a, path, value)
  assert _native.lib().splash_rotate(C.byref(a), None) == status


def test_the_c_entry_point_refuses_sizes_that_are_not_built():
  lib, a = _native.lib(), _args()
  assert lib.splash_rotate(None, None) == -1
  for t in (*a.x, *a.y):
    t.size[3] = t.stride[2] = 264
  assert lib.splash_rotate(C.byref(a), None) == -2
  for t in (*a.x, *a.y):
    t.size[3] = t.stride[2] = 64
    t.size[1] = 65536
  assert lib.splash_rotate(C.byref(a), None) == -7
  for t in (*a.x, *a.y):
    t.size[1], t.size[0], t.size[2] = 2, 1 << 16, 1 << 15
  assert lib.splash_rotate(C.byref(a), None) == -7
  for t in (*a.x, *a.y):
    t.data = None
  assert lib.splash_rotate(C.byref(a), None) == -1
