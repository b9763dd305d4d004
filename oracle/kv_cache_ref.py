"""CPU oracle of the quantised key / value cache, in 64 bits.  TEST INFRASTRUCTURE ONLY.

What the formats hold, from their definitions, and dense attention over it.  The reference has no cache: there is nothing to
pin this against but the definitions themselves (see `tokamax_b200/kv_cache.py`).
"""
from __future__ import annotations

import math

import torch

MASK_VALUE = -0.7 * float(torch.finfo(torch.float32).max)


def held(x: torch.Tensor, fmt: str, group: int | None):
  """The values that a cache holds for rows ``x [..., d]``: float64."""
  x = x.cpu().double()
  if fmt == "e4m3":
    return _held_e4m3(x)
  parts = []
  for lo in range(0, x.shape[-1], group):
    part = x[..., lo:lo + group]
    least, most = part.amin(-1, keepdim=True), part.amax(-1, keepdim=True)
    zero, scale = least.to(torch.bfloat16).double(), ((most - least) / 15).to(torch.bfloat16).double()
    step = torch.where(scale > 0, scale, 1.0)
    code = torch.where(scale > 0, ((part - zero) / step).round().clamp(0, 15), 0.0)
    value = zero + scale * code
    parts.append(torch.where(part.isfinite().all(-1, keepdim=True), value, math.nan))
  return torch.cat(parts, -1)


def products(x: torch.Tensor, fmt: str, group: int | None):
  """``|scale * code|`` of the rows: what of a value is not the zero of its group."""
  value = held(x, fmt, group)
  if fmt == "e4m3":
    return value.abs()
  x = x.cpu().double()
  zeros = [x[..., lo:lo + group].amin(-1, keepdim=True).to(torch.bfloat16).double().expand_as(x[..., lo:lo + group])
           for lo in range(0, x.shape[-1], group)]
  return (value - torch.cat(zeros, -1)).abs()


def _held_e4m3(x):
  scale = (x.abs().amax(-1, keepdim=True) / 448).to(torch.bfloat16).double()
  y = (x / torch.where(scale > 0, scale, 1.0)).clamp(-448, 448)
  y = torch.where(scale > 0, y, 0.0)
  exponent = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -20))).clamp_min(-6)
  step = 2.0 ** (exponent - 3)
  value = (y / step).round() * step * scale
  return torch.where(x.isfinite().all(-1, keepdim=True), value, math.nan)


def attend(q, k, v, *, scale, window=None, soft_cap=None, sinks=None, seen=None, weights=None):
  """One sequence: q [Hq, T, D], k [Hkv, n, D], v [Hkv, n, Dv] in float64, `seen` bool [n] (keys on a page).

  Returns o [Hq, T, Dv], logsumexp and max_logits [Hq, T], and sum_j p_j |v_j| and sum_j p_j weights_j beside o (what its
  error scales with; weights: like v, |v| if not given)."""
  hq, t, _ = q.shape
  hkv, n, dv = v.shape
  o = torch.zeros(hq, t, dv, dtype=torch.float64)
  weights = v.abs() if weights is None else weights
  size, moved = torch.zeros_like(o), torch.zeros_like(o)
  lse = torch.full((hq, t), MASK_VALUE, dtype=torch.float64)
  top = lse.clone()
  at = torch.arange(n)
  for h in range(hq):
    kh, vh = k[h * hkv // hq], v[h * hkv // hq]
    for i in range(t):
      position = n - t + i
      keep = at <= position
      if window is not None:
        keep &= at >= position - window
      if seen is not None:
        keep &= seen
      x = kh[keep] @ q[h, i] * scale
      if soft_cap is not None:
        x = torch.tanh(x / soft_cap) * soft_cap
      logits = x if sinks is None else torch.cat([x, sinks[h:h + 1].double()])
      if logits.numel() == 0:
        continue
      lse[h, i], top[h, i] = torch.logsumexp(logits, 0), logits.max()
      p = torch.exp(x - lse[h, i])
      o[h, i], size[h, i], moved[h, i] = p @ vh[keep], p @ vh[keep].abs(), p @ weights[h * hkv // hq][keep]
  return o, lse, top, size, moved
