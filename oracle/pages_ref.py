"""CPU oracle of page bounds and of the choice of pages.  TEST INFRASTRUCTURE ONLY.

Both are defined in 32 bits where they round, and in whole numbers otherwise: there is one right answer.
"""
from __future__ import annotations

import torch

_MOST = 3.4028234663852886e38


def _numbers(x):
  return x.float().nan_to_num(nan=0.0, posinf=_MOST, neginf=-_MOST)


def _codes(x, scale):
  return torch.where(scale > 0, (x / torch.where(scale > 0, scale, 1.0)).round().clamp(-127, 127), 0.0)


def bounds(k):
  """Keys [.., tokens, d] of whole pages, in 32 bits: codes int8 [.., 2, d] and scales [..]."""
  x = _numbers(k)
  x = torch.stack((x.amin(-2), x.amax(-2)), -2)
  scale = x.abs().amax((-2, -1)) / torch.tensor(127.0)
  return _codes(x, scale[..., None, None]).to(torch.int8), scale


def scores(q, codes, scales):
  """q [group, d], codes [pages, 2, d], scales [pages]: float32 [pages]."""
  x = _numbers(q)
  code = _codes(x, x.abs().max() / torch.tensor(127.0)).long()
  least, largest = codes[:, 0].long(), codes[:, 1].long()
  whole = (code[:, None] * torch.where(code[:, None] > 0, largest, least)).sum(-1).max(0).values
  return whole.float() * scales


def choose(q, codes, scales, table, lengths, n_pages, page, count, first, last):
  """As kv_cache.choose_pages, all on the CPU: q [B, heads, T, D], codes [n_pages, kv_heads, 2, d], table [B, pages], lengths a list."""
  batch, heads, t, _ = q.shape
  kv_heads = codes.shape[1]
  group = heads // kv_heads
  tables = torch.full((batch, kv_heads, t, count), -1, dtype=torch.int32)
  tokens = torch.zeros((batch, kv_heads, t), dtype=torch.int32)
  for b in range(batch):
    for i in range(t):
      position = min(lengths[b] - t + i, table.shape[1] * page - 1)
      if position < 0:
        continue
      own = position // page
      index = [j for j in range(own + 1) if 0 <= int(table[b, j]) < n_pages]
      pages = table[b, index].long()
      for h in range(kv_heads):
        score = scores(q[b, h * group:(h + 1) * group, i], codes[pages, h], scales[pages, h]).tolist()
        order = sorted(range(len(index)), key=lambda n: (not (index[n] < first or index[n] > own - last), -score[n], n))
        order = sorted(order, key=lambda n: 0 if index[n] < first or index[n] > own - last else 1)  # (always taken: whatever the score)
        taken = sorted(order[:count])
        tables[b, h, i, :len(taken)] = table[b, [index[n] for n in taken]]
        full = len(taken) * page
        tokens[b, h, i] = full - (page - 1 - position % page if taken and index[taken[-1]] == own else 0)
  return tables, tokens
