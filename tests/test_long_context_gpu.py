"""Rotary positions, bounds, choice and attention together, as a server of long contexts runs them; and the example that does so."""
import os
import runpy

import pytest
import torch

from oracle import pages_ref
from oracle import rotary_ref
from tokamax_b200 import kv_cache
from tokamax_b200 import rotary
from tokamax_b200 import splash_attention_kernel as splash
from tokamax_b200 import splash_attention_mask as mask_lib

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EXAMPLE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "cached_generation.py")


@pytest.mark.parametrize("fmt", ["int4", "e4m3"])
@pytest.mark.parametrize("turned", [False, True])
def test_the_example_with_rotary_positions_and_all_pages(fmt, turned):
  """As without a choice: tests/test_cached_generation_gpu.py has what the bound is made of."""
  run = runpy.run_path(EXAMPLE)["run"]
  server, errors = run(fmt, batch=3, prompt=600, steps=(1, 1, 3), chunk=128, turned=turned, pages=16)
  bound = 2.0 ** 0.5 * (0.09 if fmt == "int4" else 0.026) * 1.25
  for in_prompt, in_decoding in errors:
    assert in_prompt <= bound and in_decoding <= bound, errors
  assert server.lengths.tolist() == [605, 394, 183] == server.held


def test_the_example_runs_over_a_few_pages():
  _, errors = runpy.run_path(EXAMPLE)["run"]("int4", batch=2, prompt=1500, steps=(1, 2), chunk=256, turned=True, pages=4)
  assert all(torch.isfinite(torch.tensor(e)).all() for e in errors)


@pytest.mark.parametrize("fmt", ["int4", "e4m3"])
def test_a_long_chat_step_by_step(fmt):
  """Tokens come one by one and by threes, positions far out; every step's choice is the oracle's for what the cache holds, and what it
  attends to is what a dense table of the same pages gives."""
  page, heads, d, lengths = 16, 2, 64, [150, 37]
  g = torch.Generator(device=DEV).manual_seed(0)
  rot = rotary.make_rotary(d, scaling=rotary.Scaling("linear", factor=4.0), device=DEV)
  cache = kv_cache.make_kv_cache(40, page, heads, d, fmt=fmt, device=DEV)
  bounds = kv_cache.make_page_bounds(cache)
  table = torch.randperm(40, generator=g, device=DEV).int().view(2, 20)
  held = torch.zeros(2, dtype=torch.int32, device=DEV)

  def append(new):
    t = max(new)
    x = [torch.randn(2, t, heads * n, d, generator=g, device=DEV).to(torch.bfloat16).transpose(1, 2) for n in (3, 1, 1)]
    positions = held[:, None] + torch.arange(t, device=DEV)[None, :]
    q, k = rotary.rotate(rot, positions + 100000, x[0], x[1])
    kept = torch.arange(t, device=DEV)[None, :] < torch.tensor(new, device=DEV)[:, None]
    kv_cache.append(cache, k, x[2], kv_cache.slots_of(cache, table, torch.where(kept, positions, -1)))
    held.add_(torch.tensor(new, dtype=torch.int32, device=DEV))
    kv_cache.bound_pages(cache, bounds, table, held, t)
    return q

  append(lengths)
  for t in [1] * 20 + [3] * 6:
    q = append([t, t])
    tables, tokens = kv_cache.choose_pages(cache, bounds, q, table, held, 5, first=1, last=2)
    keys, _ = kv_cache.read(cache, table, held, int(held.max()), dtype=torch.float32)
    codes, scales = torch.zeros(40, heads, 2, d, dtype=torch.int8), torch.zeros(40, heads)
    for b in range(2):
      for j in range(int(held[b]) // page):
        codes[int(table[b, j])], scales[int(table[b, j])] = pages_ref.bounds(keys[b, :, j * page:(j + 1) * page].cpu())
    want = pages_ref.choose(q.cpu(), codes, scales, table.cpu(), held.tolist(), 40, page, 5, 1, 2)
    assert torch.equal(tables.cpu(), want[0]) and torch.equal(tokens.cpu(), want[1])
    got = kv_cache.attend(cache, q, tables, tokens, logits_scale=0.1)
    for h in range(heads):  # one head's and query's pages as a sequence of its own
      for i in range(t):
        dense = kv_cache.attend(cache, q[:, :, i:i + 1].contiguous(), tables[:, h, i].contiguous(), tokens[:, h, i].contiguous(), logits_scale=0.1)
        assert torch.equal(got[:, 3 * h:3 * h + 3, i], dense[:, 3 * h:3 * h + 3, 0])
  assert held.tolist() == [188, 75]


def test_training_through_rotary_positions_and_a_splash_kernel():
  """Gradients of q and k through both, against splash's own gradients turned back by the oracle."""
  s, d = 256, 64
  kernel = splash.make_splash_mha(mask_lib.CausalMask((s, s)), q_seq_shards=1)
  rot = rotary.make_rotary(d, interleaved=True, device=DEV)
  g = torch.Generator(device=DEV).manual_seed(1)
  make = lambda h: torch.randn(1, s, h, d, generator=g, device=DEV).to(torch.bfloat16).transpose(1, 2)  # noqa: E731
  q, k, v, do = make(4), make(2), make(2), make(4)
  positions = torch.arange(s, device=DEV)
  leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
  out = kernel(*rotary.rotate(rot, positions, leaves[0], leaves[1]), leaves[2], logits_scale=d ** -0.5)
  out.backward(do)
  turned = [x.detach().requires_grad_(True) for x in rotary.rotate(rot, positions, q, k)]
  inner = torch.autograd.grad(kernel(*turned, v, logits_scale=d ** -0.5), turned, do)
  freq, _ = rotary.frequencies(d)
  for leaf, grad in zip(leaves, inner):
    want, size = rotary_ref.rotate(grad, positions[None], freq, interleaved=True, inverse=True)
    # dq's partial sums may come in another order from call to call (2^-7 of a gradient's norm covers their bf16 roundings on both sides);
    # the rotation adds 2^-8 of a value
    err = (leaf.grad.cpu().double() - want).norm() / want.norm()
    assert err <= 2.0 ** -7, float(err)
    assert float(size.max()) > 0
