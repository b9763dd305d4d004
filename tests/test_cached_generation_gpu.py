"""The example that serves prompts and decoded tokens from a quantised cache: writing, reading, splash and attention together."""
import os
import runpy

import pytest
import torch

pytestmark = pytest.mark.gpu
EXAMPLE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "cached_generation.py")


@pytest.mark.parametrize("fmt", ["int4", "e4m3"])
def test_prompts_and_decoded_tokens(fmt):
  run = runpy.run_path(EXAMPLE)["run"]
  server, errors = run(fmt, batch=3, prompt=600, steps=(1, 1, 3), chunk=128)
  # A uniform code of 15 steps over the range of 64 normal values (about 4.7 sigma) is off by 0.29 * 4.7 / 15 = 0.09 of a value
  # (e4m3: half of 2^-3 at most, 0.026 rms).  Values' errors average out as the values themselves do; logits are off by the same
  # share of their own spread, which is about 1: outputs are off by about sqrt(2) times that.
  bound = 2.0 ** 0.5 * (0.09 if fmt == "int4" else 0.026) * 1.25
  for in_prompt, in_decoding in errors:
    assert in_prompt <= bound and in_decoding <= bound, errors
  assert server.lengths.tolist() == [605, 394, 183] == server.held
  used = server.table[server.table >= 0]
  assert used.unique().numel() == used.numel() == sum(-(-n // server.page_size) for n in server.held)


def test_both_ways_through_the_cache_agree():
  """The last tokens of a prompt, as a chunk through read and a splash kernel and as queries of attend: the same keys and values,
  rounded to bf16 on one of the ways."""
  space = runpy.run_path(EXAMPLE)
  server, _ = space["run"]("int4", batch=2, prompt=512, steps=(1,), chunk=256)
  from tokamax_b200 import kv_cache
  from tokamax_b200 import splash_attention_kernel as splash
  from tokamax_b200 import splash_attention_mask as mask_lib

  lengths = torch.tensor([512, 301], dtype=torch.int32, device="cuda")
  q = torch.randn(2, 8, 128, 128, device="cuda").to(torch.bfloat16)
  o = kv_cache.attend(server.cache, q, server.table, lengths, logits_scale=128 ** -0.5)
  k, v = kv_cache.read(server.cache, server.table, lengths, 512)
  kernel = splash.make_splash_mha(mask_lib.CausalMask((128, 512), 384), q_seq_shards=1)
  want = kernel(q, k, v, logits_scale=128 ** -0.5)
  # values rounded to bf16 (2^-9 rms 0.3 of it each way), probabilities too, outputs on both sides: a few 2^-9
  assert ((o[0].float() - want[0].float()).norm() / want[0].float().norm()).item() <= 4 * 2.0 ** -9
