"""Prompts in chunks and tokens one by one through a quantised key / value cache, for one attention layer.

What a serving program does with the package: a chunk of the prompts is appended to the cache, the prefix is read back as the
dense tensors that a splash kernel takes, and the chunk attends to it under a causal mask with an offset; then every decoding
step appends one token of each sequence and attends to the cache in place.  The weights are random; what is printed is how far
the layer's outputs are from attention over keys and values that were never quantised.

  python examples/cached_generation.py --fmt int4
"""
import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from tokamax_b200 import kv_cache  # noqa: E402
from tokamax_b200 import splash_attention_kernel as splash  # noqa: E402
from tokamax_b200 import splash_attention_mask as mask_lib  # noqa: E402


class Layer:
  """Projections of one attention layer, [batch, tokens, heads, d]."""

  def __init__(self, width, q_heads, kv_heads, d, device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    make = lambda heads: (torch.randn(width, heads, d, generator=g, device=device) / math.sqrt(width)).to(torch.bfloat16)  # noqa: E731
    self.w_q, self.w_k, self.w_v = make(q_heads), make(kv_heads), make(kv_heads)

  def qkv(self, x):
    """[batch, heads, tokens, d] views of the projections: the cache and the kernels read them through their strides."""
    return tuple(torch.einsum("btw,whd->bthd", x, w).transpose(1, 2) for w in (self.w_q, self.w_k, self.w_v))


class Server:
  """Sequences with a cache: pages are handed out as they grow."""

  def __init__(self, layer, batch, max_tokens, fmt, page_size=64, device="cuda"):
    self.layer, self.page_size = layer, page_size
    _, kv_heads, d = layer.w_k.shape
    pages = -(-max_tokens // page_size)
    self.cache = kv_cache.make_kv_cache(batch * pages, page_size, kv_heads, d, fmt=fmt, device=device)
    self.table = torch.full((batch, pages), -1, dtype=torch.int32, device=device)
    self.free = list(range(batch * pages))
    self.held = [0] * batch  # tokens of each sequence, on the host: it hands out the pages
    self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
    self.kernels = {}

  def _grow(self, new):
    for b, n in enumerate(new):
      first, last = -(-self.held[b] // self.page_size), -(-(self.held[b] + n) // self.page_size)
      for i in range(first, last):
        self.table[b, i] = self.free.pop()
      self.held[b] += n
    self.lengths.copy_(torch.tensor(self.held, dtype=torch.int32))

  def prefill(self, x, lengths, chunk=256):
    """x [batch, T, width], the first lengths[b] tokens of each its prompt (T a multiple of `chunk`, `chunk` one of 128).  Returns
    the layer's attention [batch, heads, T, d]; what stands behind a prompt's end is of no meaning."""
    outs = []
    for start in range(0, x.shape[1], chunk):
      end = start + chunk
      q, k, v = self.layer.qkv(x[:, start:end])
      self._grow([min(max(n - start, 0), chunk) for n in lengths])
      positions = torch.arange(start, end, device=x.device)[None, :].expand(x.shape[0], -1)
      positions = torch.where(positions < torch.as_tensor(lengths, device=x.device)[:, None], positions, -1)
      kv_cache.append(self.cache, k, v, kv_cache.slots_of(self.cache, self.table, positions))
      prefix_k, prefix_v = kv_cache.read(self.cache, self.table, self.lengths, end)
      if end not in self.kernels:
        self.kernels[end] = splash.make_splash_mha(mask_lib.CausalMask((chunk, end), start), q_seq_shards=1)
      outs.append(self.kernels[end](q, prefix_k, prefix_v, logits_scale=q.shape[-1] ** -0.5))
    return torch.cat(outs, 2)

  def decode(self, x):
    """x [batch, T, width]: the newest T tokens of every sequence.  Returns [batch, heads, T, d]."""
    q, k, v = self.layer.qkv(x)
    t = x.shape[1]
    self._grow([t] * x.shape[0])
    positions = self.lengths[:, None] - t + torch.arange(t, device=x.device)[None, :]
    kv_cache.append(self.cache, k, v, kv_cache.slots_of(self.cache, self.table, positions))
    return kv_cache.attend(self.cache, q, self.table, self.lengths, logits_scale=q.shape[-1] ** -0.5)


def plain_attention(layer, x, first):
  """Attention of tokens `first` .. of one sequence x [T, width] over all before them, in 32 bits, from unquantised K and V."""
  q, k, v = (y[0].float() for y in layer.qkv(x[None]))
  group = q.shape[0] // k.shape[0]
  k, v = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
  logits = q[:, first:] @ k.transpose(1, 2) * q.shape[-1] ** -0.5
  at = torch.arange(x.shape[0], device=x.device)
  return torch.softmax(logits.masked_fill(at[None, :] > at[first:, None], -math.inf), -1) @ v


@torch.no_grad()
def run(fmt="int4", batch=4, prompt=1000, steps=(1, 1, 1, 4), q_heads=8, kv_heads=2, d=128, width=512, chunk=256, seed=0, device="cuda"):
  """Relative errors of the prompts' and of the decoded tokens' outputs against unquantised attention."""
  g = torch.Generator(device=device).manual_seed(seed)
  layer = Layer(width, q_heads, kv_heads, d, device, seed)
  lengths = [max(1, prompt - 211 * b) for b in range(batch)]
  padded = -(-max(lengths) // chunk) * chunk
  x = torch.randn(batch, padded + sum(steps), width, generator=g, device=device).to(torch.bfloat16)
  server = Server(layer, batch, max(lengths) + sum(steps), fmt, device=device)
  prefill = server.prefill(x[:, :padded], lengths, chunk)
  decoded, at = [], padded  # (decoded tokens are the last ones of x, for every sequence)
  for t in steps:
    decoded.append(server.decode(x[:, at:at + t]))
    at += t
  decoded = torch.cat(decoded, 2)
  relative = lambda a, b: ((a.float() - b).norm() / b.norm()).item()  # noqa: E731
  errors = []
  for b, n in enumerate(lengths):
    want = plain_attention(layer, torch.cat((x[b, :n], x[b, padded:])), 0)
    errors.append((relative(prefill[b, :, :n], want[:, :n]), relative(decoded[b], want[:, n:])))
  return server, errors


if __name__ == "__main__":
  parser = argparse.ArgumentParser(description=__doc__.split("\n", maxsplit=1)[0])
  parser.add_argument("--fmt", default="int4", choices=sorted(kv_cache.FORMATS))
  parser.add_argument("--batch", type=int, default=4)
  parser.add_argument("--prompt", type=int, default=1000)
  args = parser.parse_args()
  for i, (in_prompt, in_decoding) in enumerate(run(args.fmt, args.batch, args.prompt)[1]):
    print(f"sequence {i}: relative error of the prompt's outputs {in_prompt:.4f}, of the decoded tokens' {in_decoding:.4f}")
