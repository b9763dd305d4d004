"""A quantised, paged key / value cache: written as tokens come, read back, and attended to in place.

The reference's splash path has no cache, and dequantises quantised operands before it sees them
(`tokamax/_src/quantization.py:75-78`).  This one holds keys and values in 4 or 8 bits and serves the two ways in which a
program meets them again:

  * a chunk of a prompt attends to what earlier chunks left: :func:`read` gives the prefix as the dense ``[B, H, S, D]``
    tensors that the splash kernels take;
  * a decoding step attends with one token, or a few drafted ones, of every sequence: :func:`attend` does so from the codes.

Formats:
  ``"int4"``  codes 0 .. 15 with a bf16 zero and a bf16 scale for each group of 32, 64 or 128 channels of a token's row:
              ``value = zero + scale * code``, ``zero`` the least value of the group, ``scale`` a fifteenth of its range
  ``"e4m3"``  e4m3 values with a bf16 scale for the row, ``scale = amax / 448``

Tokens lie in pages of ``page_size`` tokens.  A token's place is its slot, ``page * page_size + offset``; a sequence's pages
are a row of the page table.  Whoever owns the cache hands pages out; :func:`slots_of` turns positions into slots.

The operators serve inference: operands that require a gradient or have a tangent of forward mode are refused, and so are calls
under ``torch.jit.trace``, whose graph would not hold the launches.
"""
from __future__ import annotations

import ctypes as C
import dataclasses

import torch

from tokamax_b200 import _native
from tokamax_b200.base import DEFAULT_MASK_VALUE

FORMATS = {"int4": _native.CACHE_INT4, "e4m3": _native.CACHE_E4M3}
GROUP_SIZES = (32, 64, 128)


@dataclasses.dataclass(frozen=True, eq=False)
class KVCache:
  """Keys and values of ``n_pages`` pages; made by :func:`make_kv_cache`.

  ``k_codes`` is uint8 ``[n_pages, kv_heads, page_size, bytes of a row]`` (int4: channel c is the low or, for odd c, the high
  half of byte c // 2), ``k_scales`` bf16 ``[n_pages, kv_heads, page_size, groups, 2]`` (zero, scale) for int4 and
  ``[n_pages, kv_heads, page_size]`` for e4m3; the same for v.  Rows are padded to the widths that the kernels are built for."""
  fmt: str
  group_size: int | None
  page_size: int
  kv_heads: int
  head_dim: int
  head_dim_v: int
  k_codes: torch.Tensor
  k_scales: torch.Tensor
  v_codes: torch.Tensor
  v_scales: torch.Tensor
  native: object = dataclasses.field(repr=False)

  @property
  def n_pages(self) -> int:
    return self.k_codes.shape[0]

  @property
  def device(self) -> torch.device:
    return self.k_codes.device


def make_kv_cache(n_pages: int, page_size: int, kv_heads: int, head_dim: int, head_dim_v: int | None = None, *,
                  fmt: str = "int4", group_size: int | None = None, device="cuda") -> KVCache:
  """An empty cache.  ``page_size``: a power of two, 16 at least.  Head dims: multiples of 8 up to 256.  ``group_size``
  (int4 only, default 64 where it divides the rows, else 32): channels that share a zero and a scale."""
  if fmt not in FORMATS:
    raise ValueError(f"fmt must be one of {tuple(FORMATS)}, got {fmt!r}")
  head_dim_v = head_dim if head_dim_v is None else head_dim_v
  if n_pages < 1 or kv_heads < 1:
    raise ValueError(f"expected at least one page and one head, got {n_pages} and {kv_heads}")
  if page_size < 16 or page_size & (page_size - 1):
    raise ValueError(f"page_size must be a power of two, 16 at least, got {page_size}")
  widths = (C.c_int32 * 2)()
  at = C.cast(widths, C.POINTER(C.c_int32))
  status = _native.lib().splash_cache_row_widths(head_dim, head_dim_v, at, C.cast(C.addressof(widths) + 4, C.POINTER(C.c_int32)))
  if status == -1:
    raise ValueError(f"head dims must be positive multiples of 8, got {head_dim} / {head_dim_v}")
  if status == -2:
    raise NotImplementedError(f"head dims {head_dim} / {head_dim_v} are not built on B200")
  _native.check(status, "splash_cache_row_widths")
  rows = tuple(widths)
  if fmt == "int4":
    if group_size is None:
      group_size = 64 if all(r % 64 == 0 for r in rows) else 32
    if group_size not in GROUP_SIZES or any(r % group_size for r in rows):
      raise ValueError(f"group_size must be one of {GROUP_SIZES} and divide rows of {rows[0]} and {rows[1]} channels, got {group_size}")
  elif group_size is not None:
    raise ValueError("group_size is for int4 (an e4m3 row has one scale)")
  arrays = []
  for row in rows:
    shape = (n_pages, kv_heads, page_size)
    if fmt == "int4":
      arrays.append(torch.zeros((*shape, row // 2), dtype=torch.uint8, device=device))
      arrays.append(torch.zeros((*shape, row // group_size, 2), dtype=torch.bfloat16, device=device))
    else:
      arrays.append(torch.zeros((*shape, row), dtype=torch.uint8, device=device))
      arrays.append(torch.zeros(shape, dtype=torch.bfloat16, device=device))
  native = _native.host().KvCache(*arrays, FORMATS[fmt], group_size or 0, head_dim, head_dim_v, *rows)
  return KVCache(fmt, group_size, page_size, kv_heads, head_dim, head_dim_v, *arrays, native)


def slots_of(cache: KVCache, page_table: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
  """Slots (int64) of the tokens at ``positions [B, T]`` of the sequences of ``page_table [B, pages]``; a negative position, one
  behind the table and one on a page that the table has as -1 have none (-1: :func:`append` does not keep the token).  They are the
  same for every layer of a model: worked out once a step."""
  n_table = page_table.shape[1]
  if n_table == 0:
    return torch.full(positions.shape, -1, dtype=torch.int64, device=positions.device)
  where = positions.clamp_min(0).long()
  index = where // cache.page_size
  page = page_table.long().gather(1, index.clamp_max(n_table - 1))
  slots = page * cache.page_size + where % cache.page_size
  return torch.where((positions >= 0) & (index < n_table) & (page >= 0), slots, -1)


def append(cache: KVCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
  """Quantises ``k [B, kv_heads, T, D]`` and ``v`` (bf16, f16 or f32) into the slots ``[B, T]`` (int32 or int64).  A group (row)
  with a value that is not finite reads back as NaN.

  A slot outside the cache (-1 for padding) means that the token is not kept.  k and v are read through their strides: the
  ``[B, T, H, D]`` of a projection, transposed, is not copied.  No two tokens of a call may have the same slot."""
  _native.host().cache_append(cache.native, k, v, slots)


def read(cache: KVCache, page_table: torch.Tensor, lengths: torch.Tensor, max_len: int, *,
         dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
  """The first ``lengths[b]`` tokens of every sequence as ``k [B, kv_heads, max_len, D]`` and ``v``; zeros behind them.

  ``page_table [B, pages]`` and ``lengths [B]``: int32.  Tokens on a page outside the cache (-1) read as zeros.  Values are
  rounded to ``dtype`` once."""
  return _native.host().cache_read(cache.native, page_table, lengths, max_len, dtype)


def attend(cache: KVCache, q: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, *, logits_scale: float = 1.0,
           local_window_size: int | None = None, logits_soft_cap: float | None = None, sinks: torch.Tensor | None = None,
           mask_value: float = DEFAULT_MASK_VALUE, save_residuals: bool = False):
  """Attention of the newest T tokens of every sequence: ``q [B, q_heads, T, D]`` (bf16 or f16) to ``o [B, q_heads, T, D_v]``.

  ``lengths [B]`` counts the tokens in the cache, those of ``q`` among them: query i stands at position
  ``lengths[b] - T + i`` and sees the keys up to it, at most ``local_window_size`` back.  Keys on a page outside the cache (-1)
  are not seen.  ``sinks [q_heads]`` and ``logits_soft_cap`` mean what they mean for the splash kernels.  A row that sees
  nothing is zeros and its logsumexp and maximum the mask value.  ``save_residuals`` adds ``{"logsumexp", "max_logits"}``
  ``[B, q_heads, T]``.

  Weights times the scales of V are held to 11 bits (22 for f16 outputs), down to 2^-22 of a row's largest; logits may be up to 2^26 in
  size.  What no query sees, a page's places that were never written among it, has no part.

  Made for few rows (T times q heads per kv head up to some tens: the codes are unpacked again for every 16 of them);
  a chunk of a prompt is better off with :func:`read` and a splash kernel.  Nothing is copied to the host: lengths and pages
  may change between the replays of a captured graph."""
  o, lse, max_logits = _native.host().cache_attend(cache.native, q, page_table, lengths, logits_scale, local_window_size,
                                                   logits_soft_cap, sinks, max(mask_value, -3.0e38), save_residuals)
  if save_residuals:
    return o, {"logsumexp": lse, "max_logits": max_logits}
  return o
