"""What page bounds and the choice of pages decide without a GPU: layout, refusals, the checks of the C entry points."""
import ctypes as C
import math
import os
import re
import subprocess

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from oracle import pages_ref
from tokamax_b200 import _native
from tokamax_b200 import kv_cache


def _cache(**kw):
  return kv_cache.make_kv_cache(**dict(dict(n_pages=5, page_size=16, kv_heads=2, head_dim=64, device="cpu"), **kw))


def test_layout():
  for fmt, d, row in (("int4", 80, 96), ("e4m3", 80, 96), ("int4", 160, 192), ("e4m3", 256, 256)):
    cache = _cache(fmt=fmt, head_dim=d)
    bounds = kv_cache.make_page_bounds(cache)
    assert bounds.codes.shape == (5, 2, 2, row) and bounds.codes.dtype == torch.int8 and not bounds.codes.any()
    assert bounds.scales.shape == (5, 2) and bounds.scales.dtype == torch.float32
    bounds.codes[1, 0, 1, 3] = -7
    bounds.scales[1, 0] = 0.5
    values = bounds.values()
    assert values.shape == (5, 2, 2, d) and values.dtype == torch.float32 and float(values[1, 0, 1, 3]) == -3.5 and int(values.count_nonzero()) == 1


def _choose(cache=None, bounds=None, q=None, table=None, lengths=None, count=3, **kw):
  cache = _cache() if cache is None else cache
  bounds = kv_cache.make_page_bounds(cache) if bounds is None else bounds
  return kv_cache.choose_pages(cache, bounds, torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16) if q is None else q,
                               torch.zeros(1, 4, dtype=torch.int32) if table is None else table,
                               torch.ones(1, dtype=torch.int32) if lengths is None else lengths, count, **kw)


@pytest.mark.parametrize("kw", [
    dict(q=torch.zeros(1, 3, 1, 64)), dict(q=torch.zeros(1, 4, 1, 32)), dict(q=torch.zeros(4, 1, 64)), dict(q=torch.zeros(2, 4, 1, 64)),
    dict(q=torch.zeros(1, 0, 1, 64)), dict(table=torch.zeros(1, 4)), dict(table=torch.zeros(4, dtype=torch.int32)), dict(table=torch.zeros(1, 0, dtype=torch.int32)),
    dict(lengths=torch.ones(2, dtype=torch.int32)), dict(lengths=torch.ones(1)), dict(count=0), dict(count=1), dict(count=2, first=2), dict(first=-1), dict(last=0),
    dict(count=1 << 32), dict(last=1 << 33, count=1 << 34)])
def test_choices_that_cannot_be_made(kw):
  with pytest.raises((ValueError, RuntimeError)) as e:
    _choose(**kw)
  assert isinstance(e.value, ValueError) or "CUDA" in str(e.value)


def test_calls_on_the_cpu_are_refused():
  cache = _cache()
  bounds, i = kv_cache.make_page_bounds(cache), torch.zeros(1, dtype=torch.int32)
  with pytest.raises(RuntimeError, match="CUDA"):
    _choose()
  with pytest.raises(RuntimeError, match="CUDA"):
    kv_cache.bound_pages(cache, bounds, i[None], i, 1)


def test_calls_are_not_recorded():
  cache = _cache()
  bounds, i = kv_cache.make_page_bounds(cache), torch.zeros(1, dtype=torch.int32)
  q = torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16)
  for call in (lambda x: _choose(q=x), lambda x: kv_cache.bound_pages(cache, bounds, i[None], i, 1) or x):
    with pytest.raises(NotImplementedError, match="recorded"):
      torch.jit.trace(call, q, check_trace=False)


def test_calls_are_not_recorded_by_make_fx():
  cache = _cache()
  bounds, i = kv_cache.make_page_bounds(cache), torch.zeros(1, dtype=torch.int32)
  q = torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16)
  for call in (lambda x: _choose(q=x), lambda x: kv_cache.bound_pages(cache, bounds, i[None], i, 1) or x,
               lambda x: kv_cache.attend(cache, x, i[None], i), lambda x: kv_cache.append(cache, x, x, i[None]) or x,
               lambda x: kv_cache.read(cache, i[None], i, 1)):
    with pytest.raises(NotImplementedError, match="recorded by make_fx"):
      make_fx(call)(q)


def test_queries_with_a_derivative_are_refused():
  q = torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16)
  with pytest.raises(NotImplementedError, match="gradient"):
    _choose(q=q.clone().requires_grad_(True))
  with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="tangent"):
    _choose(q=forward_ad.make_dual(q, torch.ones_like(q)))


@pytest.mark.parametrize("table,lengths,window", [
    ((1, 2, 1, 4), (1, 2), None), ((1, 2, 1, 4), (1, 2, 2), None), ((1, 1, 1, 4), (1, 1, 1), None), ((2, 2, 1, 4), (2, 2, 1), None),
    ((1, 2, 3, 4), (1, 2, 3), None), ((1, 2, 1, 4), (1, 2, 1), 5), ((1, 2, 1, 0), (1, 2, 1), None)])
def test_tables_that_do_not_match_are_refused(table, lengths, window):
  with pytest.raises((ValueError, RuntimeError)) as e:
    kv_cache.attend(_cache(), torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16), torch.zeros(table, dtype=torch.int32),
                    torch.ones(lengths, dtype=torch.int32), local_window_size=window)
  assert isinstance(e.value, ValueError) or "CUDA" in str(e.value)


def _args(kind):
  """Arguments that pass every check up to the missing device; addresses that nobody reads."""
  a = getattr(_native, kind)()
  c = a.cache
  c.k_codes = c.k_scales = c.v_codes = c.v_scales = 4096
  c.n_pages, c.format, c.page_size, c.kv_heads, c.group, c.head_dim, c.head_dim_v, c.row_k, c.row_v = 4, 0, 16, 2, 32, 64, 64, 64, 64
  for name in ("q", "o"):
    if hasattr(a, name):
      t = getattr(a, name)
      t.data, t.dtype = 4096, 0
      for i, (n, s) in enumerate(zip((1, 2, 3, 64), (384, 192, 64, 1))):
        t.size[i], t.stride[i] = n, s
  a.page_table, a.lengths, a.table_stride, a.n_table = 4096, 4096, 2, 2
  if hasattr(a, "bounds"):
    a.bounds.codes = a.bounds.scales = 4096
  if kind == "SplashCacheBoundArgs":
    a.batch, a.newest = 1, 1
  if kind == "SplashCacheChooseArgs":
    a.tables, a.table_lengths, a.count, a.first, a.last = 4096, 4096, 4, 1, 1
  if kind == "SplashCacheAttendArgs":
    a.window = -1
  return a


def _spoilt(kind, path, value):
  a = _args(kind)
  at = a
  *way, last = re.findall(r"\w+", path)
  for step in way:
    at = getattr(at, step) if not step.isdigit() else at[int(step)]
  if last.isdigit():
    at[int(last)] = value
  else:
    setattr(at, last, value)
  return a


FAULTS = [("cache.k_codes", None, -1), ("cache.page_size", 24, -1), ("cache.format", 2, -2), ("cache.head_dim", 320, -2), ("cache.row_k", 128, -1),
          ("cache.n_pages", 1 << 31, -7), ("page_table", None, -1), ("lengths", None, -1), ("n_table", 0, -1), ("table_stride", -1, -1),
          ("n_table", (1 << 26) + 1, -7)]
BOUNDS_FAULTS = [("bounds.codes", None, -1), ("bounds.codes", 4104, -1), ("bounds.scales", None, -1), ("bounds.scales", 4098, -1)]


@pytest.mark.parametrize("kind,path,value,status", [
    *((kind, *fault) for kind in ("SplashCacheBoundArgs", "SplashCacheChooseArgs", "SplashCacheAttendArgs") for fault in FAULTS),
    *((kind, *fault) for kind in ("SplashCacheBoundArgs", "SplashCacheChooseArgs") for fault in BOUNDS_FAULTS),
    ("SplashCacheBoundArgs", "batch", 0, -1), ("SplashCacheBoundArgs", "newest", -1, -1), ("SplashCacheBoundArgs", "batch", (1 << 24) + 1, -7),
    ("SplashCacheChooseArgs", "q.dtype", 1, -2), ("SplashCacheChooseArgs", "q.size.1", 3, -1), ("SplashCacheChooseArgs", "q.size.1", 2 * 129, -7),
    ("SplashCacheChooseArgs", "q.size.3", 56, -1), ("SplashCacheChooseArgs", "q.size.2", (1 << 20) + 1, -7), ("SplashCacheChooseArgs", "q.data", None, -1),
    ("SplashCacheChooseArgs", "tables", None, -1), ("SplashCacheChooseArgs", "table_lengths", None, -1), ("SplashCacheChooseArgs", "count", 1, -1),
    ("SplashCacheChooseArgs", "first", -1, -1), ("SplashCacheChooseArgs", "last", 0, -1), ("SplashCacheChooseArgs", "first", (1 << 31) - 1, -1),
    ("SplashCacheChooseArgs", "count", (1 << 26) + 1, -7), ("SplashCacheAttendArgs", "window", 0, -1), ("SplashCacheAttendArgs", "q.size.0", 1 << 23, -7),
    ("SplashCacheAttendArgs", "q.dtype", 1, -2), ("SplashCacheAttendArgs", "o.size.2", 2, -1)])
def test_c_entry_points_refuse_before_they_touch_the_gpu(kind, path, value, status):
  fn = {"SplashCacheBoundArgs": "splash_cache_bound", "SplashCacheChooseArgs": "splash_cache_choose",
        "SplashCacheAttendArgs": "splash_cache_attend_tables"}[kind]
  a = _spoilt(kind, path, value)
  if path == "q.size.0":
    a.o.size[0] = value
  assert getattr(_native.lib(), fn)(C.byref(a), None) == status
  assert getattr(_native.lib(), fn)(None, None) == -1


def test_values_of_bounds_are_checked():
  lib, a = _native.lib(), _args("SplashCacheBoundArgs")
  assert lib.splash_cache_bound_values(None, C.byref(a.bounds), 4096, None) == lib.splash_cache_bound_values(C.byref(a.cache), None, 4096, None) == -1
  for values in (None, 4100):
    assert lib.splash_cache_bound_values(C.byref(a.cache), C.byref(a.bounds), values, None) == -1
  a.bounds.scales = None
  assert lib.splash_cache_bound_values(C.byref(a.cache), C.byref(a.bounds), 4096, None) == -1


def test_nothing_new_is_nothing_to_do():
  assert _native.lib().splash_cache_bound(C.byref(_spoilt("SplashCacheBoundArgs", "newest", 0)), None) == 0


def test_workspaces():
  lib = _native.lib()
  assert lib.splash_cache_choose_workspace_bytes(None) == lib.splash_cache_attend_tables_workspace_bytes(None) == 0
  a = _args("SplashCacheChooseArgs")
  assert lib.splash_cache_choose_workspace_bytes(C.byref(a)) == 0
  a.n_table = 40000
  size = 2 * 3 * 40000 * 4  # a score for each page of the tables of 2 heads and 3 queries
  assert lib.splash_cache_choose_workspace_bytes(C.byref(a)) == size
  assert lib.splash_cache_choose(C.byref(a), None) == -1  # it has none
  a.workspace, a.workspace_bytes = 4096, size - 1
  assert lib.splash_cache_choose(C.byref(a), None) == -1
  a.workspace, a.workspace_bytes = 4100, size
  assert lib.splash_cache_choose(C.byref(a), None) == -1
  a.count = 1
  assert lib.splash_cache_choose_workspace_bytes(C.byref(a)) == 0  # refused
  b = _args("SplashCacheAttendArgs")
  assert lib.splash_cache_attend_tables_workspace_bytes(C.byref(b)) == 0  # two pages: every item is one CTA's
  b.n_table = 4096
  size = lib.splash_cache_attend_tables_workspace_bytes(C.byref(b))
  assert 0 < size < 64 << 20
  assert lib.splash_cache_attend_tables(C.byref(b), None) == -1
  b.workspace, b.workspace_bytes = 4096, size - 1
  assert lib.splash_cache_attend_tables(C.byref(b), None) == -1


def test_up_to_8192_pages_need_no_workspace():
  lib, a = _native.lib(), _args("SplashCacheChooseArgs")
  for n_table, size in ((8192, 0), (8193, 2 * 3 * 8193 * 4)):
    a.n_table = n_table
    assert lib.splash_cache_choose_workspace_bytes(C.byref(a)) == size


def test_structs_have_the_layout_the_c_header_gives_them(tmp_path):
  root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
  structs = {"SplashPageBounds": "scales", "SplashCacheBoundArgs": "newest", "SplashCacheChooseArgs": "workspace_bytes", "SplashRotateArgs": "factor"}
  src = tmp_path / "layout.c"
  src.write_text('#include <stdio.h>\n#include "splash_b200.h"\nint main(void) {\n' + "".join(
      f'  printf("{n} %zu %zu\\n", sizeof({n}), offsetof({n}, {last}));\n' for n, last in structs.items()) + "  return 0;\n}\n")
  subprocess.run(["gcc", "-std=c99", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
  out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()
  for name, size, offset in zip(out[::3], out[1::3], out[2::3]):
    mirror = getattr(_native, name)
    assert C.sizeof(mirror) == int(size) and getattr(mirror, structs[name]).offset == int(offset), name
  assert len(out) == 3 * len(structs)


def test_the_oracle_bounds_logits():
  """With 8 bits left out the score is the largest logit that the bounds allow; with them it is off by half a step of q and of the
  bounds a channel, and rounding of 2^-20."""
  g = torch.Generator().manual_seed(0)
  k, q = torch.randn(6, 32, 64, generator=g), torch.randn(3, 64, generator=g)
  codes, scales = pages_ref.bounds(k)
  score = pages_ref.scores(q, codes, scales) * (q.abs().max() / 127)
  logits = (k @ q.T).amax((1, 2))
  off = 0.5 * scales * q.abs().sum(-1).max() + 0.5 * q.abs().max() / 127 * k.abs().amax((1, 2)) * 64
  assert (score >= logits - off * (1 + 2.0 ** -20)).all() and not math.isinf(float(score.max()))


@pytest.mark.parametrize("kw,message", [
    (dict(q=torch.zeros(1, 3, 1, 64)), "does not match a cache"), (dict(q=torch.zeros(1, 4, 1, 32)), "does not match a cache"),
    (dict(q=torch.zeros(4, 1, 64)), "does not match a cache"), (dict(q=torch.zeros(1, 0, 1, 64)), "does not match a cache"),
    (dict(q=torch.zeros(2, 4, 1, 64)), "q of 2 sequences, lengths of 1"), (dict(table=torch.zeros(1, 4)), "are int32"),
    (dict(table=torch.zeros(4, dtype=torch.int32)), r"expected \[B, pages\] and \[B\]"), (dict(table=torch.zeros(1, 0, dtype=torch.int32)), "of 0 pages"),
    (dict(lengths=torch.ones(2, dtype=torch.int32)), r"expected \[B, pages\] and \[B\]"), (dict(lengths=torch.ones(1)), "are int32"),
    (dict(q=torch.zeros(2, 4, 1, 64), table=torch.zeros(2, 4, dtype=torch.int32), lengths=torch.ones(4, dtype=torch.int32)[::2]), "lengths are contiguous"),
    *((bad, "expected first >= 0, last >= 1 and count >= first") for bad in (
        dict(count=0), dict(count=1), dict(count=2, first=2), dict(first=-1), dict(last=0), dict(count=1 << 32), dict(last=1 << 33, count=1 << 34)))])
def test_what_a_choice_is_refused_for(kw, message):
  """Each for its own reason, wherever the operands are."""
  with pytest.raises(ValueError, match=message):
    _choose(**kw)


def test_what_bounds_are_refused_for():
  cache = _cache()
  bounds, table, lengths = kv_cache.make_page_bounds(cache), torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
  for bad, message in (((table, lengths, -1), "newest is not negative"), ((table, lengths.repeat(2), 1), r"expected \[B, pages\] and \[B\]"),
                       ((table[:, :0], lengths, 1), "of 0 pages"), ((table.long(), lengths, 1), "are int32")):
    with pytest.raises(ValueError, match=message):
      kv_cache.bound_pages(cache, bounds, *bad)


TABLES_THAT_DO_NOT_MATCH = [
    ((1, 2, 1, 4), (1, 2), None, "do not match: expected .B, kv_heads, T, pages."), ((1, 2, 1, 4), (1, 2, 2), None, "do not match: expected .B, kv_heads"),
    ((1, 1, 1, 4), (1, 1, 1), None, "do not match: expected .B, kv_heads"), ((2, 2, 1, 4), (2, 2, 1), None, "do not match: expected .B, kv_heads"),
    ((1, 2, 3, 4), (1, 2, 3), None, "do not match: expected .B, kv_heads"), ((1, 2, 1, 4), (1, 2, 1), 5, "local_window_size goes by places"),
    ((1, 2, 1, 0), (1, 2, 1), None, "of 0 pages"), ((1, 2, 4), (1, 2), None, r"expected \[B, pages\] and \[B\]"),
    ((2, 4), (2,), None, "q of 1 sequences, lengths of 2")]


@pytest.mark.parametrize("table,lengths,window,message", TABLES_THAT_DO_NOT_MATCH)
def test_what_tables_are_refused_for(table, lengths, window, message):
  with pytest.raises(ValueError, match=message):
    kv_cache.attend(_cache(), torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16), torch.zeros(table, dtype=torch.int32),
                    torch.ones(lengths, dtype=torch.int32), local_window_size=window)
