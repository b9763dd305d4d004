"""What the quantised cache decides without a GPU: its layout, its refusals, slots, the checks of the C entry points."""
import ctypes as C
import re

import pytest
import torch
from torch.autograd import forward_ad

from oracle import kv_cache_ref
from tokamax_b200 import _native
from tokamax_b200 import kv_cache


def test_layout():
  cache = kv_cache.make_kv_cache(5, 32, 3, 80, fmt="int4", device="cpu")
  assert cache.group_size == 32 and cache.n_pages == 5  # rows of 80 are padded to 96
  assert cache.k_codes.shape == cache.v_codes.shape == (5, 3, 32, 48) and cache.k_scales.shape == (5, 3, 32, 3, 2)
  cache = kv_cache.make_kv_cache(2, 16, 1, 192, 128, fmt="int4", device="cpu")
  assert cache.group_size == 64 and cache.k_codes.shape[-1] == 96 and cache.v_scales.shape == (2, 1, 16, 2, 2)
  cache = kv_cache.make_kv_cache(2, 64, 1, 64, 96, fmt="e4m3", device="cpu")
  assert cache.k_codes.shape[-1] == cache.v_codes.shape[-1] == 96 and cache.k_scales.shape == (2, 1, 64)


@pytest.mark.parametrize("kw,error", [
    (dict(fmt="int8"), ValueError), (dict(page_size=24), ValueError), (dict(page_size=8), ValueError), (dict(n_pages=0), ValueError),
    (dict(kv_heads=0), ValueError), (dict(head_dim=60), ValueError), (dict(head_dim=0), ValueError),
    (dict(head_dim=320), NotImplementedError), (dict(group_size=16), ValueError), (dict(head_dim=96, group_size=64), ValueError),
    (dict(head_dim=192, head_dim_v=128, group_size=128), ValueError), (dict(fmt="e4m3", group_size=32), ValueError)])
def test_caches_that_cannot_be_made(kw, error):
  args = dict(n_pages=4, page_size=16, kv_heads=2, head_dim=64, device="cpu")
  args.update(kw)
  with pytest.raises(error):
    kv_cache.make_kv_cache(**args)


def test_slots():
  cache = kv_cache.make_kv_cache(9, 16, 1, 64, device="cpu")
  table = torch.tensor([[7, 2, -1], [0, 8, 3]], dtype=torch.int32)
  slots = kv_cache.slots_of(cache, table, torch.tensor([[0, 15, 16, 33, -1], [47, -2, 31, 5, 16]]))
  assert slots.tolist() == [[112, 127, 32, -1, -1], [63, -1, 143, 5, 128]]


def test_positions_behind_the_page_table_have_no_slot():
  cache = kv_cache.make_kv_cache(9, 16, 1, 64, device="cpu")
  table = torch.tensor([[7, 2], [0, -1]], dtype=torch.int32)
  slots = kv_cache.slots_of(cache, table, torch.tensor([[31, 32, 48, 2 ** 31 - 1], [15, 16, 33, -1]], dtype=torch.int32))
  assert slots.tolist() == [[47, -1, -1, -1], [15, -1, -1, -1]]
  far = kv_cache.slots_of(cache, table, torch.tensor([[2 ** 62], [0]]))
  assert far.dtype == torch.int64 and far.tolist() == [[-1], [0]]
  assert kv_cache.slots_of(cache, table[:, :0], torch.tensor([[0, -1], [5, 40]])).tolist() == [[-1, -1], [-1, -1]]
  assert kv_cache.slots_of(cache, table, torch.zeros(2, 0, dtype=torch.int32)).shape == (2, 0)


def test_a_cache_on_the_cpu_has_no_operators():
  cache = kv_cache.make_kv_cache(2, 16, 1, 64, device="cpu")
  x = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16)
  i = torch.zeros(1, dtype=torch.int32)
  for call in (lambda: kv_cache.append(cache, x, x, i[None]), lambda: kv_cache.read(cache, i[None], i, 4),
               lambda: kv_cache.attend(cache, x, i[None], i)):
    with pytest.raises(RuntimeError, match="CUDA"):
      call()


def _calls(cache):
  """A call of each operator, by its floating operands."""
  i = torch.zeros(1, dtype=torch.int32)
  return {"append": (lambda k, v: kv_cache.append(cache, k, v, i[None]), 2), "read": (lambda x: kv_cache.read(cache, i[None], i + 1, 4)[0] + x.sum(), 1),
          "attend": (lambda q: kv_cache.attend(cache, q, i[None], i + 1), 1)}


@pytest.mark.parametrize("name", ["append", "read", "attend"])
def test_calls_are_not_recorded(name):
  """A graph of torch.jit.trace would give back memory that nothing wrote."""
  call, n = _calls(kv_cache.make_kv_cache(2, 16, 1, 64, device="cpu"))[name]
  operands = tuple(torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16) for _ in range(n))
  with pytest.raises(NotImplementedError, match="recorded"):
    torch.jit.trace(call, operands, check_trace=False)
  with pytest.raises(RuntimeError, match="CUDA"):  # (and nothing of it is left over)
    call(*operands)


@pytest.mark.parametrize("name,which", [("append", 0), ("append", 1), ("attend", 0)])
def test_operands_with_a_derivative_are_refused(name, which):
  """A gradient or a tangent of forward mode would be lost without a word."""
  call, n = _calls(kv_cache.make_kv_cache(2, 16, 1, 64, device="cpu"))[name]
  operands = [torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16) for _ in range(n)]
  plain = operands[which]
  operands[which] = plain.clone().requires_grad_(True)
  with pytest.raises(NotImplementedError, match="gradient"):
    call(*operands)
  with forward_ad.dual_level():
    operands[which] = forward_ad.make_dual(plain, torch.ones_like(plain))
    with pytest.raises(NotImplementedError, match="tangent"):
      call(*operands)
    with torch.inference_mode(), pytest.raises(RuntimeError, match="CUDA"):  # (which takes no derivatives of either kind)
      call(*operands)


def test_sinks_with_a_derivative_are_refused():
  cache = kv_cache.make_kv_cache(2, 16, 1, 64, device="cpu")
  q, i, sinks = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32), torch.zeros(1)
  with pytest.raises(NotImplementedError, match="sinks requires"):
    kv_cache.attend(cache, q, i[None], i, sinks=sinks.clone().requires_grad_(True))
  with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="sinks has a tangent"):
    kv_cache.attend(cache, q, i[None], i, sinks=forward_ad.make_dual(sinks, torch.ones(1)))


def _args(kind):
  """Arguments that pass every check up to the missing device; addresses that nobody reads."""
  a = getattr(_native, kind)()
  c = a.cache
  c.k_codes = c.k_scales = c.v_codes = c.v_scales = 4096
  c.n_pages, c.format, c.page_size, c.kv_heads, c.group, c.head_dim, c.head_dim_v, c.row_k, c.row_v = 4, 0, 16, 2, 32, 64, 64, 64, 64
  for name in ("k", "v", "q", "o"):
    if hasattr(a, name):
      t = getattr(a, name)
      t.data, t.dtype = 4096, 0
      for i, (n, s) in enumerate(zip((1, 2, 3, 64), (384, 192, 64, 1))):
        t.size[i], t.stride[i] = n, s
  if kind != "SplashCacheAppendArgs":
    a.page_table, a.lengths, a.table_stride, a.n_table = 4096, 4096, 2, 2
  else:
    a.slots, a.slot_stride = 4096, 3
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


CACHE_FAULTS = [("cache.k_codes", None, -1), ("cache.v_scales", 4104, -1), ("cache.page_size", 24, -1), ("cache.page_size", 8, -1),
                ("cache.group", 16, -1), ("cache.format", 2, -2), ("cache.head_dim", 60, -1), ("cache.head_dim", 320, -2),
                ("cache.row_k", 128, -1), ("cache.kv_heads", 0, -1), ("cache.n_pages", 0, -1), ("cache.n_pages", 1 << 31, -7)]


@pytest.mark.parametrize("kind,path,value,status", [
    *((kind, *fault) for kind in ("SplashCacheAppendArgs", "SplashCacheReadArgs", "SplashCacheAttendArgs") for fault in CACHE_FAULTS),
    ("SplashCacheAppendArgs", "k.dtype", 2, -2), ("SplashCacheAppendArgs", "k.dtype", 3, -1), ("SplashCacheAppendArgs", "slots", None, -1),
    ("SplashCacheAppendArgs", "v.size.2", 4, -1), ("SplashCacheAppendArgs", "k.stride.2", 60, -1), ("SplashCacheAppendArgs", "k.stride.3", 2, -1),
    ("SplashCacheAppendArgs", "k.data", 4100, -1), ("SplashCacheAppendArgs", "slot_stride", -1, -1),
    ("SplashCacheReadArgs", "page_table", None, -1), ("SplashCacheReadArgs", "n_table", 0, -1), ("SplashCacheReadArgs", "k.size.0", 2, -1),
    ("SplashCacheAttendArgs", "q.dtype", 1, -2), ("SplashCacheAttendArgs", "q.size.1", 3, -1), ("SplashCacheAttendArgs", "lengths", None, -1),
    ("SplashCacheAttendArgs", "n_table", (1 << 26) + 1, -7), ("SplashCacheReadArgs", "k.size.0", 0, -1),
    ("SplashCacheAttendArgs", "soft_cap", -1.0, -1), ("SplashCacheAttendArgs", "soft_cap", float("nan"), -1),
    ("SplashCacheAttendArgs", "o.size.3", 56, -1)])
def test_c_entry_points_refuse_before_they_touch_the_gpu(kind, path, value, status):
  fn = {"SplashCacheAppendArgs": "splash_cache_append", "SplashCacheReadArgs": "splash_cache_read",
        "SplashCacheAttendArgs": "splash_cache_attend"}[kind]
  assert getattr(_native.lib(), fn)(C.byref(_spoilt(kind, path, value)), None) == status
  assert getattr(_native.lib(), fn)(None, None) == -1


def test_a_scale_that_is_no_number():
  a = _spoilt("SplashCacheAttendArgs", "scale", float("nan"))
  assert _native.lib().splash_cache_attend(C.byref(a), None) == -1
  assert _native.lib().splash_cache_attend_workspace_bytes(C.byref(a)) == 0


def test_workspace():
  lib = _native.lib()
  short = _args("SplashCacheAttendArgs")  # two pages: every item is one CTA's
  assert lib.splash_cache_attend_workspace_bytes(C.byref(short)) == 0
  a = _spoilt("SplashCacheAttendArgs", "n_table", 4096)
  assert lib.splash_cache_attend_workspace_bytes(C.byref(a)) == 0  # (a window of 0: each query sees its own key)
  a.window = -1
  size = lib.splash_cache_attend_workspace_bytes(C.byref(a))
  assert 0 < size < 64 << 20
  assert lib.splash_cache_attend(C.byref(a), None) == -1  # it has none
  assert lib.splash_cache_attend_workspace_bytes(C.byref(_spoilt("SplashCacheAttendArgs", "q.size.1", 3))) == 0
  assert lib.splash_cache_attend_workspace_bytes(None) == 0
  a.workspace, a.workspace_bytes = 4096, size - 1
  assert lib.splash_cache_attend(C.byref(a), None) == -1


def test_structs_have_the_layout_the_c_header_gives_them(tmp_path):
  import os
  import subprocess

  root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
  structs = {"SplashKvCache": "row_v", "SplashCacheAppendArgs": "slot_stride", "SplashCacheReadArgs": "lengths",
             "SplashCacheAttendArgs": "workspace_bytes"}
  src = tmp_path / "layout.c"
  src.write_text('#include <stdio.h>\n#include "splash_b200.h"\nint main(void) {\n' + "".join(
      f'  printf("{n} %zu %zu\\n", sizeof({n}), offsetof({n}, {last}));\n' for n, last in structs.items()) + "  return 0;\n}\n")
  subprocess.run(["gcc", "-std=c99", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
  out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()
  for name, size, offset in zip(out[::3], out[1::3], out[2::3]):
    mirror = getattr(_native, name)
    assert C.sizeof(mirror) == int(size) and getattr(mirror, structs[name]).offset == int(offset), name
  assert len(out) == 3 * len(structs)


def test_the_oracle_rounds_as_the_types_do():
  """e4m3 by steps of its exponents against torch's own conversion; a scale of exactly one keeps x / scale exact."""
  g = torch.Generator().manual_seed(0)
  x = torch.randn(64, 64, generator=g) * torch.exp2(torch.randint(-12, 6, (64, 64), generator=g).float())
  x[:, 0] = 448.0
  assert torch.equal(kv_cache_ref.held(x, "e4m3", None).float(), x.clamp(-448, 448).to(torch.float8_e4m3fn).float())
  y = torch.arange(16.0).repeat(2)[None]
  assert torch.equal(kv_cache_ref.held(y, "int4", 32), y.double())
