"""The quantised key / value cache against its definition in 64 bits: rows written and read back, attention over them."""
import ctypes as C
import math

import pytest
import torch

from oracle import kv_cache_ref
from tokamax_b200 import _native
from tokamax_b200 import kv_cache

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ROUNDOFF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step of the type, at most, of a value
FORMATS = [("int4", 32), ("int4", 64), ("int4", 128), ("e4m3", None)]


class Store:
  """A cache with sequences of the given lengths on scattered pages, and what it should hold."""

  def __init__(self, lengths, *, heads=2, d=64, d_v=None, fmt="int4", group=32, page=16, dtype=torch.bfloat16, seed=0, spare=0,
               keys=None, values=None):
    g = torch.Generator().manual_seed(seed)
    d_v = d if d_v is None else d_v
    used = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(used) + 1 + spare, generator=g).tolist()
    width = max(max(used), 1)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(used):
      table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
      at += n
    self.fmt, self.group, self.d, self.d_v, self.heads, self.page = fmt, group, d, d_v, heads, page
    self.lengths_list = lengths
    self.cache = kv_cache.make_kv_cache(len(order), page, heads, d, d_v, fmt=fmt, group_size=group, device=DEV)
    self.table, self.lengths = table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV)
    longest = max(max(lengths), 1)
    make = lambda c: torch.randn(len(lengths), heads, longest, c, generator=g)  # noqa: E731
    k = make(d) + torch.randn(1, heads, 1, d, generator=g) ** 3  # some channels of a head carry an offset
    v = make(d_v) * torch.exp(torch.randn(len(lengths), heads, longest, 1, generator=g))
    self.k, self.v = (x.to(dtype) for x in (k if keys is None else keys(k), v if values is None else values(v)))
    positions = torch.arange(longest)[None, :].expand(len(lengths), -1)
    positions = torch.where(positions < torch.tensor(lengths)[:, None], positions, -1).to(DEV)
    self.slots = kv_cache.slots_of(self.cache, self.table, positions)
    kv_cache.append(self.cache, self.k.to(DEV), self.v.to(DEV), self.slots)

  def held(self, b):
    n = self.lengths_list[b]
    return tuple(kv_cache_ref.held(x[b, :, :n], self.fmt, self.group) for x in (self.k, self.v))


def _check_read(store, dtype, max_len):
  k, v = kv_cache.read(store.cache, store.table, store.lengths, max_len, dtype=dtype)
  for b, n in enumerate(store.lengths_list):
    n = min(n, max_len)
    for got, ref in zip((k[b], v[b]), store.held(b)):
      assert got.dtype == dtype and not got[:, n:].any()
      # zero + scale * code is rounded to 32 bits once (zero and the product are exact), then to dtype
      assert torch.equal(got[:, :n].cpu(), ref[:, :n].float().to(dtype))


@pytest.mark.parametrize("fmt,group", FORMATS)
@pytest.mark.parametrize("d,d_v", [(64, 64), (80, 80), (96, 96), (128, 128), (128, 64), (192, 128), (160, 160), (256, 256), (8, 8)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_come_back_as_the_format_holds_them(fmt, group, d, d_v, dtype):
  try:
    store = Store([0, 1, 77, 33], heads=3, d=d, d_v=d_v, fmt=fmt, group=group, page=32, dtype=dtype)
  except ValueError as e:
    assert "group_size" in str(e) and group in (64, 128)
    return
  _check_read(store, torch.float32, 77)
  _check_read(store, dtype, 96)
  _check_read(store, torch.bfloat16, 50)  # shorter than the sequences


def test_f32_rows_are_held_to_within_half_a_step():
  """In 32 bits x / scale may fall on the other side of a tie than in 64: a step more, for values within rounding of one."""
  for fmt, group in FORMATS:
    store = Store([300], heads=2, d=128, fmt=fmt, group=group, page=64, dtype=torch.float32)
    k, v = kv_cache.read(store.cache, store.table, store.lengths, 300, dtype=torch.float32)
    for got, ref, x in zip((k[0], v[0]), store.held(0), (store.k[0], store.v[0])):
      off = (got.cpu().double() - ref).abs() > 2.0 ** -22 * (1 + ref.abs())
      assert off.float().mean() <= 1e-4, fmt
      if fmt == "int4":
        parts = x.double().unflatten(-1, (-1, group))
        scale = ((parts.amax(-1) - parts.amin(-1)) / 15).repeat_interleave(group, -1)
        # half a step; a scale rounded down leaves the last code 15 * 2^-9 of a step short; the zero's own rounding
        bound = scale * (0.5 + 15 * 2.0 ** -9) * (1 + 2.0 ** -8) + 2.0 ** -8 * parts.amin(-1).abs().repeat_interleave(group, -1)
        assert ((got.cpu().double() - x.double()).abs() <= bound).all()


def test_f32_rows_of_extreme_sizes():
  """Ranges beyond 32 bits are NaN; rows of subnormal scales, which divide by other means, hold what they can."""
  x = torch.zeros(1, 1, 4, 64)
  x[0, 0, 0, :2] = torch.tensor([3e38, -3e38])
  x[0, 0, 1] = torch.arange(64) * 1e-30
  x[0, 0, 2] = torch.arange(64) * 1e-38
  x[0, 0, 3] = torch.arange(64) * 1e30
  store = Store([4], heads=1, d=64, group=64, dtype=torch.float32, keys=lambda _: x, values=lambda _: x)
  k, _ = kv_cache.read(store.cache, store.table, store.lengths, 4, dtype=torch.float32)
  got = k[0, 0].cpu().double()
  assert got[0].isnan().all()
  for row, size in ((1, 1e-30), (2, 1e-38), (3, 1e30)):
    # half a step of 63 / 15, and a scale of 8 bits (7 below 2^-126, where steps of bf16 are 2^-133)
    step = 63 * size / 15
    assert ((got[row] - x[0, 0, row].double()).abs() <= step / 2 + 15 * (step * 2.0 ** -8 + 2.0 ** -134)).all(), row


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_int4_rows_of_subnormal_scales(dtype):
  """Scales of few bits: codes are clamped to 0 .. 15, and a channel's has no part in its neighbours'."""
  tops = [1, 7, 8, 15, 22, 23, 100, 217, 240, 255]
  x = torch.zeros(1, 1, 2 * len(tops), 64)
  for i, top in enumerate(tops):
    for row, least in ((2 * i, 0), (2 * i + 1, -3)):
      x[0, 0, row] = least + torch.arange(64) % (top + 1)
      x[0, 0, row, 5::7] = least + top
      x[0, 0, row, 32:] += 9  # (of another group: the same range)
  x = (x.double() * 2.0 ** -133).to(dtype)
  assert x.double().mul(2.0 ** 133).frac().abs().max() == 0 and x.double().max() > 255 * 2.0 ** -133
  store = Store([x.shape[2]], heads=1, d=64, group=32, dtype=dtype, keys=lambda _: x, values=lambda _: x)
  k, _ = kv_cache.read(store.cache, store.table, store.lengths, x.shape[2], dtype=torch.float32)
  assert torch.equal(k[0].cpu().double(), store.held(0)[0])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_values_beside_a_tie_are_rounded_once(dtype):
  """scale * code half way between two values of the type, and a zero far below: rounding to 32 bits first loses the zero, and the
  tie then goes to the even one."""
  x = torch.zeros(1, 1, 8, 64)
  for row, (scale, least) in enumerate([(255.0, 2.0 ** -30), (255.0, -2.0 ** -30), (129.0, 2.0 ** -25), (129.0, -2.0 ** -25), (1.9921875, 2.0 ** -38),
                                        (1.9921875, -2.0 ** -38), (131.0, -2.0 ** -38), (253.0, 2.0 ** -38)]):
    x[0, 0, row] = torch.arange(64) % 16 * scale
    x[0, 0, row, ::16] = least
  store = Store([8], heads=1, d=64, group=64, dtype=torch.float32, keys=lambda _: x, values=lambda _: -x)
  k, v = kv_cache.read(store.cache, store.table, store.lengths, 8, dtype=dtype)
  twice = False
  for got, ref in zip((k[0], v[0]), store.held(0)):
    # rounded to odd in 32 bits, then to the type: once in all
    near = ref.float()
    other = torch.nextafter(near, torch.where(ref > near.double(), math.inf, -math.inf))
    odd = torch.where((near.double() == ref) | (near.view(torch.int32) & 1 == 1), near, other)
    assert torch.equal(got.cpu(), odd.to(dtype))
    twice = twice or not torch.equal(odd.to(dtype), near.to(dtype))
  assert twice


def test_tokens_of_a_projection_are_written_through_their_strides():
  store = Store([40, 23], heads=2, d=64, group=64)
  fresh = Store([40, 23], heads=2, d=64, group=64, seed=1)
  qkv = torch.zeros(2, 40, 3, 2, 64, dtype=torch.bfloat16, device=DEV)
  qkv[:, :, 1] = store.k.to(DEV).transpose(1, 2)
  qkv[:, :, 2] = store.v.to(DEV).transpose(1, 2)
  k, v = qkv[:, :, 1].transpose(1, 2), qkv[:, :, 2].transpose(1, 2)
  assert not k.is_contiguous()
  slots = kv_cache.slots_of(fresh.cache, fresh.table, torch.where(store.slots >= 0, torch.arange(40, device=DEV)[None], -1))
  odd = torch.full((2, 81), -7, dtype=torch.int32, device=DEV)[:, ::2][:, :40]  # int32, every second element
  odd.copy_(slots)
  kv_cache.append(fresh.cache, k, v, odd)
  fresh.k, fresh.v = store.k, store.v
  _check_read(fresh, torch.float32, 40)
  odd_k = torch.zeros(2, 2, 40, 65, dtype=torch.bfloat16, device=DEV)[..., 1:]  # rows that start between 16-byte boundaries
  odd_k.copy_(k)
  kv_cache.append(fresh.cache, odd_k, v, slots)
  _check_read(fresh, torch.float32, 40)


def test_slots_outside_the_cache_are_not_kept():
  store = Store([16, 16], heads=1, d=64, spare=2)
  before = [t.clone() for t in (store.cache.k_codes, store.cache.k_scales, store.cache.v_codes, store.cache.v_scales)]
  n = store.cache.n_pages * 16
  slots = torch.tensor([[-1, n, n + 5, -(1 << 40), 1 << 40]], device=DEV)
  x = torch.randn(1, 1, 5, 64, device=DEV)
  kv_cache.append(store.cache, x, x, slots)
  kv_cache.append(store.cache, x[:, :, :3], x[:, :, :3], slots[:, :3].int())
  for a, t in zip(before, (store.cache.k_codes, store.cache.k_scales, store.cache.v_codes, store.cache.v_scales)):
    assert torch.equal(a, t)


@pytest.mark.parametrize("fmt,dtype", [("int4", torch.bfloat16), ("e4m3", torch.float32)])
def test_more_sequences_than_a_grid_has_blocks(fmt, dtype):
  """Written, read and attended to: 70000 sequences of 0 .. 2 tokens, two of a page each."""
  batch, d = 70000, 64
  g = torch.Generator(device=DEV).manual_seed(0)
  cache = kv_cache.make_kv_cache(batch // 2, 16, 1, d, fmt=fmt, device=DEV)
  lengths = (torch.arange(batch, device=DEV) % 3).int()
  table = (torch.arange(batch, device=DEV) // 2 % (batch // 2)).int()[:, None]
  k = torch.randn(batch, 1, 2, d, generator=g, device=DEV).to(torch.bfloat16)
  k[1::2] = k[::2]  # (the two sequences of a page are one)
  positions = torch.arange(2, device=DEV)[None].expand(batch, -1).clone()
  positions[1::2] = -1
  kv_cache.append(cache, k, k, kv_cache.slots_of(cache, table, positions))
  got, _ = kv_cache.read(cache, table, lengths, 2, dtype=dtype)
  want = kv_cache_ref.held(k, fmt, cache.group_size).to(DEV)
  want[lengths < 2, :, 1] = 0
  want[lengths < 1] = 0
  assert torch.equal(got, want.float().to(dtype))
  o = kv_cache.attend(cache, k[:, :, :1], table, lengths, logits_scale=0.0)
  mean = torch.where(lengths > 1, 0.5, 1.0)[:, None, None] * want.sum(2)  # a scale of 0: all keys alike
  # a term is rounded by 2^-12 of a product (P * scale), which is a group's range at most, and the sum by 2^-9 of it
  assert ((o[:, :, 0].double() - mean).abs() <= 2.0 ** -8 * want.abs().amax((1, 2, 3))[:, None, None]).all()


def test_pages_outside_the_cache_read_as_zeros_and_are_not_seen():
  store = Store([70, 64, 100], heads=2, d=64, spare=3)
  table = store.table.clone()
  table[0, 1], table[1, 0], table[2, 2], table[2, 6] = -1, store.cache.n_pages, 2 ** 31 - 1, -5
  k, _ = kv_cache.read(store.cache, table, store.lengths, 100, dtype=torch.float32)
  whole, _ = kv_cache.read(store.cache, store.table, store.lengths, 100, dtype=torch.float32)
  seen = torch.ones(3, 100, dtype=torch.bool)
  seen[0, 16:32], seen[1, :16], seen[2, 32:48], seen[2, 96:] = False, False, False, False
  assert torch.equal(k, torch.where(seen[:, None, :, None].to(DEV), whole, 0.0))
  _check_attend(store, q_heads=4, t=3, seen=seen, table=table)


@pytest.mark.parametrize("fmt,group", FORMATS)
def test_groups_with_values_that_are_not_finite_are_nan_and_constant_ones_exact(fmt, group):
  def spoil(x):
    x[0, 0, 0, 3] = math.inf
    x[0, 0, 1, 70] = -math.inf
    x[0, 1, 2, 127] = math.nan
    x[0, 1, 3] = 0.0
    x[0, 1, 4] = 1.5
    x[0, 1, 5] = -0.0
    return x

  store = Store([6], heads=2, d=128, fmt=fmt, group=group, keys=spoil, values=spoil)
  k, v = kv_cache.read(store.cache, store.table, store.lengths, 6, dtype=torch.float32)
  for got, ref in zip((k[0], v[0]), store.held(0)):
    assert torch.equal(got.cpu().isnan(), ref.isnan()) and int(ref.isnan().sum()) > 0
    # values near 1.5 of an e4m3 row are a step of its scale's rounding away; an int4 group of one value is exact
    assert torch.allclose(got.cpu().double().nan_to_num(), ref.nan_to_num(), rtol=2.0 ** -22, atol=0)
  if fmt == "int4":
    assert (k[0, 1, 4] == 1.5).all() and not k[0, 1, 3].any()


# ----------------------------------------------------------------------------------------------
# attention
# ----------------------------------------------------------------------------------------------
def _check_attend(store, *, q_heads, t=1, window=None, soft_cap=None, sinks=None, seen=None, table=None, dtype=torch.bfloat16,
                  q_scale=1.5, scale=None, seed=5):
  g = torch.Generator().manual_seed(seed)
  scale = store.d ** -0.5 if scale is None else scale
  q = (torch.randn(len(store.lengths_list), t, q_heads, store.d, generator=g) * q_scale).to(dtype).transpose(1, 2)
  o, res = kv_cache.attend(store.cache, q.to(DEV), store.table if table is None else table, store.lengths, logits_scale=scale,
                           local_window_size=window, logits_soft_cap=soft_cap,
                           sinks=None if sinks is None else sinks.to(DEV), save_residuals=True)
  assert o.dtype == dtype and o.shape == (*q.shape[:3], store.d_v)
  for b, n in enumerate(store.lengths_list):
    k, v = store.held(b)
    moved = kv_cache_ref.products(store.v[b, :, :n], store.fmt, store.group)
    ref, lse, top, size, moved = kv_cache_ref.attend(q[b].double(), k, v, scale=scale, window=window, soft_cap=soft_cap, sinks=sinks,
                                                     seen=None if seen is None else seen[b, :n], weights=moved)
    # Rounding: of P * scale to f16, 2^-11 of each term, or to two of them for f16 outputs, 2^-22 (plus a little for sums in 32
    # bits: 2^-18); of logits, 2^-24 of each
    # of some hundred partial sums of size |q| |k| scale, which moves each p, and with it o, by up to twice that in all; of
    # o to its type.
    logits = (q[b].double().norm(dim=-1).max() * (k.norm(dim=-1).max() if n else 0.0) * abs(scale)).clamp_min(1.0)
    slack = 2.0 ** -18 * logits
    err = (o[b].cpu().double() - ref).abs()
    before = ((ROUNDOFF[torch.float16] if dtype == torch.bfloat16 else 2.0 ** -22) + 2.0 ** -18) * moved + 2 * slack * size + 1e-9
    least = 2.0 ** -25 if dtype == torch.float16 else 0.0  # half a step of f16's subnormals
    bound = before + ROUNDOFF[dtype] * (ref.abs() + before) + least
    assert (err <= bound).all(), (b, n, float(err.max()), float((err / bound).max()))
    for got, want in ((res["logsumexp"], lse), (res["max_logits"], top)):
      got, dead = got[b].cpu().double(), want == kv_cache_ref.MASK_VALUE
      assert (got[dead] <= -2e38).all() and not o[b].cpu()[dead].any()
      assert ((got - want).abs()[~dead] <= slack + 2.0 ** -20 * (1 + want.abs()[~dead])).all()
  return o


@pytest.mark.parametrize("fmt,group", FORMATS)
@pytest.mark.parametrize("d,d_v", [(64, 64), (80, 80), (96, 96), (128, 128), (128, 64), (192, 128), (160, 160), (256, 256), (8, 8)])
@pytest.mark.parametrize("q_heads,t", [(2, 1), (6, 1), (16, 1), (10, 5)])
def test_attention_of_every_shape(fmt, group, d, d_v, q_heads, t):
  try:
    store = Store([0, 1, 7, 63, 64, 65, 700], d=d, d_v=d_v, fmt=fmt, group=group, page=16)
  except ValueError as e:
    assert "group_size" in str(e) and group in (64, 128)
    return
  _check_attend(store, q_heads=q_heads, t=t)


@pytest.mark.parametrize("page", [16, 32, 64, 256])
@pytest.mark.parametrize("fmt", ["int4", "e4m3"])
@pytest.mark.parametrize("lengths", [[2900], [257, 4097], list(range(3, 43))])
def test_rows_shared_by_many_ctas_and_ctas_with_many_rows(page, fmt, lengths):
  store = Store(lengths, heads=1, d=128, fmt=fmt, group=64 if fmt == "int4" else None, page=page)
  first = _check_attend(store, q_heads=4)
  again = _check_attend(store, q_heads=4)
  assert torch.equal(first, again)


@pytest.mark.parametrize("fmt,group", FORMATS)
@pytest.mark.parametrize("d,d_v", [(64, 64), (96, 96), (192, 128), (256, 256)])
@pytest.mark.parametrize("q_heads,t", [(2, 1), (16, 1), (10, 4)])
def test_f16_outputs(fmt, group, d, d_v, q_heads, t):
  try:
    store = Store([33, 700], d=d, d_v=d_v, fmt=fmt, group=group, dtype=torch.float16)
  except ValueError:
    assert group in (64, 128)
    return
  _check_attend(store, q_heads=q_heads, t=t, dtype=torch.float16)


@pytest.mark.parametrize("fmt", ["int4", "e4m3"])
@pytest.mark.parametrize("most", [90, 2500])  # every item one CTA's, or shares of them all
def test_more_sequences_than_a_cta_has_threads(fmt, most):
  lengths = [i * 37 % 90 for i in range(150)] + [most] + [i * 53 % 91 for i in range(149)] + [0, 0]
  store = Store(lengths, heads=1, d=64, fmt=fmt, group=32 if fmt == "int4" else None, page=16)
  _check_attend(store, q_heads=2)


@pytest.mark.parametrize("fmt", ["int4", "e4m3"])
@pytest.mark.parametrize("window", [0, 1, 15, 100, 5000, 2 ** 31 - 1])
@pytest.mark.parametrize("t", [1, 9])
def test_window(fmt, window, t):
  store = Store([1, 8, 9, 100, 1000, 1300], d=64, fmt=fmt, group=32 if fmt == "int4" else None)
  _check_attend(store, q_heads=4, t=t, window=window)


@pytest.mark.parametrize("fmt", ["int4", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_soft_cap_and_sinks(fmt, dtype):
  store = Store([0, 1, 33, 900, 2000], d=128, fmt=fmt, group=64 if fmt == "int4" else None, page=64, dtype=dtype)
  sinks = torch.tensor([0.5, -1.0, 2.0, 30.0, -40.0, 0.0])
  _check_attend(store, q_heads=6, soft_cap=5.0, dtype=dtype)
  _check_attend(store, q_heads=6, sinks=sinks, dtype=dtype)
  _check_attend(store, q_heads=6, t=2, soft_cap=30.0, sinks=sinks, window=64, dtype=dtype)


@pytest.mark.parametrize("fmt", ["int4", "e4m3"])
@pytest.mark.parametrize("soft_cap", [0.5, 50.0, 1000.0, 1e5])
@pytest.mark.parametrize("q_heads,t", [(4, 1), (8, 4), (10, 4)])
def test_soft_caps_far_above_and_below_the_logits(fmt, soft_cap, q_heads, t):
  """tanh's error is 1.1e-7 of itself up to 1/2 and 1.7e-7 beyond, so that a logit's is 4e-7 of the logit at most: well inside what
  _check_attend allows for its products, at any cap."""
  store = Store([1, 65, 700, 1300], d=128, fmt=fmt, group=64 if fmt == "int4" else None, page=64)
  _check_attend(store, q_heads=q_heads, t=t, soft_cap=soft_cap)


def test_sizes_of_scales_and_queries():
  """Tokens whose values differ by powers of ten, queries that are large, small and zero."""
  for fmt, group in FORMATS:
    gain = torch.tensor([1e-3, 1.0, 30.0, 0.0, 200.0]).repeat(140)[None, None, :700, None]
    store = Store([700, 5], d=128, fmt=fmt, group=group, values=lambda v: v * gain)  # pylint: disable=cell-var-from-loop
    for q_scale, scale in ((1.5, None), (3e-3, 10.0), (900.0, 2e-4), (0.0, 1.0), (1.5, -0.1), (1.5, 0.0)):
      _check_attend(store, q_heads=4, t=2, q_scale=q_scale, scale=scale)
    alike = Store([300], d=128, fmt=fmt, group=group, values=lambda v: v * 3e-6)
    _check_attend(alike, q_heads=4)


@pytest.mark.parametrize("fmt,group", FORMATS)
def test_what_lies_in_places_that_are_not_seen_has_no_part(fmt, group):
  """NaN behind the end of a sequence, in pages that nobody holds, and in keys that a window leaves out."""
  store = Store([50, 21], d=128, fmt=fmt, group=group, page=64, spare=2)
  clean = _check_attend(store, q_heads=4, t=2, window=20)
  store.cache.k_scales.view(torch.int16)[store.cache.k_scales == 0] = 0x7fff  # everything never written
  store.cache.v_scales.view(torch.int16)[store.cache.v_scales == 0] = 0x7fff
  bad = torch.full((1, 2, 1, 128), math.nan, device=DEV)
  kv_cache.append(store.cache, bad, bad, store.slots[:1, 5:6])  # in sequence 0, far outside the window
  assert torch.equal(clean, _attend_again(store, 4, 2, 20))
  kv_cache.append(store.cache, bad, bad, store.slots[:1, 48:49])  # query 0 stands at 48: both rows see it
  o = _attend_again(store, 4, 2, 20)
  assert o[0].isnan().all() and torch.equal(o[1], clean[1])
  kv_cache.append(store.cache, store.k[:1, :, 48:49].to(DEV), store.v[:1, :, 48:49].to(DEV), store.slots[:1, 48:49])
  kv_cache.append(store.cache, bad, bad, store.slots[:1, 49:50])  # the newest key: not seen by the query before it
  o = _attend_again(store, 4, 2, 20)
  assert torch.equal(o[0, :, 0], clean[0, :, 0]) and o[0, :, 1].isnan().all()


def _attend_again(store, q_heads, t, window):
  g = torch.Generator().manual_seed(5)
  q = (torch.randn(len(store.lengths_list), t, q_heads, store.d, generator=g) * 1.5).to(torch.bfloat16).transpose(1, 2)
  return kv_cache.attend(store.cache, q.to(DEV), store.table, store.lengths, logits_scale=store.d ** -0.5, local_window_size=window)


@pytest.mark.parametrize("fmt,group", FORMATS)
@pytest.mark.parametrize("d,d_v", [(64, 64), (96, 96), (128, 128), (192, 128), (160, 160), (256, 256)])
def test_row_tiles_and_page_tables_of_every_kind(fmt, group, d, d_v):
  """Up to 32 rows a tile, more in several; short tables (an item is one CTA's), long ones, and very long ones (wide heads then
  take 16 rows a tile)."""
  for page, lengths in ((16, [300, 40]), (256, [3000, 0, 17])):
    try:
      store = Store(lengths, d=d, d_v=d_v, fmt=fmt, group=group, page=page)
    except ValueError:
      assert group in (64, 128)
      return
    for q_heads, t in ((2, 3), (4, 6), (6, 7), (8, 8), (4, 19)):
      _check_attend(store, q_heads=q_heads, t=t)
    wide = torch.full((len(lengths), (1 << 18) // page), -1, dtype=torch.int32, device=DEV)
    wide[:, :store.table.shape[1]] = store.table
    _check_attend(store, q_heads=20, t=2, table=wide)


def test_lengths_beyond_the_page_table_and_below_zero():
  store = Store([64, 64], d=64, page=16)
  lengths = torch.tensor([80, -3], dtype=torch.int32, device=DEV)  # the table holds 64 tokens
  q = torch.randn(2, 2, 1, 64, device=DEV, dtype=torch.bfloat16)
  o = kv_cache.attend(store.cache, q, store.table, lengths, logits_scale=0.1)
  want = kv_cache.attend(store.cache, q, store.table, store.lengths, logits_scale=0.1)
  assert torch.equal(o[0], want[0]) and not o[1].any()
  k, _ = kv_cache.read(store.cache, store.table, lengths, 96)
  assert k[0, :, 63].any() and not k[0, :, 64:].any() and not k[1].any()


def test_queries_through_their_strides_and_nothing_at_all():
  store = Store([90, 31], d=64, group=64)
  q = torch.randn(2, 4, 3, 64, device=DEV, dtype=torch.bfloat16)
  call = lambda x: kv_cache.attend(store.cache, x, store.table, store.lengths, logits_scale=0.1)  # noqa: E731
  want = call(q)
  wide = torch.zeros(2, 3, 9, 72, device=DEV, dtype=torch.bfloat16)
  wide[:, :, 2:6, :64] = q.transpose(1, 2)
  assert torch.equal(call(wide[:, :, 2:6, :64].transpose(1, 2)), want)
  odd = torch.zeros(2, 4, 3, 67, device=DEV, dtype=torch.bfloat16)[..., 3:]
  odd.copy_(q)
  assert torch.equal(call(odd), want)
  assert call(q[:, :, :0]).shape == (2, 4, 0, 64)
  empty = store.lengths[:0]
  assert kv_cache.attend(store.cache, q[:0], store.table[:0], empty).shape == (0, 4, 3, 64)
  assert kv_cache.read(store.cache, store.table, store.lengths, 0)[0].shape == (2, 2, 0, 64)
  kv_cache.append(store.cache, q[:, :2, :0], q[:, :2, :0], store.slots[:, :0])


@pytest.mark.parametrize("offset", [1, 4, 8])
def test_contiguous_tensors_that_begin_anywhere(offset):
  """Their rows lie one behind the other, but not on boundaries of 16 bytes: a copy, which contiguous() alone does not make."""
  store = Store([90, 31], d=64, group=64)
  g = torch.Generator(device=DEV).manual_seed(0)

  def shifted(*shape):
    x = torch.randn(math.prod(shape) + offset, generator=g, device=DEV).to(torch.bfloat16)
    return x[offset:].view(shape), x[offset:].clone().view(shape)

  (q, q_aligned), (k, k_aligned), (v, v_aligned) = shifted(2, 4, 3, 64), shifted(2, 2, 3, 64), shifted(2, 2, 3, 64)
  kv_cache.append(store.cache, k_aligned, v_aligned, store.slots[:, :3])
  want = kv_cache.attend(store.cache, q_aligned, store.table, store.lengths, logits_scale=0.1)
  store = Store([90, 31], d=64, group=64)
  kv_cache.append(store.cache, k, v, store.slots[:, :3])
  assert q.is_contiguous() and torch.equal(kv_cache.attend(store.cache, q, store.table, store.lengths, logits_scale=0.1), want)
  one = k[:1, :1, :1]  # a token: contiguous, whatever its strides are
  kv_cache.append(Store([3], heads=1, d=64).cache, one, one, torch.zeros(1, 1, dtype=torch.int32, device=DEV))


def test_offsets_beyond_32_bits():
  """Codes of the pages at the end lie more than 2^32 bytes from the first."""
  page, heads, d = 4096, 8, 256
  n_pages = (1 << 32) // (page * heads * d) + 2
  cache = kv_cache.make_kv_cache(n_pages, page, heads, d, fmt="e4m3", device=DEV)
  g = torch.Generator(device=DEV).manual_seed(0)
  k, v = (torch.randn(1, heads, 100, d, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
  table = torch.tensor([[n_pages - 1], [0]], dtype=torch.int32, device=DEV)
  lengths = torch.tensor([100, 100], dtype=torch.int32, device=DEV)
  positions = torch.arange(100, device=DEV)[None]
  for row in range(2):
    kv_cache.append(cache, k, v, kv_cache.slots_of(cache, table[row:row + 1], positions))
  q = torch.randn(1, heads, 1, d, generator=g, device=DEV).to(torch.bfloat16).expand(2, -1, -1, -1)
  o = kv_cache.attend(cache, q, table, lengths, logits_scale=d ** -0.5)
  back, _ = kv_cache.read(cache, table, lengths, 100)
  assert torch.equal(o[0], o[1]) and torch.equal(back[0], back[1]) and back[0].any()
  assert torch.equal(back[0].cpu().double(), kv_cache_ref.held(k[0], "e4m3", None).to(torch.bfloat16).double())


def test_streams_and_graphs():
  store = Store([500, 900, 40], d=128, group=64, page=64)
  q = torch.randn(3, 4, 1, 128, device=DEV, dtype=torch.bfloat16)
  call = lambda: kv_cache.attend(store.cache, q, store.table, store.lengths, logits_scale=0.1)  # noqa: E731
  want = call()
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    outs = [call() for _ in range(20)]
  mine = [call() for _ in range(20)]  # two streams at a time: each call has a workspace of its own
  side.synchronize()
  assert all(torch.equal(o, want) for o in outs + mine)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    kv_cache.append(store.cache, q[:, :2], q[:, :2], store.slots[:, :1])
    o = call()
  short = torch.tensor([17, 0, 40], dtype=torch.int32, device=DEV)
  store.lengths.copy_(short)  # lengths change between replays
  graph.replay()
  kv_cache.append(store.cache, q[:, :2], q[:, :2], store.slots[:, :1])
  assert torch.equal(o, call()) and not o[1].any()


def test_refusals():
  store = Store([20, 20], d=64)
  cache, table, lengths = store.cache, store.table, store.lengths
  q = torch.zeros(2, 4, 1, 64, device=DEV, dtype=torch.bfloat16)
  k = torch.zeros(2, 2, 1, 64, device=DEV, dtype=torch.bfloat16)
  slots = store.slots[:, :1]
  for bad in (lambda: kv_cache.attend(cache, q[:, :3], table, lengths), lambda: kv_cache.attend(cache, q[..., :32], table, lengths),
              lambda: kv_cache.attend(cache, q[0], table, lengths), lambda: kv_cache.attend(cache, q, table, lengths[:1]),
              lambda: kv_cache.attend(cache, q, table.long(), lengths), lambda: kv_cache.attend(cache, q, table, lengths.long()),
              lambda: kv_cache.attend(cache, q, table.cpu(), lengths), lambda: kv_cache.attend(cache, q.cpu(), table, lengths),
              lambda: kv_cache.attend(cache, q, table, lengths, local_window_size=-1),
              lambda: kv_cache.attend(cache, q, table, lengths, logits_soft_cap=0.0),
              lambda: kv_cache.attend(cache, q, table, lengths, sinks=torch.zeros(3, device=DEV)),
              lambda: kv_cache.append(cache, k, k[..., :32], slots), lambda: kv_cache.append(cache, k, k.float(), slots),
              lambda: kv_cache.append(cache, k, k, slots.float()), lambda: kv_cache.append(cache, k, k, slots[:1]),
              lambda: kv_cache.append(cache, k[:, :1], k[:, :1], slots), lambda: kv_cache.append(cache, k, k, slots.cpu()),
              lambda: kv_cache.read(cache, table, lengths[:1], 20), lambda: kv_cache.read(cache, table, lengths, -1),
              lambda: kv_cache.read(cache, table[0], lengths, 20)):
    with pytest.raises(ValueError):
      bad()
  for bad in (lambda: kv_cache.attend(cache, q.float(), table, lengths), lambda: kv_cache.append(cache, k.double(), k.double(), slots),
              lambda: kv_cache.read(cache, table, lengths, 20, dtype=torch.int32),
              lambda: kv_cache.attend(cache, q.clone().requires_grad_(True), table, lengths),
              lambda: kv_cache.append(cache, k.clone().requires_grad_(True), k, slots)):
    with pytest.raises(NotImplementedError):
      bad()
  with torch.no_grad():
    kv_cache.attend(cache, q.clone().requires_grad_(True), table, lengths)


def test_scales_and_caps_that_are_no_numbers_are_refused():
  """A scale of NaN passed for one of nothing, a cap below the least of 32 bits for none."""
  store = Store([20], d=64)
  q = torch.zeros(1, 2, 1, 64, device=DEV, dtype=torch.bfloat16)
  for kw in (dict(logits_scale=math.nan), dict(logits_soft_cap=1e-50), dict(logits_soft_cap=math.nan), dict(logits_soft_cap=-1.0)):
    with pytest.raises(ValueError):
      kv_cache.attend(store.cache, q, store.table, store.lengths, **kw)


def test_compiled_calls_give_the_same_and_traced_ones_are_refused():
  store = Store([70, 31], d=64)
  q = torch.randn(2, 4, 1, 64, device=DEV, dtype=torch.bfloat16)

  def step(q, k):
    kv_cache.append(store.cache, k, k, store.slots[:, :1])
    return kv_cache.attend(store.cache, q, store.table, store.lengths, logits_scale=0.1) * 2.0

  want = step(q, q[:, :2])
  kv_cache.append(store.cache, store.k[:, :, :1].to(DEV), store.v[:, :, :1].to(DEV), store.slots[:, :1])
  assert torch.equal(torch.compile(step, backend="eager")(q, q[:, :2]), want)
  with pytest.raises(NotImplementedError, match="recorded"):
    torch.jit.trace(step, (q, q[:, :2]), check_trace=False)


# ----------------------------------------------------------------------------------------------
# both ways through attention: every item one CTA's, and shares that a second launch joins
# ----------------------------------------------------------------------------------------------
def _workspace_bytes(store, q_heads, t, table, window=None):
  """What splash_cache_attend asks for on these sizes: 0 where every item is one CTA's."""
  a = _native.SplashCacheAttendArgs()
  c, cache = a.cache, store.cache
  c.k_codes, c.k_scales, c.v_codes, c.v_scales = (x.data_ptr() for x in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales))
  c.n_pages, c.format, c.page_size, c.kv_heads = cache.n_pages, kv_cache.FORMATS[cache.fmt], cache.page_size, cache.kv_heads
  c.group, c.head_dim, c.head_dim_v = cache.group_size or 0, cache.head_dim, cache.head_dim_v
  widths = (C.c_int32 * 2)()
  at = C.addressof(widths)
  _native.lib().splash_cache_row_widths(cache.head_dim, cache.head_dim_v, C.cast(at, C.POINTER(C.c_int32)), C.cast(at + 4, C.POINTER(C.c_int32)))
  c.row_k, c.row_v = widths
  for x, d in ((a.q, cache.head_dim), (a.o, cache.head_dim_v)):
    x.data, x.dtype = cache.k_codes.data_ptr(), 0
    for i, (n, s) in enumerate(zip((len(store.lengths_list), q_heads, t, d), (q_heads * t * d, t * d, d, 1))):
      x.size[i], x.stride[i] = n, s
  a.page_table, a.table_stride, a.n_table, a.lengths = table.data_ptr(), table.shape[1], table.shape[1], store.lengths.data_ptr()
  a.window = -1 if window is None else window
  return _native.lib().splash_cache_attend_workspace_bytes(C.byref(a))


def _table_of(store, shares, q_heads, t, window=None):
  """The store's page table as it is, or wide enough for shares (its sequences are as they were)."""
  table = store.table
  if shares:
    table = torch.full((table.shape[0], 8192 // store.page), -1, dtype=torch.int32, device=DEV)
    table[:, :store.table.shape[1]] = store.table
  assert (_workspace_bytes(store, q_heads, t, table, window) > 0) == shares
  return table


@pytest.mark.parametrize("fmt,group", FORMATS)
@pytest.mark.parametrize("d,d_v", [(64, 64), (128, 128), (192, 128), (256, 256)])
@pytest.mark.parametrize("q_heads,t", [(2, 1), (16, 1), (10, 4)])
@pytest.mark.parametrize("shares", [False, True])
def test_arrays_that_were_never_written(fmt, group, d, d_v, q_heads, t, shares):
  """NaN wherever nothing was written, codes (0x7f and 0xff of e4m3) and scales: behind the ends of sequences, on other pages, and in
  place of tokens that stand before every window."""
  lengths = [1, 50, 77, 0, 700]
  try:
    store = Store(lengths, d=d, d_v=d_v, fmt=fmt, group=group, spare=2, page=64)
  except ValueError:
    assert group in (64, 128)
    return
  for window in (None, 20):
    table = _table_of(store, shares and window is None, q_heads, t, window)  # (a window's items are one CTA's)
    want = _check_attend(store, q_heads=q_heads, t=t, table=table, window=window)
    arrays = (store.cache.k_codes, store.cache.v_codes, store.cache.k_scales.view(torch.int16), store.cache.v_scales.view(torch.int16))
    before = [x.clone() for x in arrays]
    for x in arrays[:2]:
      x.fill_(0x7f)
      x.view(-1)[1::2] = 0xff
    for x in arrays[2:]:
      x.fill_(0x7fff)
    slots = store.slots.clone()
    if window is not None:  # what no query sees was never written either
      for b, n in enumerate(lengths):
        slots[b, :max(n - t - window, 0)] = -1
    kv_cache.append(store.cache, store.k.to(DEV), store.v.to(DEV), slots)
    assert torch.equal(want, _check_attend(store, q_heads=q_heads, t=t, table=table, window=window))
    for x, y in zip(arrays, before):
      x.copy_(y)


@pytest.mark.parametrize("shares", [False, True])
@pytest.mark.parametrize("size", [0, 10, 17, 18, 19, 20])
def test_logits_that_32_bits_hold_to_eight(size, shares):
  """Logits of 63 * 2^size that rise every 64 keys (in units of log2; at 2^26 by 8 now and then).  All keys' values are the same, and so
  is o, whatever the weights that are left."""
  n, d = 4096, 64
  c, q0 = 2.0 ** (size // 2), 2.0 ** (size - size // 2)
  q = torch.full((1, 2, 1, d), q0)
  q[..., 63] = 2.0 ** -4
  for gain in (1.0, 2.0, 4.0, 8.0, 16.0):
    for step in (0.75, 4.0, 7.0):
      def keys(k, step=step):
        k[0, 0] = c
        k[0, 0, :, 63] += torch.arange(n) // 64 * step * math.log(2.0) / q[0, 0, 0, 63]
        return k

      def values(v, gain=gain):
        v[0, 0] = v[0, 0, :1] * gain
        return v

      store = Store([n], heads=1, d=d, group=32, page=64, dtype=torch.float32, keys=keys, values=values)
      window = None if shares else 1000  # (an item is one CTA's where windows are short)
      o = kv_cache.attend(store.cache, q.to(DEV).to(torch.bfloat16), _table_of(store, shares, 2, 1, window), store.lengths, logits_scale=1.0,
                          local_window_size=window)
      want = store.held(0)[1][:, :1]
      # P * scale and the output are rounded; products are up to the group's range
      assert ((o[0].cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -11 * (want.amax() - want.amin())).all(), (gain, step)


@pytest.mark.parametrize("fmt,group", FORMATS)
@pytest.mark.parametrize("q_heads", [2, 16, 20])
@pytest.mark.parametrize("shares", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_huge_values_of_keys_without_weight(fmt, group, q_heads, shares, dtype):
  """Values 2^12 .. 2^40 times the others', at keys that no row, or every second row only, gives any weight: the rows' outputs are held
  as if those keys were not there (what _check_attend allows for is weighted by P)."""
  d, n = 128, 900
  g = torch.Generator().manual_seed(5)  # the queries that _check_attend will take
  q = (torch.randn(1, 1, q_heads, d, generator=g) * 1.5).to(dtype)[0, 0].double()
  none, half = torch.full((q_heads,), -60.0, dtype=torch.float64), torch.full((q_heads,), -60.0, dtype=torch.float64)
  half[::2] = 60.0
  # (position, logits of the rows, size of the values)
  cases = [[(3, none, 30)], [(450, none, 40), (451, none, 12)], [(899, none, 20)], [(5, none + 60, 30), (700, none + 130, 0)]]
  if dtype == torch.bfloat16:
    cases += [[(40, half, 30)], [(640, half, 13), (100, none, 40)]]
  for case in cases:
    def keys(k, case=case):
      for at, logits, _ in case:
        k[0, 0, at] = (torch.linalg.lstsq(q, logits[:, None] * d ** 0.5).solution[:, 0]).float()
      return k

    def values(v, case=case):
      for at, _, size in case:
        v[0, 0, at] *= 2.0 ** size
      return v

    store = Store([n], heads=1, d=d, fmt=fmt, group=group, page=64, keys=keys, values=values)
    _check_attend(store, q_heads=q_heads, dtype=dtype, table=_table_of(store, shares, q_heads, 1))


def test_streams_and_graphs_of_shares():
  """As test_streams_and_graphs, where items are cut into shares: two launches and a workspace."""
  store = Store([5000, 3100, 40], d=128, group=64, page=64)
  assert _workspace_bytes(store, 4, 1, store.table) > 0
  q = torch.randn(3, 4, 1, 128, device=DEV, dtype=torch.bfloat16)
  call = lambda: kv_cache.attend(store.cache, q, store.table, store.lengths, logits_scale=0.1, save_residuals=True)  # noqa: E731
  same = lambda a, b: torch.equal(a[0], b[0]) and all(torch.equal(a[1][x], b[1][x]) for x in a[1])  # noqa: E731
  want = call()
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    outs = [call() for _ in range(20)]
  mine = [call() for _ in range(20)]  # two streams at a time: each call has a workspace of its own
  side.synchronize()
  assert all(same(o, want) for o in outs + mine)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    kv_cache.append(store.cache, q[:, :2], q[:, :2], store.slots[:, :1])
    first = call()
    second = call()  # (in the place of the first one's workspace, maybe)
  for lengths in ([17, 0, 40], [5000, 1, 39], [0, 0, 0], [4999, 3100, 40]):
    store.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))  # lengths change between replays, and with them the shares
    graph.replay()
    kv_cache.append(store.cache, q[:, :2], q[:, :2], store.slots[:, :1])
    want = call()
    assert same(first, want) and same(second, want)
    for b, n in enumerate(lengths):
      assert bool(want[0][b].any()) == (n > 0)


@pytest.mark.parametrize("fmt,group", FORMATS)
@pytest.mark.parametrize("d,d_v", [(64, 64), (96, 96), (192, 128), (256, 256)])
@pytest.mark.parametrize("q_heads,t", [(2, 1), (16, 1), (10, 4)])
def test_f16_outputs_of_shares(fmt, group, d, d_v, q_heads, t):
  try:
    store = Store([33, 2700, 0, 1], d=d, d_v=d_v, fmt=fmt, group=group, page=64, dtype=torch.float16)
  except ValueError:
    assert group in (64, 128)
    return
  _check_attend(store, q_heads=q_heads, t=t, dtype=torch.float16, table=_table_of(store, True, q_heads, t))


@pytest.mark.parametrize("fmt,group", FORMATS)
def test_pages_and_lengths_outside_of_shares(fmt, group):
  """Pages that are none in the middle of long sequences, lengths beyond the table and below zero."""
  store = Store([3000, 640, 1000], d=128, fmt=fmt, group=group, page=16, spare=3)
  table = _table_of(store, True, 4, 3)
  seen = torch.ones(3, 3000, dtype=torch.bool)
  for b, pages in enumerate((range(3, 60), (0, 5, 39), range(0, 63))):
    for i, at in enumerate(pages):
      table[b, at] = (-1, store.cache.n_pages, 2 ** 31 - 1, -5)[i % 4]
      seen[b, at * 16:at * 16 + 16] = False
  seen[1, 640:], seen[2, 1000:] = True, True  # (behind the end: not looked at)
  _check_attend(store, q_heads=4, t=3, seen=seen, table=table)
  q = torch.randn(3, 4, 1, 128, device=DEV, dtype=torch.bfloat16)
  call = lambda lengths, table: kv_cache.attend(store.cache, q, table, lengths, logits_scale=0.1)  # noqa: E731
  short = store.table[:, :128].contiguous()  # 2048 tokens: the first sequence is longer
  assert _workspace_bytes(store, 4, 1, short) > 0
  lengths = torch.tensor([3000, -7, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
  o = call(lengths, short)
  full = call(torch.tensor([2048, 0, 2048], dtype=torch.int32, device=DEV), short)  # (the same shares)
  assert torch.equal(o, full) and not o[1].any() and o[0].any() and o[2].any()


@pytest.mark.parametrize("fmt,group", FORMATS)
def test_what_is_not_seen_has_no_part_in_shares(fmt, group):
  """As test_what_lies_in_places_that_are_not_seen, with NaN in the middle of what a window leaves out of long sequences."""
  store = Store([4100, 3000], d=128, fmt=fmt, group=group, page=64)
  table = _table_of(store, True, 4, 2, 2500)
  call = lambda: _check_attend(store, q_heads=4, t=2, window=2500, table=table)  # noqa: E731
  clean = call()
  bad = torch.full((1, 2, 1, 128), math.nan, device=DEV)
  for at in (5, 1000, 1596):  # query 0 stands at 4098 and sees 1598 ..
    kv_cache.append(store.cache, bad, bad, store.slots[:1, at:at + 1])
  assert torch.equal(clean, call())
  kv_cache.append(store.cache, bad, bad, store.slots[:1, 1598:1599])  # seen by query 0 alone
  o = _attend_of(store, 4, 2, 2500, table)
  assert o[0, :, 0].isnan().all() and not o[0, :, 1].isnan().any() and torch.equal(o[1], clean[1])


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("q_heads", [2, 16, 20])
def test_f16_outputs_of_values_that_cancel(group, q_heads):
  """One key has nearly all the weight, and its values are next to nothing beside a group's zero and products, which cancel."""
  def values(v):
    v[..., ::3] = v[..., ::3] * 1e-3
    return v

  for seed in range(6):
    for lengths in ([1, 2, 3, 22], [40, 7, 300, 5]):
      store = Store(lengths, d=128, fmt="int4", group=group, dtype=torch.float16, seed=seed, values=values)
      _check_attend(store, q_heads=q_heads, dtype=torch.float16, q_scale=4.0, seed=seed)
      _check_attend(store, q_heads=q_heads, t=2, dtype=torch.float16, q_scale=12.0, seed=seed)


@pytest.mark.parametrize("fmt,group", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,batch", [(131072, 300), (1900, 6000)])
def test_errors_do_not_grow_with_the_call(fmt, group, dtype, n, batch):
  """Even rows of many keys, whose outputs are far smaller than the values, in a call so large that a warp adds up thousands of them.
  Rounding P * scale is 0.35e-3 of an output's norm (int4, bf16; codes are 2.7 times the deviation of a group's values), a sum
  of products that loses 2^-25 at each of 64 steps (1024 tokens) some 5e-6 of the values, 0.5e-3 of outputs over 131072 keys: beside the
  1.65e-3 of rounding the output itself (f16: an eighth of all three), half as much again is allowed."""
  store = Store([n], heads=1, d=128, fmt=fmt, group=group, page=256, values=lambda v: v / v.norm(dim=-1, keepdim=True) * 128 ** 0.5)
  g = torch.Generator().manual_seed(3)
  q = torch.randn(1, 4, 1, 128, generator=g).to(dtype)
  k, v = store.held(0)
  p = torch.softmax(k[0] @ q[0, :, 0].double().T * 128 ** -0.5, 0)
  want = p.T @ v[0]
  o = kv_cache.attend(store.cache, q.to(DEV).expand(batch, -1, -1, -1), store.table.expand(batch, -1), store.lengths.repeat(batch),
                      logits_scale=128 ** -0.5)
  error = (o[:, :, 0].cpu().double() - want).norm(dim=(1, 2)).max()
  assert error <= 1.5 * (want.to(dtype).double() - want).norm(), float(error / want.norm())


def _attend_of(store, q_heads, t, window, table):
  g = torch.Generator().manual_seed(5)
  q = (torch.randn(len(store.lengths_list), t, q_heads, store.d, generator=g) * 1.5).to(torch.bfloat16).transpose(1, 2)
  return kv_cache.attend(store.cache, q.to(DEV), table, store.lengths, logits_scale=store.d ** -0.5, local_window_size=window)
