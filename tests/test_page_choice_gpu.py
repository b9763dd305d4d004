"""Bounds of pages, the choice of pages and attention over them: whole numbers against an oracle on the CPU, attention against 64 bits."""
import math

import pytest
import torch

from oracle import kv_cache_ref
from oracle import pages_ref
from test_kv_cache_gpu import ROUNDOFF, Store
from test_page_choice_cpu import TABLES_THAT_DO_NOT_MATCH
from tokamax_b200 import _native
from tokamax_b200 import kv_cache

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FORMATS = [("int4", 32), ("int4", 64), ("int4", 128), ("e4m3", None)]


def _store(*args, **kw):
  try:
    return Store(*args, **kw)
  except ValueError as e:
    assert "group_size" in str(e) and kw["group"] in (64, 128)
    pytest.skip("groups that do not divide the rows")


# ----------------------------------------------------------------------------------------------
# bounds
# ----------------------------------------------------------------------------------------------
def _check_bounds(store, before, bounds, newest, lengths=None, table=None):
  """Pages that the newest tokens made whole have their keys' bounds, all others what they had."""
  table = (store.table if table is None else table).cpu()
  lengths = store.lengths.tolist() if lengths is None else lengths
  k, _ = kv_cache.read(store.cache, store.table, store.lengths, int(store.lengths.max()), dtype=torch.float32)
  k, codes, scales = k.cpu(), *(t.clone() for t in before)
  for b, n in enumerate(lengths):
    n = min(n, table.shape[1] * store.page)
    for j in range(max(n - newest, 0) // store.page, max(n, 0) // store.page):
      page = int(table[b, j])
      if 0 <= page < store.cache.n_pages:
        c, s = pages_ref.bounds(k[b, :, j * store.page:(j + 1) * store.page])
        codes[page, :, :, :store.d], codes[page, :, :, store.d:], scales[page] = c, 0, s
  assert torch.equal(bounds.scales.cpu(), scales) and torch.equal(bounds.codes.cpu(), codes)
  assert torch.equal(bounds.values().cpu(), codes[..., :store.d] * scales[:, :, None, None])  # (one product of 32 bits)


@pytest.mark.parametrize("fmt,group", FORMATS)
@pytest.mark.parametrize("d", [8, 64, 80, 96, 128, 160, 192, 256])
@pytest.mark.parametrize("page", [16, 64])
def test_bounds_of_every_shape(fmt, group, d, page):
  store = _store([0, 15, 16, 17, 200, 128], heads=3, d=d, fmt=fmt, group=group, page=page, spare=1)
  bounds = kv_cache.make_page_bounds(store.cache)
  for newest in (0, 1, 17, 60, 1000):
    bounds.codes.random_(-127, 128)
    bounds.scales.fill_(7.0)
    before = bounds.codes.cpu(), bounds.scales.cpu()
    kv_cache.bound_pages(store.cache, bounds, store.table, store.lengths, newest)
    _check_bounds(store, before, bounds, newest)


def test_bounds_of_large_pages_and_of_many_sequences():
  store = Store([5000, 4096], heads=1, d=128, fmt="e4m3", group=None, page=4096)
  bounds = kv_cache.make_page_bounds(store.cache)
  before = bounds.codes.cpu(), bounds.scales.cpu()
  kv_cache.bound_pages(store.cache, bounds, store.table, store.lengths, 5000)
  _check_bounds(store, before, bounds, 5000)
  store = Store([16, 33], heads=1, d=64)
  bounds = kv_cache.make_page_bounds(store.cache)
  table = store.table.repeat(35000, 1)  # (70000 sequences, of the same pages)
  kv_cache.bound_pages(store.cache, bounds, table, store.lengths.repeat(35000), 40)
  _check_bounds(store, before=tuple(torch.zeros_like(t).cpu() for t in (bounds.codes, bounds.scales)), bounds=bounds, newest=40)


def test_bounds_token_by_token_are_those_of_one_call():
  store = Store([70, 64, 3], heads=2, d=64, page=16)
  once, steps = kv_cache.make_page_bounds(store.cache), kv_cache.make_page_bounds(store.cache)
  kv_cache.bound_pages(store.cache, once, store.table, store.lengths, 70)
  for n in range(1, 71):
    kv_cache.bound_pages(store.cache, steps, store.table, store.lengths.clamp_max(n), 1)
  assert torch.equal(once.codes, steps.codes) and torch.equal(once.scales, steps.scales) and once.codes.any()


@pytest.mark.parametrize("fmt,group", FORMATS)
def test_bounds_of_keys_that_are_no_numbers(fmt, group):
  def spoil(x):
    x[0, 0, 3, 5] = math.nan
    x[0, 0, 20] = 3e38
    x[0, 0, 21] = -3e38
    x[0, 1, :16] = math.inf  # a page of nothing else
    x[0, 1, 16:] = 0.0
    return x

  store = Store([32], heads=2, d=128, fmt=fmt, group=group, page=16, keys=spoil)
  bounds = kv_cache.make_page_bounds(store.cache)
  bounds.scales.fill_(7.0)
  before = bounds.codes.cpu(), bounds.scales.cpu()
  kv_cache.bound_pages(store.cache, bounds, store.table, store.lengths, 32)
  _check_bounds(store, before, bounds, 32)
  page = store.table[0, 0]
  assert float(bounds.scales[page, 1]) == 0 and not bounds.codes[page, 1].any() and bounds.values().isfinite().all()


def test_bounds_pass_over_pages_outside_the_cache_and_lengths_outside_the_table():
  store = Store([70, 64, 100], heads=2, d=64, spare=3)
  table = store.table.clone()
  table[0, 1], table[1, 0], table[2, 2] = -1, store.cache.n_pages, 2 ** 31 - 1
  lengths = torch.tensor([70, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=DEV)
  bounds = kv_cache.make_page_bounds(store.cache)
  before = bounds.codes.cpu(), bounds.scales.cpu()
  kv_cache.bound_pages(store.cache, bounds, table[:, :4].contiguous(), lengths, 2 ** 40)
  _check_bounds(store, before, bounds, 2 ** 40, lengths=lengths.tolist(), table=table[:, :4])


# ----------------------------------------------------------------------------------------------
# the choice
# ----------------------------------------------------------------------------------------------
class Pool:
  """Bounds of a cache that holds nothing else, and the pages of some sequences."""

  def __init__(self, lengths, *, heads=2, d=64, page=16, seed=0, table_pages=None, levels=None):
    g = torch.Generator().manual_seed(seed)
    used = [-(-max(n, 0) // page) for n in lengths]
    self.cache = kv_cache.make_kv_cache(sum(used) + 3, page, heads, d, fmt="int4", device=DEV)
    self.bounds = kv_cache.make_page_bounds(self.cache)
    centre = torch.randn(sum(used) + 3, heads, 1, d, generator=g) * 2
    half = torch.rand(sum(used) + 3, heads, 1, d, generator=g) * torch.tensor([-1.0, 1.0])[:, None]
    if levels is not None:  # few different pages
      pick = torch.arange(sum(used) + 3) % levels
      centre, half = centre[pick], half[pick]
    codes, scales = pages_ref.bounds((centre + half))
    self.codes, self.scales = codes, scales
    self.bounds.codes[..., :d] = codes.to(DEV)
    self.bounds.scales.copy_(scales)
    order = torch.randperm(sum(used) + 3, generator=g).int()
    self.table = torch.full((len(lengths), table_pages or max(max(used), 1)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(used):
      self.table[b, :n] = order[at:at + n]
      at += n
    self.lengths, self.page, self.d, self.heads = lengths, page, d, heads

  def q(self, group, t, dtype=torch.bfloat16, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(len(self.lengths), t, self.heads * group, self.d, generator=g).to(dtype).transpose(1, 2)

  def check(self, q, count, first=1, last=1):
    lengths = torch.tensor(self.lengths, dtype=torch.int32, device=DEV)
    got = kv_cache.choose_pages(self.cache, self.bounds, q.to(DEV), self.table.to(DEV), lengths, count, first=first, last=last)
    want = pages_ref.choose(q, self.codes, self.scales, self.table, self.lengths, self.cache.n_pages, self.page, count, first, last)
    assert got[0].dtype == got[1].dtype == torch.int32
    assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[0].cpu(), want[0])
    return got


@pytest.mark.parametrize("d", [8, 64, 80, 96, 128, 160, 192, 256])
@pytest.mark.parametrize("group,t", [(1, 1), (4, 1), (8, 2), (9, 1), (20, 3)])
def test_choices_of_every_shape(d, group, t):
  pool = Pool([0, 1, 15, 16, 17, 333, 640], d=d)
  for dtype, count, first, last in ((torch.bfloat16, 5, 1, 1), (torch.float16, 12, 0, 3), (torch.bfloat16, 64, 2, 2)):
    pool.check(pool.q(group, t, dtype), count, first, last)


@pytest.mark.parametrize("lengths,heads", [([2000], 1), ([5000, 3], 2), ([16 * 2047 + 5], 3), ([777, 1300, 4000, 90] * 6, 2)])
def test_choices_of_long_sequences(lengths, heads):
  """Several CTAs a query and one, more pages than a CTA has threads."""
  pool = Pool(lengths, heads=heads)
  pool.check(pool.q(4, 1), 64, 1, 2)
  pool.check(pool.q(2, 1, seed=2), 7, 0, 1)


@pytest.mark.parametrize("levels", [1, 2, 5])
def test_of_equal_scores_the_first_are_taken(levels):
  pool = Pool([1500, 40, 321], levels=levels)
  for count in (2, 10, 50):
    pool.check(pool.q(3, 2), count, 1, 1)
    pool.check(pool.q(3, 2), count, 0, 2)


def test_queries_of_zeros_and_scores_below_zero():
  pool = Pool([700, 64])
  pool.check(torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16), 9)  # all scores 0, of both signs
  pool.codes.copy_(-pool.codes.abs() - 1)
  pool.codes.clamp_(-127, 127)
  pool.bounds.codes[..., :64] = pool.codes.to(DEV)
  pool.check(pool.q(2, 1).abs() + 1, 9)
  pool.scales[::3] = 0.0
  pool.bounds.scales.copy_(pool.scales)
  pool.check(pool.q(2, 1).abs() + 1, 9)


def test_queries_and_bounds_of_every_size():
  pool = Pool([700, 64])
  g = torch.Generator().manual_seed(3)
  pool.scales *= torch.exp2(torch.randint(-140, 120, pool.scales.shape, generator=g).float())  # subnormals among them, and overflow
  pool.bounds.scales.copy_(pool.scales)
  q = pool.q(2, 3)
  q[0, 0, 0, 3], q[0, 1, 1, 7], q[1, 2, 2, 0] = math.inf, math.nan, -math.inf
  q[0, 2, 1] = 1e-39
  q[0, 3, 1] = 0.0
  pool.check(q, 9)
  pool.check(q, 20, 0, 1)


def test_bounds_that_nobody_wrote_choose_some_pages():
  """Whatever lies in the scales, NaN too: as many pages as asked for, of the sequence."""
  pool = Pool([900, 31])
  pool.bounds.scales.view(torch.int32).random_(-2 ** 31, 2 ** 31 - 1)
  pool.bounds.scales.view(torch.int32)[::2] = 0x7fffffff
  pool.bounds.scales.view(torch.int32)[1::4] = -1
  tables, lengths = kv_cache.choose_pages(pool.cache, pool.bounds, pool.q(2, 1).to(DEV), pool.table.to(DEV),
                                          torch.tensor(pool.lengths, dtype=torch.int32, device=DEV), 10)
  for h in range(2):
    taken = tables[0, h, 0].tolist()
    assert len(set(taken)) == 10 and set(taken) <= set(pool.table[0].tolist()) and int(lengths[0, h, 0]) == 9 * 16 + 900 % 16


def test_pages_outside_the_cache_are_not_chosen():
  pool = Pool([700, 64, 90], table_pages=60)
  pool.table[0, 1], pool.table[0, 20], pool.table[1, 0], pool.table[2, 5] = -1, pool.cache.n_pages, 2 ** 31 - 1, -2 ** 31  # (the last: a query's own)
  for count in (4, 30, 100):
    pool.check(pool.q(2, 3), count, 2, 2)
  pool.table[1] = -1  # none at all
  pool.check(pool.q(2, 3), 6, 2, 2)


def test_lengths_beyond_the_table_and_below_zero():
  pool = Pool([640, 300, 300])
  pool.lengths = [2 ** 31 - 1, -2 ** 31, -1]
  pool.check(pool.q(2, 2), 6)
  pool.lengths = [641, 2, 0]
  pool.check(pool.q(2, 5), 6)


@pytest.mark.parametrize("n_table", [32768, 32769, 70000])
def test_wide_tables(n_table):
  """Scores on the chip and, for more pages, in a workspace."""
  pool = Pool([16 * 300 + 4, 77], heads=1, table_pages=n_table)
  small = pool.check(pool.q(2, 2), 40)
  long_one = torch.arange(n_table, dtype=torch.int32) % pool.cache.n_pages
  lengths = torch.tensor([n_table * 16 - 3], dtype=torch.int32, device=DEV)
  q = pool.q(2, 1)[:1].to(DEV)
  tables, tokens = kv_cache.choose_pages(pool.cache, pool.bounds, q, long_one[None].to(DEV), lengths, 500)
  score = pages_ref.scores(q[0, :, 0].cpu(), pool.codes[long_one.long(), 0], pool.scales[long_one.long(), 0])
  score[0] = score[-1] = math.inf
  taken = torch.sort(torch.sort(score, descending=True, stable=True).indices[:500]).values
  assert torch.equal(tables[0, 0, 0].cpu(), long_one[taken]) and int(tokens) == 500 * 16 - 3
  assert small[0].shape == (2, 1, 2, 40)


@pytest.mark.parametrize("d,group", [(64, 2), (80, 9), (128, 4), (160, 5), (256, 2), (256, 128)])
@pytest.mark.parametrize("n_table", [1024, 1025, 8191, 8192, 8193, 20000])
def test_tables_on_both_sides_of_each_limit_in_every_width(n_table, d, group):
  """Four warps a CTA up to 1024 pages, eight above; scores on the chip up to 8192, in a workspace above; a cluster a row where rows are
  few, a CTA where they are many.  128 q heads of 256 channels and 8192 pages are the most shared memory that a CTA asks for."""
  pool = Pool([16 * 300 + 4], heads=1, d=d, seed=n_table)
  table = torch.arange(n_table, dtype=torch.int32) * 7 % pool.cache.n_pages
  q, count = pool.q(group, 1)[:1].to(DEV), 500
  score = pages_ref.scores(q[0, :, 0].cpu(), pool.codes[table.long(), 0], pool.scales[table.long(), 0])
  for pages in (n_table, n_table - 333):
    order = score[:pages].clone()
    order[0] = order[-1] = math.inf
    taken = torch.sort(torch.sort(order, descending=True, stable=True).indices[:count]).values
    for rows in (1, 300):  # (sequences of the same pages)
      lengths = torch.full((rows,), pages * 16 - 3, dtype=torch.int32, device=DEV)
      tables, tokens = kv_cache.choose_pages(pool.cache, pool.bounds, q.expand(rows, -1, -1, -1), table[None].expand(rows, -1).to(DEV), lengths, count)
      assert torch.equal(tables.cpu(), table[taken].expand(rows, 1, 1, -1)) and (tokens == count * 16 - 3).all()


def test_drafted_tokens_choose_as_they_would_one_by_one():
  pool = Pool([1000, 37, 64])
  q = pool.q(4, 5).to(DEV)
  lengths = torch.tensor(pool.lengths, dtype=torch.int32, device=DEV)
  table = pool.table.to(DEV)
  tables, tokens = kv_cache.choose_pages(pool.cache, pool.bounds, q, table, lengths, 8)
  for i in range(5):
    one = kv_cache.choose_pages(pool.cache, pool.bounds, q[:, :, i:i + 1], table, lengths - (4 - i), 8)
    assert torch.equal(one[0][:, :, 0], tables[:, :, i]) and torch.equal(one[1][:, :, 0], tokens[:, :, i])


def test_more_sequences_than_a_grid_has_rows():
  """70000 queries, of two sequences."""
  pool = Pool([640, 100], heads=1)
  q = pool.q(2, 1).to(DEV)
  lengths = torch.tensor(pool.lengths, dtype=torch.int32, device=DEV)
  want = kv_cache.choose_pages(pool.cache, pool.bounds, q, pool.table.to(DEV), lengths, 8)
  got = kv_cache.choose_pages(pool.cache, pool.bounds, q.repeat(35000, 1, 1, 1), pool.table.to(DEV).repeat(35000, 1), lengths.repeat(35000), 8)
  assert torch.equal(got[0], want[0].repeat(35000, 1, 1, 1)) and torch.equal(got[1], want[1].repeat(35000, 1, 1))


def test_operands_through_their_strides_and_nothing_at_all():
  pool = Pool([640, 100])
  lengths, table = torch.tensor(pool.lengths, dtype=torch.int32, device=DEV), pool.table.to(DEV)
  call = lambda q, t=table: kv_cache.choose_pages(pool.cache, pool.bounds, q, t, lengths, 8)  # noqa: E731
  q = pool.q(2, 3).to(DEV)
  want = call(q.contiguous())
  odd = torch.zeros(2, 4, 3, 67, device=DEV, dtype=torch.bfloat16)[..., 3:]
  odd.copy_(q)
  wide = torch.zeros(2, 2 * table.shape[1], dtype=torch.int32, device=DEV)[:, ::2]
  wide.copy_(table)
  for got in (call(q), call(odd), call(q, wide)):
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
  tables, tokens = call(q[:, :, :0])
  assert tables.shape == (2, 2, 0, 8) and tokens.shape == (2, 2, 0)
  tables, tokens = kv_cache.choose_pages(pool.cache, pool.bounds, q[:0], table[:0], lengths[:0], 8)
  assert tables.shape == (0, 2, 3, 8)
  kv_cache.bound_pages(pool.cache, pool.bounds, table[:0], lengths[:0], 8)


# ----------------------------------------------------------------------------------------------
# attention over tables of chosen pages
# ----------------------------------------------------------------------------------------------
def _check_attend(store, tables, tokens, *, q_heads, t=1, soft_cap=None, sinks=None, dtype=torch.bfloat16, seed=5):
  """The tolerances of tests/test_kv_cache_gpu.py, which derives them."""
  g = torch.Generator().manual_seed(seed)
  scale, group = store.d ** -0.5, q_heads // store.heads
  q = (torch.randn(len(store.lengths_list), t, q_heads, store.d, generator=g) * 1.5).to(dtype).transpose(1, 2)
  o, res = kv_cache.attend(store.cache, q.to(DEV), tables.to(DEV), tokens.to(DEV), logits_scale=scale, logits_soft_cap=soft_cap,
                           sinks=None if sinks is None else sinks.to(DEV), save_residuals=True)
  assert o.dtype == dtype and o.shape == (*q.shape[:3], store.d_v)
  where = {int(page): (b, j) for b, row in enumerate(store.table.tolist()) for j, page in enumerate(row) if page >= 0}
  for b in range(tables.shape[0]):
    for h in range(store.heads):
      for i in range(t):
        n = min(max(int(tokens[b, h, i]), 0), tables.shape[3] * store.page)
        k, v, moved = [], [], []
        for at in range(n):
          page = int(tables[b, h, i, at // store.page])
          if page not in where:
            continue
          s, j = where[page]
          for to, held in zip((k, v, moved), _held(store, s)):
            to.append(held[h, j * store.page + at % store.page])
        stack = lambda x, d: torch.stack(x)[None] if x else torch.zeros(1, 0, d, dtype=torch.float64)  # noqa: E731
        k, v, moved = stack(k, store.d), stack(v, store.d_v), stack(moved, store.d_v)
        heads = slice(h * group, (h + 1) * group)
        rows = q[b, heads, i:i + 1].double()
        ref, lse, top, size, moved = kv_cache_ref.attend(rows, k, v, scale=scale, soft_cap=soft_cap, sinks=None if sinks is None else sinks[heads], weights=moved)
        logits = (rows.norm(dim=-1).max() * (k.norm(dim=-1).max() if k.shape[1] else 0.0) * scale).clamp_min(1.0)
        slack = 2.0 ** -18 * logits
        got = o[b, heads, i:i + 1].cpu().double()
        before = ((ROUNDOFF[torch.float16] if dtype == torch.bfloat16 else 2.0 ** -22) + 2.0 ** -18) * moved + 2 * slack * size + 1e-9
        bound = before + ROUNDOFF[dtype] * (ref.abs() + before) + (2.0 ** -25 if dtype == torch.float16 else 0.0)
        assert ((got - ref).abs() <= bound).all(), (b, h, i, n, float(((got - ref).abs() / bound).max()))
        for name, want in (("logsumexp", lse), ("max_logits", top)):
          x, dead = res[name][b, heads, i:i + 1].cpu().double(), want == kv_cache_ref.MASK_VALUE
          assert (x[dead] <= -2e38).all() and not got[dead].any()
          assert ((x - want).abs()[~dead] <= slack + 2.0 ** -20 * (1 + want.abs()[~dead])).all()
  return o


def _held(store, b):
  """Keys, values and what of the values is not the zero of a group, of sequence b, worked out once; zeros where a page was never written."""
  if not hasattr(store, "held_rows"):
    store.held_rows = {}
  if b not in store.held_rows:
    n = store.lengths_list[b]
    held = (*store.held(b), kv_cache_ref.products(store.v[b, :, :n], store.fmt, store.group))
    store.held_rows[b] = tuple(torch.nn.functional.pad(x, (0, 0, 0, -n % store.page)) for x in held)
  return store.held_rows[b]


def _random_tables(store, t, count, seed=0):
  """Some pages of a sequence for each kv head and query, in order, its own the last."""
  g = torch.Generator().manual_seed(seed)
  table = store.table.cpu()
  tables = torch.full((len(store.lengths_list), store.heads, t, count), -1, dtype=torch.int32)
  tokens = torch.zeros(tables.shape[:3], dtype=torch.int32)
  for b, n in enumerate(store.lengths_list):
    for h in range(store.heads):
      for i in range(t):
        position = n - t + i
        if position < 0:
          continue
        own = position // store.page
        taken = torch.sort(torch.randperm(own, generator=g)[:count - 1]).values.tolist() + [own]
        tables[b, h, i, :len(taken)] = table[b, taken]
        tokens[b, h, i] = (len(taken) - 1) * store.page + position % store.page + 1
  return tables, tokens


@pytest.mark.parametrize("fmt,group", FORMATS)
@pytest.mark.parametrize("d,d_v", [(64, 64), (80, 80), (96, 96), (128, 128), (128, 64), (192, 128), (256, 256), (8, 8)])
@pytest.mark.parametrize("q_heads,t", [(3, 1), (12, 2), (27, 1), (75, 1)])
def test_attention_over_tables_of_every_shape(fmt, group, d, d_v, q_heads, t):
  store = _store([0, 1, 17, 300], heads=3, d=d, d_v=d_v, fmt=fmt, group=group, page=16)
  tables, tokens = _random_tables(store, t, 6)
  _check_attend(store, tables, tokens, q_heads=q_heads, t=t)


@pytest.mark.parametrize("fmt,group", [("int4", 64), ("e4m3", None)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_items_cut_into_shares(fmt, group, dtype):
  """Tables of more tokens than one CTA takes, joined by a second launch; caps and sinks."""
  store = Store([3000, 5, 2100], heads=2, d=64, fmt=fmt, group=group, page=64, dtype=dtype)
  tables, tokens = _random_tables(store, 2, 40)
  sinks = torch.tensor([0.5, -1.0, 3.0, 0.0])
  first = _check_attend(store, tables, tokens, q_heads=4, t=2, dtype=dtype)
  again = _check_attend(store, tables, tokens, q_heads=4, t=2, dtype=dtype)
  assert torch.equal(first, again)
  _check_attend(store, tables, tokens, q_heads=4, t=2, soft_cap=20.0, sinks=sinks, dtype=dtype)


@pytest.mark.parametrize("fmt,group", [("int4", 128), ("e4m3", None)])
@pytest.mark.parametrize("batch,t,pages", [(1, 1, 20), (1, 1, 70), (1, 2, 700), (10, 1, 40), (10, 4, 40), (20, 8, 20), (50, 7, 12)])
def test_items_of_clusters_of_every_size(fmt, group, batch, t, pages):
  """Few items and many, tables with room for few tokens and many more than there are: a CTA an item, clusters of two to eight, and
  shares.  Lengths from nothing to the whole table."""
  store = Store([(37 * b * b + 1) % 300 for b in range(batch - 1)] + [640], heads=2, d=128, fmt=fmt, group=group, page=16)
  tables, tokens = _random_tables(store, t, min(pages, 40))
  tables = torch.nn.functional.pad(tables, (0, pages - min(pages, 40)), value=-1)
  first = _check_attend(store, tables, tokens, q_heads=6, t=t)
  assert torch.equal(first, _check_attend(store, tables, tokens, q_heads=6, t=t))


def test_more_tables_than_a_cta_has_threads():
  store = Store([3 * i for i in range(70)], heads=3, d=64, page=16)
  tables, tokens = _random_tables(store, 1, 200)  # (3200 tokens of room: shares)
  _check_attend(store, tables, tokens, q_heads=6)
  _check_attend(store, tables[..., :8], tokens.clamp_max(8 * 16), q_heads=6)


def test_tables_with_pages_outside_the_cache_lengths_outside_the_table_and_the_same_page_twice():
  for pages in (5, 100):
    store = Store([200, 90], heads=2, d=64, page=16)
    tables, tokens = _random_tables(store, 2, 5)
    tables = torch.nn.functional.pad(tables, (0, pages - 5), value=-1)
    tables[0, 0, 0, 1], tables[0, 1, 1, 0], tables[1, 0, 0, 2] = -1, store.cache.n_pages, 2 ** 31 - 1
    tables[1, 1, 1, 1] = tables[1, 1, 1, 0]
    tokens[0, 0, 1], tokens[1, 0, 1] = 2 ** 31 - 1, -5
    tokens[1, 1, 0] = 0
    _check_attend(store, tables, tokens, q_heads=4, t=2)


def test_tables_through_their_strides_and_nothing_at_all():
  store = Store([200, 90], heads=2, d=64, page=16)
  tables, tokens = (x.to(DEV) for x in _random_tables(store, 2, 5))
  q = torch.randn(2, 4, 2, 64, device=DEV, dtype=torch.bfloat16)
  call = lambda *a: kv_cache.attend(store.cache, *a, logits_scale=0.1)  # noqa: E731
  want = call(q, tables, tokens)
  wide = torch.full((2, 2, 2, 11), -1, dtype=torch.int32, device=DEV)
  wide[..., :10:2] = tables
  turned = tables.permute(3, 2, 1, 0).contiguous().permute(3, 2, 1, 0)
  for t in (wide[..., :10:2], turned, wide[..., :10:2].contiguous()):
    assert torch.equal(call(q, t, tokens), want)
  assert torch.equal(call(q, tables, tokens.permute(2, 1, 0).contiguous().permute(2, 1, 0)), want)
  one = tables[:, :1, :1].expand(-1, 2, 2, -1)  # a table for all of a sequence
  assert torch.equal(call(q, one, tokens), call(q, one.contiguous(), tokens))
  assert call(q[:, :, :0], tables[:, :, :0], tokens[:, :, :0]).shape == (2, 4, 0, 64)
  assert call(q[:0], tables[:0], tokens[:0]).shape == (0, 4, 2, 64)


def test_outputs_lie_as_the_queries_do():
  store = Store([200, 90], heads=2, d=64, page=16)
  tables, tokens = (x.to(DEV) for x in _random_tables(store, 3, 5))
  q = torch.randn(2, 3, 8, 64, device=DEV, dtype=torch.bfloat16)[:, :, :4].transpose(1, 2)  # a part of a projection
  for pages in ((tables, tokens), (store.table, store.lengths)):
    out = kv_cache.attend(store.cache, q, *pages, logits_scale=0.1)
    assert out.stride() == torch.empty_like(q).stride() and out.transpose(1, 2).is_contiguous()
    assert torch.equal(out, kv_cache.attend(store.cache, q.contiguous(), *pages, logits_scale=0.1))


@pytest.mark.parametrize("fmt,group", FORMATS)
def test_a_choice_of_all_pages_is_attention_over_the_whole(fmt, group):
  """The same keys in the same order: bf16 outputs differ by roundings of sums of 32 bits at most, a step of bf16 where one is beside a tie."""
  store = Store([0, 1, 300, 640, 77], heads=2, d=128, fmt=fmt, group=group, page=16)
  bounds = kv_cache.make_page_bounds(store.cache)
  kv_cache.bound_pages(store.cache, bounds, store.table, store.lengths, 640)
  q = torch.randn(5, 8, 3, 128, device=DEV, dtype=torch.bfloat16)
  tables, tokens = kv_cache.choose_pages(store.cache, bounds, q, store.table, store.lengths, 40)
  got = kv_cache.attend(store.cache, q, tables, tokens, logits_scale=0.1)
  want = kv_cache.attend(store.cache, q, store.table, store.lengths, logits_scale=0.1)
  # rounding of P * scale to f16 (2^-11 of each term) against other maxima, then a bf16 step: sizes of values are 2^4 of an output's at most
  assert ((got.float() - want.float()).abs() <= 2.0 ** -7 * want.float().abs() + 2.0 ** -7 * want.float().abs().max()).all()
  positions = store.lengths[:, None] - 3 + torch.arange(3, device=DEV)[None, :] + 1
  assert torch.equal(tokens, positions.clamp_min(0)[:, None].expand(-1, 2, -1))


# ----------------------------------------------------------------------------------------------
# together, and where it runs
# ----------------------------------------------------------------------------------------------
def test_streams_and_graphs():
  """A step of bounds, choice and attention, captured; lengths, pages and queries change between the replays."""
  store = Store([700, 300, 64], heads=2, d=64, page=16)
  bounds = kv_cache.make_page_bounds(store.cache)
  kv_cache.bound_pages(store.cache, bounds, store.table, store.lengths, 700)
  q, lengths, table = torch.randn(3, 4, 1, 64, device=DEV, dtype=torch.bfloat16), store.lengths.clone(), store.table.clone()

  def step():
    kv_cache.bound_pages(store.cache, bounds, table, lengths, 1)
    tables, tokens = kv_cache.choose_pages(store.cache, bounds, q, table, lengths, 8)
    return tables, tokens, kv_cache.attend(store.cache, q, tables, tokens, logits_scale=0.1)

  want = step()
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    got = step()
  torch.cuda.current_stream().wait_stream(side)
  assert all(torch.equal(a, b) for a, b in zip(got, want))
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    got = step()
  for n in (0, 1, 100, 250):
    lengths.copy_((store.lengths - n).clamp_min(0))
    q.add_(0.25)
    table.copy_(store.table.flip(0) if n == 250 else store.table)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_two_graphs_with_workspaces_side_by_side():
  """Wide tables and cut items: each capture has a workspace of its own."""
  stores = [Store([3000, 2500], heads=1, d=64, page=16, seed=s) for s in (0, 1)]
  calls = []
  for n, store in enumerate(stores):
    bounds = kv_cache.make_page_bounds(store.cache)
    kv_cache.bound_pages(store.cache, bounds, store.table, store.lengths, 3000)
    wide = torch.full((2, 33000), -1, dtype=torch.int32, device=DEV)
    wide[:, :store.table.shape[1]] = store.table
    q = torch.randn(2, 4, 1, 64, device=DEV, dtype=torch.bfloat16)

    def call(store=store, bounds=bounds, wide=wide, q=q):
      tables, tokens = kv_cache.choose_pages(store.cache, bounds, q, wide, store.lengths, 150)
      return kv_cache.attend(store.cache, q, tables, tokens, logits_scale=0.1)

    calls.append(call)
  want = [call() for call in calls]
  graphs, got = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], [None, None]
  for n in (0, 1):
    with torch.cuda.graph(graphs[n]):
      got[n] = calls[n]()
  streams = [torch.cuda.Stream(), torch.cuda.Stream()]
  for n in (0, 1):
    streams[n].wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(streams[n]):
      for _ in range(5):
        graphs[n].replay()
  torch.cuda.synchronize()
  assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_compiled_calls_give_the_same_and_transforms_are_refused():
  store = Store([700, 300], heads=2, d=64, page=16)
  bounds, q = kv_cache.make_page_bounds(store.cache), torch.randn(2, 4, 1, 64, device=DEV, dtype=torch.bfloat16)

  def step(q):
    kv_cache.bound_pages(store.cache, bounds, store.table, store.lengths, 700)
    return kv_cache.attend(store.cache, q, *kv_cache.choose_pages(store.cache, bounds, q, store.table, store.lengths, 8), logits_scale=0.1) * 2.0

  assert torch.equal(torch.compile(step, backend="eager")(q), step(q))
  choose = lambda x: kv_cache.choose_pages(store.cache, bounds, x, store.table, store.lengths, 8)  # noqa: E731
  for transform in (lambda: torch.func.vmap(choose)(q[None]), lambda: torch.func.grad(lambda x: step(x).sum())(q)):
    with pytest.raises((RuntimeError, NotImplementedError)):
      transform()


def test_refusals():
  store = Store([20], heads=2, d=64)
  bounds, other = kv_cache.make_page_bounds(store.cache), kv_cache.make_page_bounds(Store([20, 20], heads=2, d=64).cache)
  q = torch.zeros(1, 4, 1, 64, device=DEV, dtype=torch.bfloat16)
  with pytest.raises(ValueError, match="not of a cache"):
    kv_cache.bound_pages(store.cache, other, store.table, store.lengths, 1)
  with pytest.raises(ValueError, match="not of a cache"):
    kv_cache.choose_pages(store.cache, other, q, store.table, store.lengths, 4)
  with pytest.raises(ValueError, match="on cpu"):
    kv_cache.choose_pages(store.cache, bounds, q.cpu(), store.table, store.lengths, 4)
  with pytest.raises(ValueError, match="on cpu"):
    kv_cache.choose_pages(store.cache, bounds, q, store.table.cpu(), store.lengths, 4)
  with pytest.raises(ValueError, match="newest"):
    kv_cache.bound_pages(store.cache, bounds, store.table, store.lengths, -1)
  with pytest.raises(NotImplementedError, match="not built"):
    kv_cache.choose_pages(store.cache, bounds, q.float(), store.table, store.lengths, 4)
  with pytest.raises(_native.SplashError, match="-7"):
    kv_cache.choose_pages(store.cache, bounds, q.expand(-1, 4, -1, -1).repeat(1, 65, 1, 1), store.table, store.lengths, 4)
  with pytest.raises(ValueError, match="count"):
    kv_cache.choose_pages(store.cache, bounds, q, store.table, store.lengths, 1)


@pytest.mark.parametrize("table,lengths,window,message", TABLES_THAT_DO_NOT_MATCH)
def test_what_tables_are_refused_for(table, lengths, window, message):
  """The kernel takes the extents of tables and lengths from q and the cache: what does not match them is not looked at."""
  cache = kv_cache.make_kv_cache(5, 16, 2, 64, device=DEV)
  with pytest.raises(ValueError, match=message):
    kv_cache.attend(cache, torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(table, dtype=torch.int32, device=DEV),
                    torch.ones(lengths, dtype=torch.int32, device=DEV), local_window_size=window)


@pytest.mark.parametrize("kw", [dict(count=0), dict(count=1), dict(count=2, first=2), dict(first=-1), dict(last=0), dict(count=1 << 32),
                                dict(last=1 << 33, count=1 << 34)])
def test_counts_that_are_refused(kw):
  cache = kv_cache.make_kv_cache(5, 16, 2, 64, device=DEV)
  i = torch.ones(1, dtype=torch.int32, device=DEV)
  with pytest.raises(ValueError, match="expected first >= 0, last >= 1 and count >= first"):
    kv_cache.choose_pages(cache, kv_cache.make_page_bounds(cache), torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16, device=DEV), i[:, None], i,
                          **dict(dict(count=3), **kw))
  with pytest.raises(ValueError, match="q of 2 sequences, lengths of 1"):
    kv_cache.choose_pages(cache, kv_cache.make_page_bounds(cache), torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16, device=DEV), i[:, None], i, 3)
