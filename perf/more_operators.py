"""Timing cases of rotary positions, and of attention over the pages of a cache that a cheap score chooses.

A case is a dict of plain values.  ``kind`` says which operators it goes through:

  rotate  ``rotary.rotate`` of queries and keys; with ``train`` its gradients too
  bound   ``kv_cache.bound_pages``: the channels' least and largest keys of each whole page, in 8 bits
  choose  ``kv_cache.choose_pages``: for each kv head and query the pages whose bounds allow the largest logits
  attend  ``kv_cache.attend`` over tables of chosen pages
  step    choose and attend, as a layer's decoding step does

The cache is one of 4 or 8 bits: ``fmt`` int4 (a bf16 zero and scale for ``group`` channels) or e4m3 (a bf16 scale for a row),
in pages of ``page`` tokens that lie anywhere in a pool.
"""

import math
import random

import numpy as np
import torch

own = False

_WIDTHS = ((64, 64), (96, 96), (128, 128), (192, 128), (192, 192), (256, 256))  # rows are padded to one of these

_ROTATE = dict(kind="rotate", batch=1, t=1, q_heads=32, kv_heads=8, d=128, dim=128, interleaved=False, base=10000.0, scaling="none",
               far=0, heads_first=False, train=False, dtype="bfloat16")
_PAGES = dict(kind="choose", fmt="int4", group=64, page=64, batch=1, least=1, most=1024, t=1, newest=1, count=16, first=1, last=1,
              q_heads=32, kv_heads=8, d=128, d_v=0, soft_cap=0.0, sinks=False, dtype="bfloat16")


def _case(**kw):
  c = dict(_ROTATE if kw["kind"] == "rotate" else _PAGES, **kw)
  if "d_v" in c:
    c["d_v"] = c["d_v"] or c["d"]
  return c


def listed():
  return [
      # A decoding step of eight chats in a small model, far into their contexts: all launch and latency.
      _case(kind="rotate", name="rotate_token", batch=8, q_heads=8, kv_heads=2, d=64, dim=64, far=100000),
      # Prompts of 4096 tokens for the cache, queries and keys as the projections leave them, frequencies scaled for long contexts.
      _case(kind="rotate", name="rotate_prompts", batch=4, t=4096, base=500000.0, scaling="bands"),
      # A training step's share of one layer: 2 x 8192 tokens, forward and gradients. The largest of its kind.
      _case(kind="rotate", name="rotate_train", batch=2, t=8192, train=True, heads_first=True),
      # Everything odd: 517 tokens, 32 of 80 channels, neighbours as pairs, f16, gradients.
      _case(kind="rotate", name="rotate_part", batch=3, t=517, q_heads=12, kv_heads=4, d=80, dim=32, interleaved=True, far=30000,
            scaling="by_parts", train=True, dtype="float16"),
      # Four prompts of up to 8192 tokens have gone into the cache: all their whole pages.
      _case(kind="bound", name="bound_prompts", batch=4, least=2048, most=8192, newest=8192),
      # A chunk of 517 tokens behind what earlier chunks left; eight bits, head dim 80.
      _case(kind="bound", name="bound_chunk_e4m3", fmt="e4m3", page=32, batch=3, least=1999, most=6001, newest=517, kv_heads=4, d=80),
      # One very long document: 2048 pages, of which each kv head takes 64.
      _case(kind="choose", name="choose_long", least=131072, most=131072, count=64, last=2),
      # A full server: long contexts in every slot.
      _case(kind="choose", name="choose_server", batch=32, least=8192, most=32768, count=64, last=2),
      # One token of a short sequence in a small model goes over eight pages of sixteen tokens.
      _case(kind="attend", name="attend_one", group=32, page=16, least=777, most=777, count=8, q_heads=8, kv_heads=2, d=64),
      # The server's attention over its 64 pages: the largest.
      _case(kind="attend", name="attend_server", batch=32, least=8192, most=32768, count=64),
      # Five drafted tokens of each sequence, each with pages of its own; eight bits, sinks, head dim 80, f16; some are short.
      _case(kind="attend", name="attend_drafts_e4m3", fmt="e4m3", page=32, batch=12, least=5, most=9000, t=5, count=48, q_heads=20,
            kv_heads=4, d=80, sinks=True, dtype="float16"),
      # Choose and attend: the decoding step of a batch of long chats.
      _case(kind="step", name="step_batch", batch=16, least=4000, most=60000, count=48, first=1, last=2),
  ]


# ----------------------------------------------------------------------------------------------
# drawing more cases of the same ranges
# ----------------------------------------------------------------------------------------------
def _len(rng, lo, hi):
  """An odd number between lo and hi, even over the logarithm."""
  return int(math.exp(rng.uniform(math.log(lo), math.log(hi)))) | 1


def draw(rng: random.Random):
  largest = {}
  for c in listed():
    w = work(c)
    most = largest.setdefault(c["kind"], {"bytes": 0.0, "flops": 0.0})
    for key in most:
      most[key] = max(most[key], w[key])
  while True:
    kind = rng.choice(["rotate", "rotate", "bound", "choose", "attend", "attend", "step"])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 8, 16])
    heads = dict(kv_heads=kv_heads, q_heads=kv_heads * rng.choice([1, 2, 4, 4, 5, 8]), dtype=rng.choice(["bfloat16", "bfloat16", "float16"]))
    batch = max(1, round(math.exp(rng.uniform(0.0, math.log(32)))))
    if kind == "rotate":
      d = rng.choice([64, 80, 96, 128, 128, 192, 256])
      c = _case(kind=kind, **heads, batch=batch, t=rng.choice([1, _len(rng, 1, 8192), _len(rng, 64, 8192)]), d=d,
                dim=rng.choice([d, d, d // 2, 32]), interleaved=rng.random() < 0.4, far=rng.choice([0, 1000, 1000000]),
                base=rng.choice([10000.0, 500000.0]), scaling=rng.choice(["none", "linear", "base", "by_parts", "bands"]),
                heads_first=rng.random() < 0.5, train=rng.random() < 0.5)
      if rng.random() < 0.2:
        c["dtype"] = "float32"
    else:
      d, d_v = rng.choice([(64, 64), (80, 80), (96, 96), (128, 128), (128, 128), (192, 128), (256, 256)])
      page = rng.choice([16, 32, 64, 64, 128])
      most = _len(rng, 64, 32768)
      first, last = rng.choice([0, 1, 1, 2]), rng.choice([1, 1, 2, 4])
      c = _case(kind=kind, **heads, batch=batch, page=page, most=most, least=rng.choice([0, 1, most // 4, most]), d=d, d_v=d_v,
                fmt=rng.choice(["int4", "int4", "e4m3"]), first=first, last=last,
                group=rng.choice([g for g in (32, 64, 128) if max(d, d_v) % g == 0 and min(d, d_v) % g == 0 or g == 32]),
                t=1 if kind == "bound" else rng.choice([1, 1, 1, 2, 3, 5]), newest=rng.choice([1, _len(rng, 1, most), most]),
                count=max(first + last, min(-(-most // page), _len(rng, 4, 128))))
      if kind != "bound":
        c["soft_cap"], c["sinks"] = rng.choice([0.0, 0.0, 30.0]), rng.random() < 0.3
    w, most = work(c), largest[kind]
    if w["bytes"] <= most["bytes"] and w["flops"] <= max(most["flops"], 1.0) and w["bytes"] > 0:
      return c


# ----------------------------------------------------------------------------------------------
# rotary positions: inputs and the plain form
# ----------------------------------------------------------------------------------------------
_SCALINGS = {  # what each is made from, as a model's configuration has it
    "none": {}, "linear": {"factor": 4.0}, "base": {"factor": 8.0}, "by_parts": {"factor": 16.0, "original": 4096},
    "bands": {"factor": 8.0, "original": 8192}}


def _frequencies(c):
  """Radians a token of each pair of channels, in 64 bits, and what the rotated channels are multiplied by."""
  pair = np.arange(c["dim"] // 2, dtype=np.float64)
  spec, base, pairs = _SCALINGS[c["scaling"]], c["base"], c["dim"] // 2
  if c["scaling"] == "base":  # the last pair turns `factor` times slower, the first as before
    base = base * spec["factor"] ** (pairs / (pairs - 1.0))
  freq = base ** (-pair / pairs)
  if c["scaling"] == "linear":
    return freq / spec["factor"], 1.0
  if c["scaling"] == "by_parts":  # pairs of 32 turns and more over the original length as before, of one and fewer slower, a ramp between
    at = lambda turns: pairs * math.log(spec["original"] / (turns * 2 * math.pi)) / math.log(base)  # noqa: E731
    lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), 2 * pairs - 1)
    slow = np.clip((pair - lo) / max(hi - lo, 0.001), 0.0, 1.0)
    return freq * (1 - slow) + freq / spec["factor"] * slow, 0.1 * math.log(spec["factor"]) + 1.0
  if c["scaling"] == "bands":  # wave lengths over the original length slower, under a quarter of it as before, between by their turns
    turns = spec["original"] * freq / (2 * math.pi)
    keep = np.clip((turns - 1.0) / (4.0 - 1.0), 0.0, 1.0)
    return freq / spec["factor"] * (1 - keep) + freq * keep, 1.0
  return freq, 1.0


def _prepare_rotate(c, seed):
  dev, dtype = torch.device("cuda"), getattr(torch, c["dtype"])
  gen = torch.Generator(device=dev).manual_seed(seed)

  def rows(heads):
    """[batch, heads, t, d], stored heads first or, as a projection leaves it, tokens first."""
    if c["heads_first"]:
      return torch.randn((c["batch"], heads, c["t"], c["d"]), generator=gen, device=dev).to(dtype)
    return torch.randn((c["batch"], c["t"], heads, c["d"]), generator=gen, device=dev).to(dtype).transpose(1, 2)

  first = torch.randint(0, c["far"] + 1, (c["batch"], 1), generator=gen, device=dev)
  freq, factor = _frequencies(c)
  s = {"case": c, "q": rows(c["q_heads"]), "k": rows(c["kv_heads"]), "positions": first + torch.arange(c["t"], device=dev)[None, :],
       "freq": torch.from_numpy(freq).to(dev), "factor": factor}
  if c["train"]:
    s["grads"] = (rows(c["q_heads"]), rows(c["kv_heads"]))
  if own:  # the frequencies in the form that a model's layers share
    from tokamax_b200 import rotary
    s["rotary"] = rotary.make_rotary(c["dim"], base=c["base"], interleaved=c["interleaved"], device=dev,
                                     scaling=rotary.Scaling(c["scaling"], **_SCALINGS[c["scaling"]]) if c["scaling"] != "none" else None)
  return s


def _plain_rotate(state, x, back=False):
  c, dim = state["case"], state["case"]["dim"]
  angle = state["positions"].double()[:, None, :, None] * state["freq"]
  cos, sin = (torch.cos(angle) * state["factor"]).float(), (torch.sin(angle) * state["factor"]).float()
  if back:
    sin = -sin
  y = x.float()
  a, b = (y[..., 0:dim:2], y[..., 1:dim:2]) if c["interleaved"] else (y[..., :dim // 2], y[..., dim // 2:dim])
  a, b = a * cos - b * sin, b * cos + a * sin
  turned = torch.stack((a, b), -1).flatten(-2) if c["interleaved"] else torch.cat((a, b), -1)
  return torch.cat((turned, y[..., dim:]), -1).to(x.dtype)


def _run_rotate(state):
  c, q, k = state["case"], state["q"], state["k"]
  if own:
    from tokamax_b200 import rotary
    if not c["train"]:
      q, k = rotary.rotate(state["rotary"], state["positions"], q, k)
      return {"q": q, "k": k}
    q, k = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
    out = rotary.rotate(state["rotary"], state["positions"], q, k)
    dq, dk = torch.autograd.grad(out, (q, k), state["grads"])
    return {"q": out[0].detach(), "k": out[1].detach(), "dq": dq, "dk": dk}
  out = {"q": _plain_rotate(state, q), "k": _plain_rotate(state, k)}
  if c["train"]:
    out.update(dq=_plain_rotate(state, state["grads"][0], True), dk=_plain_rotate(state, state["grads"][1], True))
  return out


# ----------------------------------------------------------------------------------------------
# pages: inputs
# ----------------------------------------------------------------------------------------------
def _rows_of(c):
  return next(w for w in _WIDTHS if c["d"] <= w[0] and c["d_v"] <= w[1])


def _lengths(c, seed):
  rng = random.Random(seed * 7919 + 13)
  held = [rng.randint(c["least"], c["most"]) for _ in range(c["batch"])]
  held[0] = c["most"]
  if c["batch"] > 1:
    held[-1] = c["least"]
  return held


def _random_rows(c, gen, n_pages, d, row, keys):
  """Codes and scales of whole pages [n_pages, kv_heads, page, ..], as the cache holds them: keys have channels with an offset that
  all tokens of a head share and drift from page to page, values differ in size."""
  dev = gen.device
  rand = lambda *shape: torch.randn(shape, generator=gen, device=dev)  # noqa: E731
  heads, page = c["kv_heads"], c["page"]
  x = rand(n_pages, heads, page, d)
  if keys:
    x += rand(1, heads, 1, d) ** 3 + 0.7 * rand(n_pages, heads, 1, d)
  else:
    x *= torch.exp(0.5 * rand(n_pages, heads, page, 1))
  x = torch.nn.functional.pad(x, (0, row - d)).to(torch.bfloat16).float()
  if c["fmt"] == "e4m3":
    scale = (x.abs().amax(-1) / 448.0).to(torch.bfloat16)
    return (x / scale.float()[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), scale
  parts = x.unflatten(-1, (-1, c["group"]))
  zero = parts.amin(-1).to(torch.bfloat16)
  scale = ((parts.amax(-1) - parts.amin(-1)) / 15.0).to(torch.bfloat16)
  step = torch.where(scale > 0, scale, 1.0).float()[..., None]
  codes = torch.round((parts - zero.float()[..., None]) / step).clamp(0, 15).to(torch.uint8).flatten(-2)
  return codes[..., 0::2] | (codes[..., 1::2] << 4), torch.stack((zero, scale), -1)


def _random_bounds(c, gen, n_pages, row):
  """Codes and scales of the bounds of pages whose keys are as those above."""
  rand = lambda *shape: torch.randn(shape, generator=gen, device=gen.device)  # noqa: E731
  heads = c["kv_heads"]
  centre = rand(1, heads, c["d"]) ** 3 + 0.7 * rand(n_pages, heads, c["d"])
  lo, hi = centre - 2.3 - 0.4 * rand(n_pages, heads, c["d"]).abs(), centre + 2.3 + 0.4 * rand(n_pages, heads, c["d"]).abs()
  x = torch.nn.functional.pad(torch.stack((lo, hi), 2), (0, row - c["d"]))
  scale = x.abs().amax((2, 3)) / 127
  return torch.round(x / scale[:, :, None, None]).clamp(-127, 127).to(torch.int8), scale


def _pool(c, used):
  """Pages of the pool: where the bounds of all of it come back, room for the longest sequences."""
  return (c["batch"] * -(-c["most"] // c["page"]) if c["kind"] == "bound" else sum(used)) + 1


def _prepare_pages(c, seed):
  dev = torch.device("cuda")
  gen = torch.Generator(device=dev).manual_seed(seed)
  held, page = _lengths(c, seed), c["page"]
  row_k, row_v = _rows_of(c)
  used = [-(-n // page) for n in held]
  n_pages, width = _pool(c, used), max(max(used), 1)
  order = torch.randperm(n_pages, generator=gen, device=dev).int()  # pages of a sequence lie anywhere in the pool
  at = torch.arange(width, device=dev)[None, :]
  used_t = torch.tensor(used, device=dev)[:, None]
  table = torch.where(at < used_t, order[((used_t.cumsum(0) - used_t) + at).clamp_max(n_pages - 1)], -1)
  lengths = torch.tensor(held, dtype=torch.int32, device=dev)
  s = {"case": c, "table": table, "lengths": lengths, "n_pages": n_pages}
  if c["kind"] in ("bound", "attend", "step"):
    s["k_codes"], s["k_scales"] = _random_rows(c, gen, n_pages, c["d"], row_k, True)
  if c["kind"] in ("attend", "step"):
    s["v_codes"], s["v_scales"] = _random_rows(c, gen, n_pages, c["d_v"], row_v, False)
  if c["kind"] == "bound":  # what an earlier owner of a page left
    s["bound_codes"] = torch.randint(-127, 128, (n_pages, c["kv_heads"], 2, row_k), generator=gen, device=dev, dtype=torch.int8)
    s["bound_codes"][..., c["d"]:] = 0
    s["bound_scales"] = torch.rand((n_pages, c["kv_heads"]), generator=gen, device=dev)
  if c["kind"] in ("choose", "step"):
    s["bound_codes"], s["bound_scales"] = _random_bounds(c, gen, n_pages, row_k)
  if c["kind"] != "bound":
    q = torch.randn((c["batch"], c["t"], c["q_heads"], c["d"]), generator=gen, device=dev) * 1.5
    s["q"] = q.to(getattr(torch, c["dtype"])).transpose(1, 2)
    s["sinks"] = torch.randn(c["q_heads"], generator=gen, device=dev) if c["sinks"] else None
    s["scale"] = c["d"] ** -0.5
  if c["kind"] == "attend":
    s["tables"], s["table_lengths"] = _random_choice(c, gen, table, lengths)
  if own:  # the handles of the same arrays
    from tokamax_b200 import kv_cache
    s["cache"] = kv_cache.make_kv_cache(n_pages, page, c["kv_heads"], c["d"], c["d_v"], fmt=c["fmt"],
                                        group_size=c["group"] if c["fmt"] == "int4" else None, device=dev)
    for name in ("k_codes", "k_scales", "v_codes", "v_scales"):
      if name in s:
        getattr(s["cache"], name).copy_(s.pop(name))
    if "bound_codes" in s:
      s["bounds"] = kv_cache.make_page_bounds(s["cache"])
      s["bounds"].codes.copy_(s.pop("bound_codes"))
      s["bounds"].scales.copy_(s.pop("bound_scales"))
  return s


def _random_choice(c, gen, table, lengths):
  """Tables [batch, kv_heads, t, count] of pages taken at random, the query's own the last, and the tokens that they hold."""
  shape = (c["batch"], c["kv_heads"], c["t"])
  position = lengths[:, None].long() - c["t"] + torch.arange(c["t"], device=gen.device)[None, :]
  position = position[:, None, :].expand(shape)
  own_page = torch.div(position, c["page"], rounding_mode="floor")
  index = torch.arange(table.shape[1], device=gen.device)
  rank = torch.rand((*shape, table.shape[1]), generator=gen, device=gen.device)
  rank = torch.where(index == own_page[..., None], 2.0, rank).masked_fill(index > own_page[..., None], -1.0)
  return _as_tables(c, table, rank, own_page, position)


def prepare(case, seed):
  """What the program holds before the call: projections and positions, or the cache, its bounds and the page table."""
  c = dict(case)
  return _prepare_rotate(c, seed) if c["kind"] == "rotate" else _prepare_pages(c, seed)


def run(state):
  c = state["case"]
  if c["kind"] == "rotate":
    return _run_rotate(state)
  if own:
    from tokamax_b200 import kv_cache
    cache = state["cache"]
    if c["kind"] == "bound":
      kv_cache.bound_pages(cache, state["bounds"], state["table"], state["lengths"], c["newest"])
      return {"bounds": state["bounds"].values()}
    out = {}
    tables, lengths = state.get("tables"), state.get("table_lengths")
    if c["kind"] != "attend":
      tables, lengths = kv_cache.choose_pages(cache, state["bounds"], state["q"], state["table"], state["lengths"], c["count"],
                                              first=c["first"], last=c["last"])
      out.update(tables=tables, lengths=lengths)
    if c["kind"] != "choose":
      out["out"] = kv_cache.attend(cache, state["q"], tables, lengths, logits_scale=state["scale"],
                                   logits_soft_cap=c["soft_cap"] or None, sinks=state["sinks"])
    return out
  if c["kind"] == "bound":
    return {"bounds": _plain_bounds(state)}
  out = {}
  tables, lengths = state.get("tables"), state.get("table_lengths")
  if c["kind"] != "attend":
    tables, lengths = _plain_choose(state)
    out.update(tables=tables, lengths=lengths)
  if c["kind"] != "choose":
    out["out"] = _plain_attend(state, tables, lengths)
  return out


# ----------------------------------------------------------------------------------------------
# pages: plain forms
# ----------------------------------------------------------------------------------------------
def _plain_rows(c, codes, scales, d):
  """Values of rows [.., bytes] in 32 bits, [.., d]."""
  if c["fmt"] == "e4m3":
    return codes.view(torch.float8_e4m3fn)[..., :d].float() * scales.float()[..., None]
  x = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float().unflatten(-1, (-1, c["group"]))
  zero, scale = scales[..., 0].float()[..., None], scales[..., 1].float()[..., None]
  return (x * scale + zero).flatten(-2)[..., :d]


def _plain_bounds(state):
  """Writes the bounds of the pages that the newest tokens have made whole; returns the values of all, [n_pages, kv_heads, 2, d]."""
  c, d = state["case"], state["case"]["d"]
  table, lengths, page = state["table"], state["lengths"].long(), c["page"]
  n = min(table.shape[1], c["newest"] // page + 1)  # pages of a sequence, at most
  index = torch.div((lengths - c["newest"]).clamp_min(0), page, rounding_mode="floor")[:, None] + torch.arange(n, device=table.device)
  whole = (index + 1) * page <= lengths[:, None]
  pages = torch.where(whole, table.long().gather(1, index.clamp_max(table.shape[1] - 1)), -1)
  pages = pages[pages >= 0]
  x = _plain_rows(c, state["k_codes"][pages], state["k_scales"][pages], d).nan_to_num(0.0)
  x = torch.stack((x.amin(2), x.amax(2)), 2)
  divisor = torch.full((1,), 127.0, device=x.device)
  scale = x.abs().amax((2, 3)) / divisor
  step = torch.where(scale > 0, scale, 1.0)[:, :, None, None]
  state["bound_codes"][pages, :, :, :d] = torch.round(x / step).clamp(-127, 127).to(torch.int8)
  state["bound_scales"][pages] = scale
  return state["bound_codes"][..., :d].float() * state["bound_scales"][:, :, None, None]


def _as_tables(c, table, rank, own_page, position):
  """The pages of the `count` highest ranks (of those that are not negative), in the order of the sequence, and how many tokens
  they hold."""
  n = min(c["count"], rank.shape[-1])
  best, index = torch.sort(rank, dim=-1, descending=True, stable=True)
  index = torch.where(best[..., :n] >= 0, index[..., :n], rank.shape[-1])
  index = torch.sort(index, dim=-1).values
  taken = index < rank.shape[-1]
  pages = table[:, None, None, :].expand(*rank.shape).gather(-1, index.clamp_max(rank.shape[-1] - 1))
  pages = torch.where(taken, pages, -1)
  pages = torch.nn.functional.pad(pages, (0, c["count"] - n), value=-1)
  missing = (own_page + 1) * c["page"] - (position + 1)  # of the query's own page, which is the last
  tokens = taken.sum(-1) * c["page"] - missing
  return pages.int(), torch.where(position >= 0, tokens, 0).int()


def _plain_choose(state):
  """Scores are whole numbers times a page's scale: of q in 8 bits with the bound on its side, the largest of a kv head's q heads."""
  c, q, table = state["case"], state["q"], state["table"]
  shape = (c["batch"], c["kv_heads"], c["t"])
  group = c["q_heads"] // c["kv_heads"]
  x = q.float().nan_to_num(0.0).unflatten(1, (c["kv_heads"], group)).transpose(2, 3)  # [batch, kv_heads, t, group, d]
  divisor = torch.full((1,), 127.0, device=x.device)
  scale = x.abs().amax((3, 4), keepdim=True) / divisor
  code = torch.round(x / torch.where(scale > 0, scale, 1.0)).clamp(-127, 127)
  pages = table.long().clamp_min(0)
  lo, hi = (state["bound_codes"][pages, :, side, :c["d"]].float().permute(0, 2, 3, 1)[:, :, None] for side in (0, 1))  # [b, h, 1, d, pages]
  score = code.clamp_min(0) @ hi + code.clamp_max(0) @ lo  # whole numbers below 2^24
  score = score.amax(3) * state["bound_scales"][pages].transpose(1, 2)[:, :, None]
  position = state["lengths"][:, None].long() - c["t"] + torch.arange(c["t"], device=q.device)[None, :]
  position = position[:, None, :].expand(shape)
  own_page = torch.div(position, c["page"], rounding_mode="floor")
  index = torch.arange(table.shape[1], device=q.device)
  # as ranks: whole numbers in the order of the scores, so that what is always taken comes before and what cannot be behind
  order = torch.sort(score, dim=-1, descending=False, stable=True).values
  rank = torch.searchsorted(order, score.contiguous())
  always = (index < c["first"]) | (index > own_page[..., None] - c["last"])
  rank = torch.where(always, table.shape[1], rank).masked_fill(index > own_page[..., None], -1)
  return _as_tables(c, table, rank, own_page, position)


def _plain_attend(state, tables, lengths):
  c, q = state["case"], state["q"]
  group = c["q_heads"] // c["kv_heads"]
  pages, head = tables.long().clamp_min(0), torch.arange(c["kv_heads"], device=q.device)[None, :, None, None]
  k = _plain_rows(c, state["k_codes"][pages, head], state["k_scales"][pages, head], c["d"]).flatten(3, 4)
  x = q.float().unflatten(1, (c["kv_heads"], group)).transpose(2, 3)  # [batch, kv_heads, t, group, d]
  x = (x @ k.transpose(-1, -2)) * state["scale"]
  del k
  if c["soft_cap"]:
    x = torch.tanh(x / c["soft_cap"]) * c["soft_cap"]
  x = x.masked_fill(torch.arange(x.shape[-1], device=q.device) >= lengths[..., None, None], -math.inf)
  top = x.amax(-1, keepdim=True)
  sink = None
  if state["sinks"] is not None:
    sink = state["sinks"].view(1, c["kv_heads"], 1, group, 1)
    top = torch.maximum(top, sink)
  top = torch.where(top > -math.inf, top, 0.0)
  p = torch.exp(x - top)
  total = p.sum(-1, keepdim=True)
  if sink is not None:
    total = total + torch.exp(sink - top)
  v = _plain_rows(c, state["v_codes"][pages, head], state["v_scales"][pages, head], c["d_v"]).flatten(3, 4)
  o = (p @ v) / torch.where(total > 0, total, 1.0)
  return o.transpose(2, 3).flatten(1, 2).to(q.dtype)


# ----------------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------------
def _row_bytes(c, row):
  return row / 2 + 4 * (row // c["group"]) if c["fmt"] == "int4" else row + 2


def work(case):
  """Each input once and each output once; the products of the attention (lengths: of seed 0)."""
  c = case
  if c["kind"] == "rotate":
    values = c["batch"] * c["t"] * (c["q_heads"] + c["kv_heads"]) * c["d"]
    nbytes = 2 * values * (4 if c["dtype"] == "float32" else 2) + 8 * c["batch"] * c["t"]
    return {"bytes": float(nbytes * (2 if c["train"] else 1)), "flops": 0.0}
  held, page = _lengths(c, 0), c["page"]
  row_k, row_v = _rows_of(c)
  if c["kind"] == "bound":
    pages = sum(n // page - max(n - c["newest"], 0) // page for n in held) * c["kv_heads"]
    every = _pool(c, held) * c["kv_heads"]
    return {"bytes": float(pages * (page * _row_bytes(c, row_k) + 2 * c["d"] + 4) + every * 10 * c["d"]), "flops": 0.0}
  nbytes = flops = 0.0
  queries = c["batch"] * c["t"]
  if c["kind"] != "attend":
    nbytes += sum(-(-n // page) for n in held) * c["kv_heads"] * (2 * c["d"] + 4)
    nbytes += queries * (2 * c["q_heads"] * c["d"] + 4 * c["kv_heads"] * (c["count"] + 1))
    flops += 4.0 * c["d"] * c["q_heads"] * c["t"] * sum(-(-n // page) for n in held)
  if c["kind"] != "choose":
    seen = [min(max(n - c["t"] + 1 + i, 0), c["count"] * page) for n in held for i in range(c["t"])]
    once = sum(min(n, sum(seen[b * c["t"]:(b + 1) * c["t"]])) for b, n in enumerate(held))  # a page is read once for all queries
    nbytes += once * c["kv_heads"] * (_row_bytes(c, row_k) + _row_bytes(c, row_v)) + queries * c["q_heads"] * 2 * (c["d"] + c["d_v"])
    flops += 2.0 * sum(seen) * c["q_heads"] * (c["d"] + c["d_v"])
  return {"bytes": nbytes, "flops": flops}


# ----------------------------------------------------------------------------------------------
# the same results in 64 bits
# ----------------------------------------------------------------------------------------------
def _exact_rotate(s):
  c = s["case"]
  dim, out = c["dim"], {}
  pairs = torch.arange(dim // 2, device=s["q"].device)
  one, two = (2 * pairs, 2 * pairs + 1) if c["interleaved"] else (pairs, pairs + dim // 2)
  turn = torch.polar(torch.full((), s["factor"], dtype=torch.float64, device=s["q"].device), s["positions"].double()[..., None] * s["freq"])
  for name, x, sign in (("q", s["q"], 1), ("k", s["k"], 1), *((("dq", s["grads"][0], -1), ("dk", s["grads"][1], -1)) if c["train"] else ())):
    y = x.double()
    z = torch.complex(y[..., one].contiguous(), y[..., two].contiguous()) * (turn if sign > 0 else turn.conj())[:, None]
    y[..., one], y[..., two] = z.real, z.imag
    out[name] = y
  return out


def _exact_values(c, codes, scales, d):
  """What rows of codes stand for, in 64 bits."""
  if c["fmt"] == "e4m3":
    bits = codes.long()
    exponent, fraction = (bits >> 3) & 15, (bits & 7).double()
    size = torch.where(exponent > 0, (1 + fraction / 8) * torch.exp2(exponent.double() - 7), fraction / 8 * 2.0 ** -6)
    return (torch.where(bits > 127, -size, size) * scales.double()[..., None])[..., :d]
  x = torch.empty((*codes.shape[:-1], 2 * codes.shape[-1]), dtype=torch.float64, device=codes.device)
  x[..., 0::2], x[..., 1::2] = (codes % 16).double(), (codes // 16).double()
  x *= scales[..., 1].double().repeat_interleave(c["group"], -1)
  return (x + scales[..., 0].double().repeat_interleave(c["group"], -1))[..., :d]


def _exact_bounds(s):
  c, d, page = s["case"], s["case"]["d"], s["case"]["page"]
  codes, scales = s["bound_codes"][..., :d].double(), s["bound_scales"].double()
  table = s["table"].tolist()
  for b, n in enumerate(s["lengths"].tolist()):
    pages = table[b][max(n - c["newest"], 0) // page:n // page]
    if pages:
      x = _exact_values(c, s["k_codes"][pages], s["k_scales"][pages], d)
      x = torch.stack((x.min(2).values, x.max(2).values), 2)
      # the scale is one of 32 bits, and which whole number is the nearest is said in 32 bits
      scales[pages] = (x.abs().flatten(2).max(-1).values.float() / torch.full((1,), 127.0, device=x.device)).double()
      codes[pages] = torch.round((x / scales[pages][:, :, None, None]).float().double())
  return codes * scales[:, :, None, None]


def _exact_choice(s):
  """Lists of (page, tokens seen in it) for each (sequence, kv head, query)."""
  c, page = s["case"], s["case"]["page"]
  group, found = c["q_heads"] // c["kv_heads"], {}
  lo, hi = (s["bound_codes"][:, :, side, :c["d"]].double() for side in (0, 1))
  table = s["table"].tolist()
  for b, n in enumerate(s["lengths"].tolist()):
    pages = table[b][:-(-n // page)]
    for i in range(c["t"]):
      position = n - c["t"] + i
      for h in range(c["kv_heads"]):
        if position < 0:
          found[b, h, i] = []
          continue
        x = s["q"][b, h * group:(h + 1) * group, i].float()
        scale = x.abs().max() / torch.full((), 127.0, device=x.device)
        code = torch.round((x.double() / scale.double()).float().double()) if scale > 0 else torch.zeros_like(x, dtype=torch.float64)
        here = position // page
        at = torch.tensor(pages[:here + 1], device=x.device)
        score = torch.maximum(code[:, None] * lo[at, h], code[:, None] * hi[at, h]).sum(-1).max(0).values
        score = (score.float() * s["bound_scales"][at, h]).tolist()
        order = sorted(range(here + 1), key=lambda j: (-math.inf if j < c["first"] or j > here - c["last"] else -score[j], j))
        found[b, h, i] = [(pages[j], position % page + 1 if j == here else page) for j in sorted(order[:c["count"]])]
  return found


def exact(case, seed):
  """What ``run`` returns: rotations as products of complex numbers, bounds and dense attention page by page, in 64 bits."""
  c = dict(case)
  global own
  was, own = own, False  # (the arrays, without the framework's handles)
  try:
    s = prepare(c, seed)
  finally:
    own = was
  if c["kind"] == "rotate":
    return _exact_rotate(s)
  if c["kind"] == "bound":
    return {"bounds": _exact_bounds(s)}
  if c["kind"] == "choose":
    return None  # whole numbers alone
  if c["batch"] * c["kv_heads"] * c["t"] > 4096:
    return None
  if c["kind"] == "step":
    choice = _exact_choice(s)
  else:
    page, choice = c["page"], {}
    tables, lengths = s["tables"].tolist(), s["table_lengths"].tolist()
    for b in range(c["batch"]):
      for h in range(c["kv_heads"]):
        for i in range(c["t"]):
          n = lengths[b][h][i]
          choice[b, h, i] = [(p, min(page, n - j * page)) for j, p in enumerate(tables[b][h][i]) if j * page < n]
  group = c["q_heads"] // c["kv_heads"]
  out = torch.zeros((c["batch"], c["q_heads"], c["t"], c["d_v"]), dtype=torch.float64, device=s["q"].device)
  for (b, h, i), pages in choice.items():
    if not pages:
      continue
    at, n = [p for p, _ in pages], sum(m for _, m in pages)
    k = _exact_values(c, s["k_codes"][at, h], s["k_scales"][at, h], c["d"]).flatten(0, 1)[:n]
    v = _exact_values(c, s["v_codes"][at, h], s["v_scales"][at, h], c["d_v"]).flatten(0, 1)[:n]
    heads = slice(h * group, (h + 1) * group)
    logits = s["q"][b, heads, i].double() @ k.T / math.sqrt(c["d"])
    if c["soft_cap"]:
      logits = c["soft_cap"] * torch.tanh(logits / c["soft_cap"])
    total = torch.logsumexp(logits, -1, keepdim=True)
    if s["sinks"] is not None:
      total = torch.logaddexp(total, s["sinks"][heads].double()[:, None])
    out[b, heads, i] = torch.exp(logits - total) @ v
  return {"tables": None, "lengths": None, "out": out} if c["kind"] == "step" else {"out": out}
