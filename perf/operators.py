"""Timing cases of the quantised key / value cache: writing it, reading it back, and attention over it.

A case is a dict of plain values.  ``kind`` says which operators it goes through:

  write   ``kv_cache.append`` of new tokens and ``kv_cache.read`` of the sequences that they join
  read    ``kv_cache.read`` alone: the cached prefix that a chunk of a prompt is about to attend to
  attend  ``kv_cache.attend``: the attention of the newest ``t`` tokens of every sequence

A cache holds tokens in pages of ``page`` tokens, scattered over a pool.  ``fmt`` is how it holds a token's row of
one head: ``int4`` (codes 0 .. 15; a bf16 scale and a bf16 zero for each ``group`` channels) or ``e4m3`` (one bf16
scale for the row).  Sequences have ``least`` .. ``most`` tokens, another number each.  The plain forms below hold
the same codes in a layout of their own.
"""

import math
import random

import torch

own = False

MASK_VALUE = -0.7 * 3.4028234663852886e38  # logsumexp of a row that sees nothing

_DEFAULTS = dict(kind="attend", fmt="int4", group=64, page=64, batch=1, least=1, most=1024, t=1, q_heads=32, kv_heads=8,
                 d=128, d_v=0, window=0, soft_cap=0.0, sinks=False, residuals=False, dtype="bfloat16")


def _case(**kw):
  c = dict(_DEFAULTS, **kw)
  c["d_v"] = c["d_v"] or c["d"]
  return c


def listed():
  return [
      # A chat's first decoding steps in a small model: one token for each of eight sequences. All launches and latency.
      _case(name="write_token", kind="write", group=32, page=16, batch=8, least=1, most=31, t=1, q_heads=8, kv_heads=2, d=64),
      # Prompts of up to 4096 tokens, padded to the longest, go into an empty cache.
      _case(name="write_prompts", kind="write", batch=4, least=0, most=0, t=4096),
      # A chunk of a prompt behind what earlier chunks left, everything odd: 517 tokens, a head dim of 80, f16.
      _case(name="write_chunk_e4m3", kind="write", fmt="e4m3", page=32, batch=3, least=1999, most=6001, t=517, q_heads=12,
            kv_heads=4, d=80, dtype="float16"),
      # The prefix of a chunked prefill, of two sequences.
      _case(name="read_prefix", kind="read", batch=2, least=9000, most=16384),
      # The same from eight bits, for long documents.
      _case(name="read_long_e4m3", kind="read", fmt="e4m3", page=128, batch=4, least=20000, most=32768),
      # One token of one short sequence in a small model.
      _case(name="attend_one", group=32, page=16, least=777, most=777, q_heads=8, kv_heads=2, d=64),
      # A batch of chats of all lengths, grouped heads: the ordinary decoding step.
      _case(name="attend_batch", batch=64, least=200, most=4096),
      # One very long document: a single row has to fill the GPU.
      _case(name="attend_long", least=131072, most=131072),
      # A full server: long contexts in every slot. The largest.
      _case(name="attend_server", batch=32, least=8192, most=32768),
      # Sliding window and sinks, head dim 64, eight bits, f16.
      _case(name="attend_window_sinks", fmt="e4m3", page=32, batch=24, least=1, most=6016, q_heads=64, kv_heads=8, d=64,
            window=1024, sinks=True, dtype="float16"),
      # Five drafted tokens a sequence are checked at once; the program keeps the logsumexp.
      _case(name="attend_drafts", fmt="e4m3", batch=16, least=1000, most=8192, t=5, residuals=True),
      # One kv head for all, head dim 256, soft cap; one sequence has no tokens yet.
      _case(name="attend_mqa_hd256", group=128, page=32, batch=12, least=0, most=10000, q_heads=16, kv_heads=1, d=256,
            soft_cap=50.0),
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
    kind = rng.choice(["write", "read", "attend", "attend", "attend"])
    fmt = rng.choice(["int4", "int4", "e4m3"])
    d, d_v = rng.choice([(64, 64), (80, 80), (96, 96), (128, 128), (128, 128), (192, 128), (256, 256)])
    group = rng.choice([g for g in (32, 64, 128) if max(d, d_v) % g == 0 and min(d, d_v) % g == 0 or g == 32])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 8, 16])
    c = dict(kind=kind, fmt=fmt, d=d, d_v=d_v, group=group, kv_heads=kv_heads, q_heads=kv_heads * rng.choice([1, 2, 4, 4, 5, 8]),
             page=rng.choice([16, 32, 64, 128]), dtype=rng.choice(["bfloat16", "bfloat16", "float16"]),
             batch=max(1, round(math.exp(rng.uniform(0.0, math.log(64))))))
    if kind == "write":
      c["t"] = rng.choice([1, _len(rng, 1, 4096)])
      c["most"] = rng.choice([0, _len(rng, 1, 8192)])
    else:
      c["most"] = _len(rng, 64, 32768)
    c["least"] = rng.choice([0, 1, c["most"] // 4, c["most"]]) if c["most"] else 0
    if kind == "attend":
      c["t"] = rng.choice([1, 1, 1, 2, 3, 5, 8])
      c["window"] = rng.choice([0, 0, rng.randrange(16, max(17, c["most"]))])
      c["soft_cap"] = rng.choice([0.0, 0.0, 30.0, 50.0])
      c["sinks"] = rng.random() < 0.3
      c["least"] = max(c["least"], c["t"] if c["least"] else 0)
      c["most"] = max(c["most"], c["least"])
    c = _case(**c)
    w, most = work(c), largest[kind]
    if w["bytes"] <= most["bytes"] and w["flops"] <= max(most["flops"], 1.0):
      return c


# ----------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------
def _lengths(c, seed):
  """Tokens that each sequence has in the cache, and how many new ones a write brings."""
  rng = random.Random(seed * 7919 + 13)
  held = [rng.randint(c["least"], c["most"]) for _ in range(c["batch"])]
  held[0] = c["most"]
  if c["batch"] > 1:
    held[-1] = c["least"]
  new = [0] * c["batch"]
  if c["kind"] == "write":
    new = [c["t"]] + [rng.randint(max(1, c["t"] // 8), c["t"]) for _ in range(c["batch"] - 1)]
  return held, new


def _tokens(c, seed, b, n, device):
  """Keys and values of `n` tokens of sequence b, [kv_heads, n, d]: some channels of a head carry an offset that all
  its keys share, and tokens differ in the size of their values."""
  gen = torch.Generator(device=device).manual_seed((seed * 1009 + b) % (1 << 62))
  rand = lambda *shape: torch.randn(shape, generator=gen, device=device)  # noqa: E731
  offset = rand(c["kv_heads"], 1, c["d"]) ** 3
  size = torch.exp(0.5 * rand(c["kv_heads"], n, 1))
  dtype = getattr(torch, c["dtype"])
  return (rand(c["kv_heads"], n, c["d"]) + offset).to(dtype), (rand(c["kv_heads"], n, c["d_v"]) * size).to(dtype)


def prepare(case, seed):
  """What the program holds before the call: the cache with the tokens of earlier calls, the page table, the new tokens
  or the queries, on the device."""
  c = dict(case)
  dev = torch.device("cuda")
  held, new = _lengths(c, seed)
  total = [a + b for a, b in zip(held, new)]
  page = c["page"]
  longest = max(max(total), 1)
  pages_each = -(-longest // page)
  used = [-(-n // page) for n in total]
  order = list(range(sum(used) + 1))
  random.Random(seed).shuffle(order)  # pages of a sequence lie anywhere in the pool
  rows, at = [], 0
  for n in used:
    rows.append(order[at:at + n] + [0] * (pages_each - n))
    at += n
  table = torch.tensor(rows, dtype=torch.int32, device=dev)
  lengths = torch.tensor(total, dtype=torch.int32, device=dev)
  s = {"case": c, "table": table, "lengths": lengths, "longest": longest, "held": held, "new": new}
  if own:
    from tokamax_b200 import kv_cache
    s["cache"] = kv_cache.make_kv_cache(len(order), page, c["kv_heads"], c["d"], c["d_v"], fmt=c["fmt"],
                                        group_size=c["group"] if c["fmt"] == "int4" else None, device=dev)
  else:
    s["pool"] = _plain_pool(c, len(order) * page, dev)

  def slots(b, first, n):
    pos = torch.arange(first, first + n, device=dev)
    return table[b].long()[pos // page] * page + pos % page

  dtype = getattr(torch, c["dtype"])
  new_slots = torch.full((c["batch"], c["t"]), -1, dtype=torch.int64, device=dev)
  # new tokens as a projection leaves them, [batch, t, heads, d], seen as [batch, heads, t, d]
  new_k = torch.zeros((c["batch"], c["t"], c["kv_heads"], c["d"]), dtype=dtype, device=dev).transpose(1, 2)
  new_v = torch.zeros((c["batch"], c["t"], c["kv_heads"], c["d_v"]), dtype=dtype, device=dev).transpose(1, 2)
  for b in range(c["batch"]):
    if total[b] == 0:
      continue
    k, v = _tokens(c, seed, b, total[b], dev)
    if held[b]:
      at = slots(b, 0, held[b])
      if own:
        kv_cache.append(s["cache"], k[None, :, :held[b]], v[None, :, :held[b]], at[None])
      else:
        _plain_write(c, s["pool"], k[:, :held[b]], v[:, :held[b]], at)
    if new[b]:
      new_slots[b, :new[b]] = slots(b, held[b], new[b])
      new_k[b, :, :new[b]] = k[:, held[b]:]
      new_v[b, :, :new[b]] = v[:, held[b]:]
  if c["kind"] == "write":
    s.update(k=new_k, v=new_v, slots=new_slots)
  if c["kind"] == "attend":
    gen = torch.Generator(device=dev).manual_seed(seed + (1 << 40))
    q = torch.randn((c["batch"], c["t"], c["q_heads"], c["d"]), generator=gen, device=dev) * 1.5
    s["q"] = q.to(dtype).transpose(1, 2)
    s["sinks"] = torch.randn(c["q_heads"], generator=gen, device=dev) if c["sinks"] else None
    s["scale"] = c["d"] ** -0.5
  return s


def run(state):
  c = state["case"]
  if own:
    from tokamax_b200 import kv_cache
    dtype = getattr(torch, c["dtype"])
    if c["kind"] == "write":
      kv_cache.append(state["cache"], state["k"], state["v"], state["slots"])
    if c["kind"] in ("write", "read"):
      k, v = kv_cache.read(state["cache"], state["table"], state["lengths"], state["longest"], dtype=dtype)
      return {"k": k, "v": v}
    out = kv_cache.attend(state["cache"], state["q"], state["table"], state["lengths"], logits_scale=state["scale"],
                          local_window_size=c["window"] or None, logits_soft_cap=c["soft_cap"] or None,
                          sinks=state["sinks"], save_residuals=c["residuals"])
    return {"out": out[0], "logsumexp": out[1]["logsumexp"]} if c["residuals"] else {"out": out}
  if c["kind"] == "write":
    for b in range(c["batch"]):
      _plain_write(c, state["pool"], state["k"][b], state["v"][b], state["slots"][b])
  if c["kind"] in ("write", "read"):
    return _plain_read(state)
  return _plain_attend(state)


# ----------------------------------------------------------------------------------------------
# plain forms
# ----------------------------------------------------------------------------------------------
def _parts(c, d):
  """First and last channel of every group of a row of d channels."""
  step = c["group"] if c["fmt"] == "int4" else d
  return [(lo, min(lo + step, d)) for lo in range(0, d, step)]


def _plain_pool(c, n_slots, dev):
  """Codes [slot, kv head, channel] (int4: two to a byte) and scales [slot, kv head, group]; the last slot takes what
  no sequence keeps."""
  pool = {}
  for name, d in (("k", c["d"]), ("v", c["d_v"])):
    shape = (n_slots + 1, c["kv_heads"])
    if c["fmt"] == "int4":
      pool[name] = torch.zeros((*shape, d // 2), dtype=torch.uint8, device=dev)
      pool[name + "_zero"] = torch.zeros((*shape, len(_parts(c, d))), dtype=torch.bfloat16, device=dev)
      pool[name + "_scale"] = torch.zeros((*shape, len(_parts(c, d))), dtype=torch.bfloat16, device=dev)
    else:
      pool[name] = torch.zeros((*shape, d), dtype=torch.float8_e4m3fn, device=dev)
      pool[name + "_scale"] = torch.zeros((*shape, 1), dtype=torch.bfloat16, device=dev)
  return pool


def _plain_write(c, pool, k, v, slots):
  """k, v [kv_heads, n, d] into the slots; a slot of -1 is not kept."""
  at = torch.where(slots < 0, pool["k"].shape[0] - 1, slots)
  # divisors as tensors: a division by a plain number may be done as a product with its rounded reciprocal
  steps, most_code = (torch.full((1,), x, device=k.device) for x in (15.0, 448.0))
  for name, rows in (("k", k), ("v", v)):
    x = rows.transpose(0, 1).float()
    codes, scales, zeros = [], [], []
    for lo, hi in _parts(c, x.shape[-1]):
      part = x[..., lo:hi]
      if c["fmt"] == "int4":
        least, most = part.amin(-1, keepdim=True), part.amax(-1, keepdim=True)
        scale, zero = ((most - least) / steps).to(torch.bfloat16), least.to(torch.bfloat16)
        step = torch.where(scale > 0, scale, 1.0).float()
        codes.append(torch.round((part - zero.float()) / step).clamp(0, 15).to(torch.uint8))
        zeros.append(zero)
      else:
        scale = (part.abs().amax(-1, keepdim=True) / most_code).to(torch.bfloat16)
        codes.append((part / torch.where(scale > 0, scale, 1.0).float()).clamp(-448.0, 448.0).to(torch.float8_e4m3fn))
      scales.append(scale)
    codes = torch.cat(codes, -1) if len(codes) > 1 else codes[0]
    if c["fmt"] == "int4":
      codes = codes[..., 0::2] | (codes[..., 1::2] << 4)
      pool[name + "_zero"][at] = torch.cat(zeros, -1)
    pool[name].view(torch.uint8)[at] = codes.view(torch.uint8)
    pool[name + "_scale"][at] = torch.cat(scales, -1)


def _plain_rows(c, pool, name, at, d):
  """The values of the rows `at` in 32 bits, [..., kv_heads, d]."""
  codes = pool[name].view(torch.uint8)[at]
  scale = pool[name + "_scale"][at].float()
  if c["fmt"] != "int4":
    return codes.view(torch.float8_e4m3fn).float() * scale
  zero = pool[name + "_zero"][at].float()
  x = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()
  for i, (lo, hi) in enumerate(_parts(c, d)):
    x[..., lo:hi] = x[..., lo:hi] * scale[..., i:i + 1] + zero[..., i:i + 1]
  return x


def _plain_slots(state, b, n):
  c = state["case"]
  pos = torch.arange(n, device=state["table"].device)
  return state["table"][b].long()[pos // c["page"]] * c["page"] + pos % c["page"]


def _plain_read(state):
  c, n = state["case"], state["longest"]
  dtype, dev = getattr(torch, c["dtype"]), state["table"].device
  live = torch.arange(n, device=dev)[None, :] < state["lengths"][:, None]
  out = {}
  for name, d in (("k", c["d"]), ("v", c["d_v"])):
    out[name] = torch.empty((c["batch"], c["kv_heads"], n, d), dtype=dtype, device=dev)
    for b in range(c["batch"]):
      x = _plain_rows(c, state["pool"], name, _plain_slots(state, b, n), d)
      out[name][b] = torch.where(live[b][:, None, None], x, 0.0).to(dtype).transpose(0, 1)
  return out


def _plain_attend(state):
  c = state["case"]
  q, t, n = state["q"], c["t"], state["longest"]
  group = c["q_heads"] // c["kv_heads"]
  out = torch.empty((c["batch"], c["q_heads"], t, c["d_v"]), dtype=q.dtype, device=q.device)
  lse = torch.empty((c["batch"], c["q_heads"], t), dtype=torch.float32, device=q.device)
  at_k = torch.arange(n, device=q.device)
  for b in range(c["batch"]):
    slots = _plain_slots(state, b, n)
    k = _plain_rows(c, state["pool"], "k", slots, c["d"]).transpose(0, 1)
    v = _plain_rows(c, state["pool"], "v", slots, c["d_v"]).transpose(0, 1)
    rows = q[b].float().reshape(c["kv_heads"], group * t, c["d"])
    x = (rows @ k.transpose(1, 2)) * state["scale"]
    if c["soft_cap"]:
      x = torch.tanh(x / c["soft_cap"]) * c["soft_cap"]
    at_q = (state["lengths"][b] - t + torch.arange(t, device=q.device))[:, None]
    keep = at_k[None, :] <= at_q
    if c["window"]:
      keep = keep & (at_k[None, :] >= at_q - c["window"])
    x = x.view(c["kv_heads"], group, t, n).masked_fill(~keep, -math.inf)
    top = x.amax(-1, keepdim=True)
    sink = None
    if state["sinks"] is not None:
      sink = state["sinks"].view(c["kv_heads"], group, 1, 1)
      top = torch.maximum(top, sink)
    top = torch.where(top > -math.inf, top, 0.0)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    if sink is not None:
      total = total + torch.exp(sink - top)
    o = (p.view(c["kv_heads"], group * t, n) @ v).view(c["kv_heads"], group, t, c["d_v"])
    out[b] = (o / torch.where(total > 0, total, 1.0)).view(c["q_heads"], t, c["d_v"]).to(q.dtype)
    lse[b] = torch.where(total > 0, top + torch.log(total), MASK_VALUE).view(c["q_heads"], t)
  return {"out": out, "logsumexp": lse} if c["residuals"] else {"out": out}


# ----------------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------------
def _row_bytes(c):
  """Bytes of one token of one kv head in the cache, keys and values."""
  if c["fmt"] == "int4":
    return sum(d / 2 + 4 * len(_parts(c, d)) for d in (c["d"], c["d_v"]))
  return c["d"] + c["d_v"] + 4


def work(case):
  """Each input once and each output once; the products of the attention (lengths: of seed 0)."""
  c = case
  held, new = _lengths(c, 0)
  wide = 2 * (c["d"] + c["d_v"]) * c["kv_heads"]  # a token's keys and values in 16 bits
  if c["kind"] != "attend":
    tokens = sum(held) + sum(new)
    back = wide * c["batch"] * max(max(a + b for a, b in zip(held, new)), 1)
    # written rows go out and are read again by the read, which is a call of its own
    nbytes = sum(new) * (wide + _row_bytes(c) * c["kv_heads"]) + tokens * _row_bytes(c) * c["kv_heads"] + back
    return {"bytes": float(nbytes), "flops": 0.0}
  pairs, tokens = 0, 0
  for n in held:
    seen = [min(max(n - c["t"] + i + 1, 0), c["window"] + 1 if c["window"] else n) for i in range(c["t"])]
    pairs += sum(seen)
    tokens += min(n, c["window"] + c["t"]) if c["window"] else n
  q_rows = c["batch"] * c["q_heads"] * c["t"]
  nbytes = tokens * c["kv_heads"] * _row_bytes(c) + q_rows * 2 * (c["d"] + c["d_v"]) + 4 * q_rows * c["residuals"]
  return {"bytes": float(nbytes), "flops": 2.0 * pairs * c["q_heads"] * (c["d"] + c["d_v"])}


# ----------------------------------------------------------------------------------------------
# the same results in 64 bits
# ----------------------------------------------------------------------------------------------
def _held_values(c, x):
  """What the cache holds for the rows x [heads, n, d], in 64 bits, from the definition of its format."""
  x = x.double()
  if c["fmt"] == "e4m3":
    scale = (x.abs().amax(-1, keepdim=True) / 448).bfloat16().double()
    y = torch.where(scale > 0, x / scale, torch.zeros_like(x)).clamp(-448, 448)
    _, exponent = torch.frexp(y)  # |y| in [2^(exponent - 1), 2^exponent): three bits below the leading one
    step = torch.exp2((exponent - 1).clamp_min(-6).double() - 3)
    return torch.round(y / step) * step * scale
  out = torch.empty_like(x)
  for first in range(0, x.shape[-1], c["group"]):
    y = x[..., first:first + c["group"]]
    zero = y.min(-1, keepdim=True).values.bfloat16().double()
    scale = ((y.max(-1, keepdim=True).values - y.min(-1, keepdim=True).values) / 15).bfloat16().double()
    code = torch.where(scale > 0, torch.round((y - zero) / scale), torch.zeros_like(y)).clamp(0, 15)
    out[..., first:first + c["group"]] = zero + scale * code
  return out


def exact(case, seed):
  """What ``run`` returns: rows as the cache holds them, or dense attention over them, in 64 bits."""
  c = dict(case)
  dev = torch.device("cuda")
  held, new = _lengths(c, seed)
  total = [a + b for a, b in zip(held, new)]
  longest = max(max(total), 1)
  if c["kind"] != "attend":
    out = {"k": torch.zeros((c["batch"], c["kv_heads"], longest, c["d"]), dtype=torch.float64, device=dev),
           "v": torch.zeros((c["batch"], c["kv_heads"], longest, c["d_v"]), dtype=torch.float64, device=dev)}
    for b, n in enumerate(total):
      if n:
        for name, x in zip(("k", "v"), _tokens(c, seed, b, n, dev)):
          out[name][b, :, :n] = _held_values(c, x)
    return out
  gen = torch.Generator(device=dev).manual_seed(seed + (1 << 40))
  q = torch.randn((c["batch"], c["t"], c["q_heads"], c["d"]), generator=gen, device=dev) * 1.5
  q = q.to(getattr(torch, c["dtype"])).double()
  sinks = torch.randn(c["q_heads"], generator=gen, device=dev).double() if c["sinks"] else None
  out = torch.zeros((c["batch"], c["q_heads"], c["t"], c["d_v"]), dtype=torch.float64, device=dev)
  lse = torch.full((c["batch"], c["q_heads"], c["t"]), MASK_VALUE, dtype=torch.float64, device=dev)
  for b, n in enumerate(total):
    if n == 0:
      if sinks is not None:
        lse[b] = sinks[:, None]
      continue
    k, v = (_held_values(c, x) for x in _tokens(c, seed, b, n, dev))
    for h in range(c["q_heads"]):
      kh, vh = k[h * c["kv_heads"] // c["q_heads"]], v[h * c["kv_heads"] // c["q_heads"]]
      x = (q[b, :, h] @ kh.T) / math.sqrt(c["d"])
      if c["soft_cap"]:
        x = c["soft_cap"] * torch.tanh(x / c["soft_cap"])
      for i in range(c["t"]):
        last = n - c["t"] + i
        first = max(0, last - c["window"]) if c["window"] else 0
        logits = x[i, first:last + 1] if last >= 0 else x[i, :0]
        if sinks is not None:
          logits = torch.cat((logits, sinks[h:h + 1]))
        if logits.numel() == 0:
          continue
        lse[b, h, i] = torch.logsumexp(logits, 0)
        if last >= 0:
          out[b, h, i] = torch.exp(x[i, first:last + 1] - lse[b, h, i]) @ vh[first:last + 1]
  return {"out": out, "logsumexp": lse} if c["residuals"] else {"out": out}
