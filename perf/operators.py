"""The operators of a generation's cache, measured: writing it in 8 bits, reading it back, attention of new tokens over it,
and attention of a batch whose sequences share a long prefix.

Sizes are generic serving shapes beside the benchmark's own (32 heads of 128, 4096 keys of which 512 + 256 are kept): caches of
ragged and odd lengths, 8-bit ones with a scale for each row (a token's key or value of one head), 16-bit ones, grouped and
ungrouped heads, from one sequence to 128.
"""
import math

import torch

own = False

D = 128
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
MOST = {"int8": 127.0, "e4m3": 448.0}  # largest code
SMALLEST = 2.0 ** -100                 # of a scale


def listed():
  return [
      # one decode step's keys and values of a batch, written behind what each sequence has: the smallest, latency
      {"name": "write_step", "kind": "write", "dtype": "bf16", "cache": "int8", "B": 16, "T": 1, "Hkv": 8, "cap": 1024},
      # a padded batch of prompts after its prefill, written from the first row on
      {"name": "write_prompts", "kind": "write", "dtype": "f16", "cache": "e4m3", "B": 4, "T": 2001, "Hkv": 8, "cap": 2500},
      # the headline configuration's selection (512 heavy hitters and the last 256 of 4096) compacted into an 8-bit cache
      {"name": "compact_h2o_4k", "kind": "compact", "dtype": "f16", "cache": "int8", "B": 1, "S": 4096, "Hkv": 32, "n": 768,
       "cap": 1280},
      # a ragged cache read back whole, for a kernel that takes 16 bits
      {"name": "read_ragged_5k", "kind": "read", "dtype": "bf16", "cache": "e4m3", "B": 2, "Hkv": 8, "cap": 5003},
      # the rows that a selection keeps, read back from a cache of every prompt's keys
      {"name": "read_kept", "kind": "read", "dtype": "f16", "cache": "int8", "B": 4, "Hkv": 32, "cap": 2048, "n": 512},
      # one token of one conversation, a short cache: latency
      {"name": "attn_one_token", "kind": "attn", "dtype": "f16", "cache": "e4m3", "B": 1, "Sq": 1, "H": 32, "Hkv": 8,
       "cap": 1024},
      # a decode step of a batch with grouped heads over ragged caches of an odd length
      {"name": "attn_step_gqa", "kind": "attn", "dtype": "bf16", "cache": "int8", "B": 16, "Sq": 1, "H": 32, "Hkv": 8,
       "cap": 4001},
      # the same without grouping over long caches: the most bytes
      {"name": "attn_step_16k", "kind": "attn", "dtype": "bf16", "cache": "e4m3", "B": 8, "Sq": 1, "H": 32, "Hkv": 32,
       "cap": 16384},
      # a chunk of a prompt over a long 8-bit cache: more query rows than one tile
      {"name": "attn_chunk_8k", "kind": "attn", "dtype": "bf16", "cache": "int8", "B": 2, "Sq": 100, "H": 32, "Hkv": 8,
       "cap": 8003},
      # four samples of one prompt, 16 bits, soon after they parted: latency
      {"name": "prefix_few_samples", "kind": "prefix", "dtype": "f16", "cache": "f16", "G": 1, "B": 4, "Sq": 1, "H": 32,
       "Hkv": 8, "P": 2048, "cap": 200},
      # a full batch behind one long system prompt, 16 bits: the most operations
      {"name": "prefix_batch_32k", "kind": "prefix", "dtype": "bf16", "cache": "bf16", "G": 1, "B": 128, "Sq": 1, "H": 32,
       "Hkv": 8, "P": 32768, "cap": 512},
      # eight samples each of four prompts of different lengths, five query heads to a key/value head, 8 bits
      {"name": "prefix_samples_e4m3", "kind": "prefix", "dtype": "f16", "cache": "e4m3", "G": 4, "B": 32, "Sq": 1, "H": 40,
       "Hkv": 8, "P": 6001, "cap": 700},
  ]


def _log_int(rng, lo, hi):
  return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
  kind = rng.choice(["write", "compact", "read", "attn", "attn", "attn", "prefix", "prefix"])
  dtype = rng.choice(["f16", "bf16"])
  Hkv = rng.choice([4, 8, 8, 32])
  case = {"kind": kind, "dtype": dtype, "cache": rng.choice(["int8", "e4m3"]), "Hkv": Hkv}
  if kind == "write":
    T = rng.choice([1, _log_int(rng, 2, 4000)])
    B = _log_int(rng, 1, 64) if T == 1 else rng.choice([1, 2, 3, 4])
    return {**case, "B": B, "T": T, "cap": T + _log_int(rng, 30, 1000)}
  if kind == "compact":
    S = _log_int(rng, 300, 8192)
    n = max(1, S // rng.choice([3, 5, 8]))
    return {**case, "B": rng.choice([1, 2, 4]), "S": S, "n": n, "cap": n + rng.randrange(1, 500)}
  if kind == "read":
    cap = _log_int(rng, 300, 8000)
    case = {**case, "B": rng.choice([1, 2, 4]), "cap": cap}
    return {**case, "n": max(1, cap // rng.choice([3, 4, 7]))} if rng.random() < 0.5 else case
  H = Hkv * rng.choice([1, 2, 4, 5] if Hkv < 32 else [1, 2])
  if kind == "attn":
    Sq = rng.choice([1, 1, 1, 2, 4, _log_int(rng, 5, 300)])
    cap = Sq + _log_int(rng, 100, 16000)
    B = _log_int(rng, 1, max(1, min(32, 130000 // cap)))
    return {**case, "B": B, "Sq": Sq, "H": H, "cap": cap, "cache": rng.choice(["int8", "e4m3", dtype])}
  G = rng.choice([1, 1, 2, 4])
  return {**case, "G": G, "B": G * _log_int(rng, 1, 128 // G), "Sq": rng.choice([1, 1, 1, 2, 3]), "H": H,
          "P": _log_int(rng, 200, 32000 // G), "cap": 3 + _log_int(rng, 30, 500), "cache": rng.choice(["int8", "e4m3", dtype])}


def _lengths(n, most, least=1):
  """From half of `most` to all of it, spread over `n` sequences."""
  return [max(least, most - (37 * i % n) * most // (2 * n)) for i in range(n)]


def _cache_rows(N, S, H, dtype):
  """[N, S, H, 128] whose rows of one head follow each other in memory."""
  return torch.zeros((N, H, S, D), dtype=torch.uint8 if dtype.itemsize == 1 else dtype, device="cuda").view(dtype).transpose(1, 2)


def _cache_scales(N, S, H):
  return torch.zeros((N, H, (S + 3) // 4 * 4), dtype=torch.float32, device="cuda")[..., :S]


def _quantise(x, fmt):
  """x [..., 128] -> (codes, scales [...])."""
  x = x.float()
  amax = x.abs().amax(-1).clamp_min(MOST[fmt] * SMALLEST)
  fine = torch.isfinite(amax)
  # (x * MOST is exact, and the quotient correctly rounded: a value midway between two codes goes to the even one)
  y = torch.where(fine[..., None], x * MOST[fmt] / amax[..., None], 0.0)
  return (y.round() if fmt == "int8" else y).to(DTYPES[fmt]), torch.where(fine, amax / MOST[fmt], torch.nan)


def prepare(case, seed):
  g = torch.Generator(device="cuda").manual_seed(seed)
  dt, kind, fmt, B, Hkv = DTYPES[case["dtype"]], case["kind"], case["cache"], case["B"], case["Hkv"]

  def normal(*shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=dt)

  def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")

  def kept(n, S):  # ascending, as a selection gives them
    return torch.rand((B, Hkv, S), generator=g, device="cuda").topk(n, -1).indices.sort(-1).values.int().contiguous()

  def cache(N, S):
    """A cache that has been written: (k, v) or (k, v, k_scale, v_scale).  Some of a head's channels are larger than others."""
    size = (1 + 3 * (torch.rand((Hkv, D), generator=g, device="cuda") > 0.95)).to(dt)
    k, v = _cache_rows(N, S, Hkv, DTYPES[fmt]), _cache_rows(N, S, Hkv, DTYPES[fmt])
    if fmt not in MOST:
      k.copy_(normal(N, S, Hkv, D) * size)
      v.copy_(normal(N, S, Hkv, D))
      return k, v
    scales = [_cache_scales(N, S, Hkv), _cache_scales(N, S, Hkv)]
    for rows, scale, factor in ((k, scales[0], size), (v, scales[1], 1)):
      code, sc = _quantise(normal(N, S, Hkv, D) * factor, fmt)
      rows.copy_(code)
      scale.copy_(sc.transpose(1, 2))
    return k, v, scales[0], scales[1]

  state = {"case": dict(case)}
  if kind in ("write", "compact"):
    n = case["n"] if kind == "compact" else case["T"]
    rows = case["S"] if kind == "compact" else n
    state["cache"] = (_cache_rows(B, case["cap"], Hkv, DTYPES[fmt]), _cache_rows(B, case["cap"], Hkv, DTYPES[fmt]),
                      _cache_scales(B, case["cap"], Hkv), _cache_scales(B, case["cap"], Hkv))
    state["k"], state["v"] = normal(B, rows, Hkv, D), normal(B, rows, Hkv, D)
    if kind == "compact":
      state["idx"] = kept(n, rows)
    else:
      state["start"] = ints(_lengths(B, case["cap"] - n, 0) if n == 1 else [0] * B)
      state["count"] = ints(_lengths(B, n))
    return state
  state["cache"] = cache(B, case["cap"])
  if kind == "read":
    if "n" in case:
      state["idx"] = kept(case["n"], case["cap"])
    else:
      state["kv_len"] = ints(_lengths(B, case["cap"]))
    return state
  state["q"] = normal(B, case["Sq"], case["H"], D)
  state["kv_len"] = ints(_lengths(B, case["cap"], case["Sq"]))
  if kind == "prefix":
    state["prefix"] = cache(case["G"], case["P"])
    state["prefix_len"] = ints(_lengths(case["G"], case["P"]))
  return state


def _own_run(state):
  import flashtensor_b200 as ft
  from flashtensor_b200 import ops
  case = state["case"]
  cache = ft.KVCache(*state["cache"])
  kind = case["kind"]
  if kind == "write":
    ops.quant_kv(state["k"], state["v"], cache, start=state["start"], count=state["count"])
    return state["cache"]
  if kind == "compact":
    ops.quant_kv(state["k"], state["v"], cache, idx=state["idx"])
    return state["cache"]
  if kind == "read":
    return ops.dequant_kv(cache, DTYPES[case["dtype"]], idx=state.get("idx"), kv_len=state.get("kv_len"))
  if kind == "attn":
    return ops.attn_cache(state["q"], cache, kv_len=state["kv_len"])
  return ops.attn_prefix(state["q"], ft.KVCache(*state["prefix"]), cache, kv_len=state["kv_len"],
                         prefix_len=state["prefix_len"])


def _values(rows, scale=None):
  """The values that a cache's rows stand for, in 32 bits."""
  return rows.float() if scale is None else rows.float() * scale.transpose(1, 2)[..., None]


def _logits(q, k, kv_len, causal):
  """q [B, Sq, H, 128], k [N, S, Hkv, 128], each of its N sequences for B / N of q's: scaled logits [B, Sq, H, S], -inf where masked."""
  B, Sq, H, _ = q.shape
  N, S, Hkv, _ = k.shape
  rows = q.view(N, B // N * Sq, Hkv, H // Hkv, D).transpose(1, 2).reshape(N, Hkv, -1, D)
  x = rows @ k.permute(0, 2, 3, 1) * D ** -0.5
  x = x.view(N, Hkv, B // N * Sq, H // Hkv, S).transpose(1, 2).reshape(B, Sq, H, S)
  seen = kv_len.long().repeat_interleave(B // N)[:, None].expand(B, Sq)
  if causal:
    seen = seen - Sq + 1 + torch.arange(Sq, device=q.device)
  return x.masked_fill(torch.arange(S, device=q.device) >= seen[:, :, None, None], -torch.inf)


def _weighted(w, v):
  """w [B, Sq, H, S], v [N, S, Hkv, 128] -> [B, Sq, H, 128]."""
  B, Sq, H, S = w.shape
  N, _, Hkv, _ = v.shape
  rows = w.view(N, B // N * Sq, Hkv, H // Hkv, S).transpose(1, 2).reshape(N, Hkv, -1, S)
  y = rows @ v.transpose(1, 2)
  return y.view(N, Hkv, B // N * Sq, H // Hkv, D).transpose(1, 2).reshape(B, Sq, H, D)


def _put(rows, scales, x, idx, start, count, fmt):
  """Writes x [B, T, Hkv, 128] (or its rows idx [B, Hkv, n]) into a cache."""
  if idx is not None:
    x = x.gather(1, idx.long().transpose(1, 2)[..., None].expand(-1, -1, -1, D))
  code, scale = _quantise(x, fmt)
  B, T = x.shape[:2]
  t = torch.arange(T, device=x.device)
  b = torch.arange(B, device=x.device)[:, None]
  at = t[None] if start is None else start.long()[:, None] + t
  b, at = b.expand(B, T), at.expand(B, T)
  by_row = scales.transpose(1, 2)
  if count is not None:
    real = (t[None] < count[:, None])[..., None]
    code = torch.where(real[..., None], code.view(torch.uint8), rows.view(torch.uint8)[b, at]).view(code.dtype)
    scale = torch.where(real, scale, by_row[b, at])
  rows.view(torch.uint8)[b, at] = code.view(torch.uint8)
  by_row[b, at] = scale


def run(state):
  if own:
    return _own_run(state)
  case = state["case"]
  kind, dt, cache = case["kind"], DTYPES[case["dtype"]], state["cache"]
  if kind in ("write", "compact"):
    _put(cache[0], cache[2], state["k"], state.get("idx"), state.get("start"), state.get("count"), case["cache"])
    _put(cache[1], cache[3], state["v"], state.get("idx"), state.get("start"), state.get("count"), case["cache"])
    return cache
  k, v = _values(cache[0], *cache[2:3]), _values(cache[1], *cache[3:4])
  if kind == "read":
    if "idx" in state:
      at = state["idx"].long().transpose(1, 2)[..., None].expand(-1, -1, -1, D)
      return k.gather(1, at).to(dt), v.gather(1, at).to(dt)
    real = (torch.arange(case["cap"], device=k.device) < state["kv_len"][:, None])[..., None, None]
    return torch.where(real, k, 0).to(dt), torch.where(real, v, 0).to(dt)
  q = state["q"].float()
  x = _logits(q, k, state["kv_len"], True)
  if kind == "attn":
    p = torch.exp(x - x.amax(-1, keepdim=True))
    return (_weighted(p, v) / p.sum(-1, keepdim=True)).to(dt)
  prefix = state["prefix"]
  pk, pv = _values(prefix[0], *prefix[2:3]), _values(prefix[1], *prefix[3:4])
  y = _logits(q, pk, state["prefix_len"], False)
  top = torch.maximum(x.amax(-1, keepdim=True), y.amax(-1, keepdim=True))
  x, y = torch.exp(x - top), torch.exp(y - top)
  return ((_weighted(x, v) + _weighted(y, pv)) / (x.sum(-1, keepdim=True) + y.sum(-1, keepdim=True))).to(dt)


def work(case):
  kind, B, Hkv = case["kind"], case["B"], case["Hkv"]
  width = 1 if case["cache"] in MOST else 2
  row = 2 * (D * width + (4 if width == 1 else 0))  # a token's key and value of one head in the cache
  if kind in ("write", "compact"):
    rows = Hkv * (B * case["n"] if kind == "compact" else sum(_lengths(B, case["T"])))
    return {"bytes": rows * (2 * D * 2 + row) + (4 * rows if kind == "compact" else 8 * B), "flops": rows * 2 * D * 3}
  if kind == "read":
    rows = Hkv * (B * case["n"] if "n" in case else sum(_lengths(B, case["cap"])))
    written = Hkv * B * case.get("n", case["cap"])
    return {"bytes": rows * row + written * 2 * D * 2 + (4 * rows if "n" in case else 4 * B), "flops": rows * 2 * D}
  Sq, H = case["Sq"], case["H"]
  lens = _lengths(B, case["cap"], Sq)
  pairs = H * sum(Sq * n - Sq * (Sq - 1) // 2 for n in lens)
  nbytes = 2 * B * Sq * H * D * 2 + Hkv * sum(lens) * row + 4 * B
  if kind == "prefix":
    shared = _lengths(case["G"], case["P"])
    pairs += H * Sq * B // case["G"] * sum(shared)
    nbytes += Hkv * sum(shared) * row + 4 * case["G"]
  return {"bytes": nbytes, "flops": 4 * D * pairs}


def _exact_codes(x, fmt):
  """(codes, scales) of x [..., 128] in 64 bits."""
  x = x.double()
  amax = torch.clamp(x.abs().max(-1).values, min=MOST[fmt] * SMALLEST)
  scale = amax / MOST[fmt]
  y = x * MOST[fmt] / amax.unsqueeze(-1)
  if fmt == "int8":
    return torch.round(y), scale
  # e4m3: four significant bits down to 2^-6, steps of 2^-9 below
  step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
  return torch.round(y / step) * step, scale


def _exact_cache(cache, b, n):
  """Keys and values [Hkv, n, 128] of sequence b in 64 bits."""
  found = []
  for which in (0, 1):
    rows = cache[which][b, :n].double().transpose(0, 1)
    found.append(rows * cache[2 + which][b, :, :n].double().unsqueeze(-1) if len(cache) == 4 else rows)
  return found


def exact(case, seed):
  state = prepare(case, seed)
  kind, cache, B, Hkv = case["kind"], state["cache"], case["B"], case["Hkv"]
  if kind in ("write", "compact"):
    out = [c.double() for c in cache]
    for b in range(B):
      first = int(state["start"][b]) if "start" in state else 0
      for which, x in ((0, state["k"][b]), (1, state["v"][b])):
        if "idx" in state:
          x = torch.stack([x[state["idx"][b, h].long(), h] for h in range(Hkv)], 1)
        else:
          x = x[:int(state["count"][b])]
        codes, scales = _exact_codes(x, case["cache"])
        out[which][b, first:first + x.shape[0]] = codes
        out[2 + which][b, :, first:first + x.shape[0]] = scales.T
    if case["cache"] == "int8":
      out[0], out[1] = out[0].to(torch.int8), out[1].to(torch.int8)
    return tuple(out)
  if kind == "read":
    n = case.get("n", case["cap"])
    outs = [torch.zeros((B, n, Hkv, D), dtype=torch.float64, device="cuda") for _ in range(2)]
    for b in range(B):
      upto = int(state["kv_len"][b]) if "kv_len" in state else case["cap"]
      for out, rows in zip(outs, _exact_cache(cache, b, upto)):
        if "idx" in state:
          out[b] = torch.stack([rows[h, state["idx"][b, h].long()] for h in range(Hkv)], 1)
        else:
          out[b, :upto] = rows.transpose(0, 1)
    return tuple(outs)
  Sq, group = case["Sq"], case["H"] // Hkv
  out = torch.empty((B, Sq, case["H"], D), dtype=torch.float64, device="cuda")
  for b in range(B):
    n = int(state["kv_len"][b])
    k, v = _exact_cache(cache, b, n)
    q = state["q"][b].double().view(Sq, Hkv, group, D).permute(1, 2, 0, 3)  # [Hkv, group, Sq, 128]
    s = torch.matmul(q, k.transpose(1, 2).unsqueeze(1)) / math.sqrt(D)
    late = torch.ones((Sq, n), dtype=torch.bool, device="cuda").triu(n - Sq + 1)
    s = s.masked_fill(late, float("-inf"))
    if kind == "prefix":
      g = b * case["G"] // B
      pk, pv = _exact_cache(state["prefix"], g, int(state["prefix_len"][g]))
      s = torch.cat((torch.matmul(q, pk.transpose(1, 2).unsqueeze(1)) / math.sqrt(D), s), -1)
      v = torch.cat((pv, v), 1)
    out[b] = torch.matmul(torch.softmax(s, -1), v.unsqueeze(1)).permute(2, 0, 1, 3).reshape(Sq, case["H"], D)
  return out
