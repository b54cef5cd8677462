"""GPU: the 8-bit cache (written, compacted into, read back) and attention over caches and shared prefixes, against plain
implementations in 64 bits.

Codes, scales and values read back have one right answer and are compared exactly.  An attention output may be off by what
its roundings add up to, which `_attention` bounds for every output from the same inputs in 64 bits:
  - the output's own rounding, `half` = finfo(q.dtype).eps / 2 of it;
  - the weights' before the second product: `half` of each (f16, 2^-11, or bf16, 2^-8), and 2^-25 of the largest
    where a weight is subnormal in f16;
  - over an 8-bit cache, bf16 queries as f16 under a power of two: 2^-25 of a row's largest value in every term; and keys and values,
    where more than 16 rows use them, as f16 under a power of two of the largest of 32: 2^-11 of each, 2^-24 of the
    largest where it is subnormal;
  - f32 arithmetic: 2^-24 for each of a dot product's 128 terms, 2^-20 for an exponential, 2^-22 for each of the few rescalings.
"""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

D = 128
MOST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
FORMATS = [torch.int8, torch.float8_e4m3fn]
TYPES = [torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def ops(built_lib):
  if not torch.cuda.is_available():
    pytest.fail("the GPU tests need a CUDA device")
  from flashtensor_b200 import ops as _ops
  yield _ops
  assert _ops.device_status() == (0, 0)


def ft():
  import flashtensor_b200
  return flashtensor_b200


def gen(seed):
  return torch.Generator(device="cuda").manual_seed(seed)


def ints(values):
  return torch.tensor(values, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------------------
# plain implementations
# ------------------------------------------------------------------------------------------
def codes_of(x, fmt):
  """(codes, scales) of x [..., 128] by the definition, in 64 bits."""
  x = x.double()
  amax = x.abs().amax(-1)
  fine = torch.isfinite(amax)
  a = torch.where(fine, amax, 0.0).clamp(min=MOST[fmt] * 2.0 ** -100)
  y = torch.where(fine[..., None], x, 0.0) * MOST[fmt] / a[..., None]
  if fmt == torch.int8:
    code = y.round().to(torch.int8)
  else:
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    code = ((y / step).round() * step).float().to(fmt)
  return code, torch.where(fine, a / MOST[fmt], float("nan"))


def raw(t):
  return t.contiguous().view(torch.uint8 if t.element_size() == 1 else torch.int16)


def same(a, b):
  """The same bits (NaN and signed zeros included)."""
  return torch.equal(raw(a), raw(b)) if a.dtype != torch.float32 else torch.equal(a.contiguous().view(torch.int32), b.contiguous().view(torch.int32))


def make_cache(N, S, H, fmt, seed, dtype=torch.float16, spread=1.0, token_major=False):
  """A filled KVCache; 8-bit ones hold quantised normal values."""
  g = gen(seed)
  c = ft().KVCache.empty(N, S, H, dtype=fmt)
  if token_major:
    scales = (c.k_scale, c.v_scale) if c.k_scale is not None else ()
    c = ft().KVCache(*[torch.empty(N, S, H, D, dtype=fmt, device="cuda") for _ in range(2)], *scales)
  for rows, scale in ((c.k, c.k_scale), (c.v, c.v_scale)):
    x = torch.randn(N, S, H, D, generator=g, device="cuda").to(dtype) * spread
    if scale is None:
      rows.copy_(x)
    else:
      code, sc = codes_of(x, fmt)
      rows.view(torch.uint8).copy_(code.view(torch.uint8))
      scale.copy_(sc.float().transpose(1, 2))
  return c


def values(c):
  """(k, v) of a cache in 64 bits."""
  if c.k_scale is None:
    return c.k.double(), c.v.double()
  return (c.k.float().double() * c.k_scale.double().transpose(1, 2)[..., None],
          c.v.float().double() * c.v_scale.double().transpose(1, 2)[..., None])


def _attention(q, cache, kv_len=None, causal=True, prefix=None, prefix_len=None, scale=D ** -0.5):
  """(out, lse, bound of an output's error, bound of an lse's) in 64 bits, one sequence at a time."""
  B, Sq, H, _ = q.shape
  Hkv = cache.k.shape[2]
  group = H // Hkv
  half = torch.finfo(q.dtype).eps / 2
  out, lse = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.empty(B, H, Sq, dtype=torch.float64, device="cuda")
  tol, lse_tol = torch.empty_like(out), torch.empty_like(lse)
  for b in range(B):
    n = cache.k.shape[1] if kv_len is None else min(max(int(kv_len[b]), 0), cache.k.shape[1])
    one = lambda c, i, m: values(ft().KVCache(c.k[i:i + 1, :m], c.v[i:i + 1, :m], *([] if c.k_scale is None else [
        c.k_scale[i:i + 1, :, :m], c.v_scale[i:i + 1, :, :m]])))
    k, v = one(cache, b, n)
    seen = torch.ones(Sq, n, dtype=torch.bool, device="cuda")
    if causal:
      seen = seen.tril(n - Sq)
    if prefix is not None:
      g = b * prefix.k.shape[0] // B
      m = prefix.k.shape[1] if prefix_len is None else min(max(int(prefix_len[g]), 0), prefix.k.shape[1])
      pk, pv = one(prefix, g, m)
      k, v = torch.cat((pk, k), 1), torch.cat((pv, v), 1)
      seen = torch.cat((torch.ones(Sq, m, dtype=torch.bool, device="cuda"), seen), 1)
    qs = q[b].double().reshape(Sq, Hkv, group, D).permute(1, 2, 0, 3)           # [Hkv, group, Sq, D]
    k, v = k[0].permute(1, 0, 2)[:, None], v[0].permute(1, 0, 2)[:, None]    # [Hkv, 1, n, D]
    s = (qs @ k.transpose(2, 3) * scale).masked_fill(~seen, -torch.inf)
    absdot = (qs.abs() @ k.abs().transpose(2, 3) * scale).masked_fill(~seen, 0.0)
    absdot = absdot.amax(-1) if s.shape[-1] else torch.zeros(s.shape[:-1], dtype=torch.float64, device="cuda")
    top = s.amax(-1, keepdim=True) if s.shape[-1] else torch.full((*s.shape[:-1], 1), -torch.inf, dtype=torch.float64, device="cuda")
    p = torch.exp(s - top.clamp(min=-1e300))
    l = p.sum(-1, keepdim=True)
    o = torch.where(l > 0, p @ v / l.clamp(min=1e-300), 0.0)
    a = torch.where(l > 0, p @ v.abs() / l.clamp(min=1e-300), 0.0)
    most = v.abs().amax() if v.numel() else 0.0
    # (2^-25 of a query row's largest value against the largest key, 2^-24 of the largest key value against the query)
    eight = cache.k_scale is not None or (prefix is not None and prefix.k_scale is not None)
    small = (2.0 ** -25 * qs.abs().amax(-1) * (k.abs().sum(-1).amax() if k.numel() else 0.0) +
             2.0 ** -24 * qs.abs().sum(-1) * (k.abs().amax() if k.numel() else 0.0)) * scale if eight else 0.0
    by_logit = (128 * 2.0 ** -24 + (2.0 ** -11 if eight else 0)) * absdot + small + 2.0 ** -20
    of_weight = torch.expm1(2 * by_logit)[..., None] + half + 2.0 ** -18
    of_value = 2.0 ** -11 * a + 2.0 ** -24 * most if eight else 0.0
    bound = half * o.abs() + of_weight * (a + o.abs()) * 1.02 + of_value + s.shape[-1] * 2.0 ** -25 * most
    put = lambda t: t.permute(2, 0, 1, 3).reshape(Sq, H, D)
    out[b], tol[b] = put(o), put(bound)
    lse[b] = (top[..., 0] / 0.6931471805599453 + torch.log2(l[..., 0])).reshape(H, Sq)
    lse_tol[b] = (1.4427 * 2 * by_logit + 2.0 ** -20 + 2.0 ** -22 * lse[b].reshape(Hkv, group, Sq).abs().nan_to_num(0, 0, 0)).reshape(H, Sq)
  return out, lse, tol, lse_tol


def check_attention(got, lse, want, what=""):
  out, ref_lse, tol, lse_tol = want
  assert torch.isfinite(got).all(), what
  worst = ((got.double() - out).abs() / tol.clamp(min=1e-300)).masked_fill((got.double() == out), 0).max()
  assert worst <= 1, f"{what}: {worst:.2f} of the bound"
  if lse is not None:
    empty = torch.isinf(ref_lse)
    assert torch.equal(lse[empty].double(), ref_lse[empty]), what
    worst = ((lse.double() - ref_lse).abs() / lse_tol)[~empty]
    assert worst.numel() == 0 or worst.max() <= 1, f"{what}: lse {worst.max():.2f} of the bound"


# ------------------------------------------------------------------------------------------
# writing and reading back
# ------------------------------------------------------------------------------------------
def awkward_rows(T, dtype, seed):
  """[1, T, 3, 128]: normal rows of many sizes, zeros, the smallest and largest values, infinities, NaN, exact ties."""
  info = torch.finfo(dtype)
  g = gen(seed)
  x = torch.randn(1, T, 3, D, generator=g, device="cuda")
  x *= torch.exp2(torch.randint(-12, 5, (1, T, 3, 1), generator=g, device="cuda").float())
  x = x.to(dtype)
  kinds = [
      torch.zeros(D),
      torch.full((D,), info.smallest_normal / 8),
      torch.full((D,), -info.max),
      torch.arange(D) - 63.5,                      # halves under a largest of 64.5
      torch.cat((torch.tensor([127.0]), torch.arange(D - 1) / 2 - 31)),  # scale 1: ties to even
      torch.cat((torch.tensor([448.0]), torch.linspace(0, 20, D - 1))),
      torch.cat((torch.tensor([torch.inf]), torch.ones(D - 1))),
      torch.cat((torch.ones(D - 1), torch.tensor([torch.nan]))),
      torch.cat((torch.tensor([info.max]), torch.full((D - 1,), info.smallest_normal / 4))),
  ]
  for i, r in enumerate(kinds):
    if i < T:
      x[0, i, i % 3] = r.to(dtype).cuda()
  return x


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("fmt", FORMATS, ids=str)
@pytest.mark.parametrize("T", [1, 9, 33, 300])
def test_written_rows_are_the_exact_codes(ops, T, fmt, dtype):
  k, v = awkward_rows(T, dtype, 1), awkward_rows(T, dtype, 2).flip(1)
  cache = ft().KVCache.empty(1, T + 3, 3, dtype=fmt)
  for t in (cache.k, cache.v):
    t.view(torch.uint8).fill_(0x5a)
  cache.k_scale.fill_(-7), cache.v_scale.fill_(-7)
  cache.write(k, v, start=ints([2]))
  for rows, scale, x in ((cache.k, cache.k_scale, k), (cache.v, cache.v_scale, v)):
    code, sc = codes_of(x, fmt)
    assert same(rows[:, 2:2 + T], code)
    sc = sc.transpose(1, 2)
    assert torch.equal(torch.isnan(scale[..., 2:2 + T]), torch.isnan(sc))
    # (one division in f32)
    assert ((scale[..., 2:2 + T].double() - sc).abs() <= sc.abs() * 2.0 ** -24).logical_or(torch.isnan(sc)).all()
    for at in (slice(0, 2), slice(2 + T, None)):
      assert (rows[:, at].contiguous().view(torch.uint8) == 0x5a).all() and (scale[..., at] == -7).all()


@pytest.mark.parametrize("fmt", FORMATS, ids=str)
def test_padding_and_rows_outside_the_cache_are_not_written(ops, fmt):
  B, T, H, cap = 6, 70, 2, 80
  g = gen(3)
  k = torch.randn(B, T, H + 1, D, generator=g, device="cuda").half()[:, :, 1:]   # strided
  v = torch.randn(B, H, T, D, generator=g, device="cuda").half().transpose(1, 2)
  start, count = [0, 5, 60, -20, 79, 2 ** 31 - 1], [70, 33, 70, 60, 1, 70]
  for s, c in ((start, count), (start, None), (None, count), (None, [0, -1, 1, 200, 31, 32])):
    cache = ft().KVCache.empty(B, cap, H, dtype=fmt)
    cache.k.view(torch.uint8).fill_(0x11), cache.v.view(torch.uint8).fill_(0x22)
    cache.k_scale.fill_(3), cache.v_scale.fill_(4)
    cache.write(k, v, start=None if s is None else ints(s), count=None if c is None else ints(c))
    for rows, scale, x, byte, was in ((cache.k, cache.k_scale, k, 0x11, 3), (cache.v, cache.v_scale, v, 0x22, 4)):
      code, sc = codes_of(x, fmt)
      want = torch.full((B, cap, H, D), byte, dtype=torch.uint8, device="cuda")
      want_sc = torch.full((B, cap, H), float(was), device="cuda")
      for b in range(B):
        for i in range(min(T, T if c is None else max(c[b], 0))):
          to = (0 if s is None else s[b]) + i
          if 0 <= to < cap:
            want[b, to], want_sc[b, to] = code[b, i].view(torch.uint8), sc[b, i].float()
      assert torch.equal(rows.contiguous().view(torch.uint8), want)
      assert torch.allclose(scale.transpose(1, 2), want_sc, rtol=2.0 ** -23, atol=0)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("fmt", FORMATS, ids=str)
def test_compaction_by_indices(ops, fmt, dtype):
  B, S, H, n = 2, 200, 3, 45
  g = gen(4)
  k, v = (torch.randn(B, S, H, D, generator=g, device="cuda").to(dtype) for _ in range(2))
  idx = torch.randint(0, S, (B, H, n), generator=g, device="cuda", dtype=torch.int32)  # (any order, repeated ones too)
  idx[0, 0, :4] = ints([-5, S, S + 100, S - 1])
  near = idx.long().clamp(0, S - 1).transpose(1, 2)[..., None].expand(-1, -1, -1, D)
  cache = ft().KVCache.empty(B, n, H, dtype=fmt).write(k, v, idx=idx)
  for rows, scale, x in ((cache.k, cache.k_scale, k), (cache.v, cache.v_scale, v)):
    code, sc = codes_of(x.gather(1, near), fmt)
    assert same(rows, code) and torch.allclose(scale.transpose(1, 2).double(), sc, rtol=2.0 ** -23, atol=0)
  # more indices than source rows, onto the end of a cache, some of them real
  idx = torch.randint(0, 7, (B, H, n), generator=g, device="cuda", dtype=torch.int32)
  cache.write(k[:, :7], v[:, :7], idx=idx, start=ints([20, 0]), count=ints([40, 10]))
  code, _ = codes_of(k.gather(1, idx.long().transpose(1, 2)[..., None].expand(-1, -1, -1, D)), fmt)
  assert same(cache.k[0, 20:], code[0, :25]) and same(cache.k[1, :10], code[1, :10])
  old, _ = codes_of(k.gather(1, near), fmt)
  assert same(cache.k[0, :20], old[0, :20]) and same(cache.k[1, 10:], old[1, 10:])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("fmt", FORMATS, ids=str)
def test_reading_back(ops, fmt, dtype):
  B, S, H = 3, 101, 2
  cache = make_cache(B, S, H, fmt, 5)
  cache.k_scale[0, 0, 3], cache.v_scale[1, 1, 7] = torch.nan, 60000.0
  if fmt == torch.float8_e4m3fn:
    cache.k.view(torch.uint8)[2, 5, 1, 9] = 0x7f  # its NaN
  cache.k.view(torch.uint8)[0, 9, 0] = torch.arange(128, dtype=torch.uint8, device="cuda") * 2  # every code
  # f32 products, rounded once: what torch's conversion gives
  want = [(r.float() * s.transpose(1, 2)[..., None]).to(dtype) for r, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]
  eq = lambda a, b: torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(), b.nan_to_num())
  for a, b in zip(cache.read(dtype), want):
    assert a.dtype == dtype and eq(a, b)
  for a, b in zip(cache.read(dtype, length=37), want):
    assert a.shape == (B, 37, H, D) and eq(a, b[:, :37])
  lens = [0, 64, 500]
  real = torch.arange(S, device="cuda")[None] < ints(lens)[:, None]
  for a, b in zip(cache.read(dtype, kv_len=ints(lens)), want):
    assert eq(a, torch.where(real[..., None, None], b, 0.0))
  idx = torch.randint(0, S, (B, H, 50), generator=gen(6), device="cuda", dtype=torch.int32)
  idx[1, 0, :3] = ints([-1, S, 2 ** 31 - 1])
  at = idx.long().clamp(0, S - 1).transpose(1, 2)
  for a, b in zip(cache.read(dtype, idx=idx, kv_len=ints([101, 64, -3])), want):
    g = b.gather(1, at[..., None].expand(-1, -1, -1, D))
    assert eq(a, torch.where((at < ints([101, 64, -3])[:, None, None])[..., None], g, 0.0))


# ------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------
SHAPES = [  # B, Sq, H, Hkv, capacity, lengths
    (1, 1, 1, 1, 1, [1]),
    (3, 1, 4, 2, 130, [1, 64, 130]),
    (2, 1, 8, 8, 65, [65, 17]),
    (2, 1, 32, 8, 1001, [1001, 640]),
    (1, 1, 16, 1, 5000, [4999]),
    (1, 4, 16, 4, 700, [603]),
    (2, 3, 10, 2, 300, [300, 150]),
    (2, 17, 2, 2, 400, [399, 17]),
    (1, 5, 20, 4, 1500, [1400]),
    (1, 130, 6, 2, 600, [555]),
    (2, 300, 2, 1, 900, [300, 801]),
    (1, 2, 128, 1, 260, [255]),
    (1, 64, 5, 1, 2100, [2050]),
]


def q_of(B, Sq, H, dtype, seed, size=1.0):
  return (torch.randn(B, Sq, H, D, generator=gen(seed), device="cuda") * size).to(dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("fmt", [None] + FORMATS, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attention_over_ragged_caches(ops, shape, fmt, dtype):
  B, Sq, H, Hkv, cap, lens = shape
  cache = make_cache(B, cap, Hkv, fmt or dtype, 7, dtype)
  q, n = q_of(B, Sq, H, dtype, 8, 1.5), ints(lens)
  for causal in (True, False):
    got, lse = ops.attn_cache(q, cache, n, causal=causal, return_lse=True)
    check_attention(got, lse, _attention(q, cache, lens, causal), f"causal={causal}")
  assert same(ft().CacheAttn(Hkv, H).forward(q, cache, n), ops.attn_cache(q, cache, n))


# many units and few, of one part or several: B, Sq, H, Hkv, capacity
UNITS = [(150, 1, 2, 1, 70), (400, 1, 4, 1, 40), (100, 2, 8, 4, 90), (75, 4, 16, 2, 300), (60, 4, 16, 4, 100), (20, 4, 16, 4, 800),
         (100, 20, 2, 1, 500), (20, 70, 8, 4, 333), (40, 1, 24, 1, 1700), (9, 1, 16, 8, 1500), (3, 1, 8, 8, 4000), (1, 1, 8, 8, 16000),
         (2, 1, 16, 2, 30000), (1, 2, 5, 5, 20000)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("fmt", [None] + FORMATS, ids=str)
@pytest.mark.parametrize("shape", UNITS, ids=str)
def test_attention_of_many_and_few_units(ops, shape, fmt, dtype):
  B, Sq, H, Hkv, cap = shape
  cache = make_cache(B, cap, Hkv, fmt or dtype, 160, dtype)
  lens = [0 if i % 7 == 3 else cap - 13 * i % cap for i in range(B)]
  q, n = q_of(B, Sq, H, dtype, 161, 1.5), ints(lens)
  got, lse = ops.attn_cache(q, cache, kv_len=n, return_lse=True)
  check_attention(got, lse, _attention(q, cache, lens), "")


@pytest.mark.parametrize("fmt", [None] + FORMATS, ids=str)
@pytest.mark.parametrize("Sq, group", [(1, 4), (4, 1), (9, 4)])
def test_attention_without_lengths_and_with_a_scale(ops, fmt, Sq, group):
  cache = make_cache(2, 333, 2, fmt or torch.bfloat16, 9, torch.bfloat16)
  q = q_of(2, Sq, 2 * group, torch.bfloat16, 10)
  got, lse = ops.attn_cache(q, cache, softmax_scale=0.3, return_lse=True)
  check_attention(got, lse, _attention(q, cache, scale=0.3))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("fmt", [None] + FORMATS, ids=str)
@pytest.mark.parametrize("Sq, group", [(1, 2), (3, 2), (40, 2)])
def test_rows_that_see_nothing_are_zero(ops, Sq, group, fmt, dtype):
  # empty sequences, lengths below and beyond what there is, more new tokens than rows: the first see nothing
  lens = [0, -4, 1, 200, 2 ** 31 - 1, max(Sq - 1, 1)]
  cache = make_cache(6, 100, 1, fmt or dtype, 11, dtype)
  q = q_of(6, Sq, group, dtype, 12)
  for causal in (True, False):
    got, lse = ops.attn_cache(q, cache, ints(lens), causal=causal, return_lse=True)
    want = _attention(q, cache, lens, causal)
    check_attention(got, lse, want)
    assert not got[torch.isinf(want[1]).transpose(1, 2)].any() and torch.isinf(want[1]).any()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("fmt", [None] + FORMATS, ids=str)
@pytest.mark.parametrize("Sq, group", [(1, 4), (2, 8), (33, 2), (150, 1)])
def test_what_lies_behind_a_sequence_does_not_matter(ops, Sq, group, fmt, dtype):
  B, cap, Hkv, lens = 2, 500, 2, [450, 203]
  cache = make_cache(B, cap, Hkv, fmt or dtype, 13, dtype)
  q = q_of(B, Sq, Hkv * group, dtype, 14)
  clean, clean_lse = ops.attn_cache(q, cache, ints(lens), return_lse=True)
  for b, n in enumerate(lens):
    if fmt is None:
      cache.k[b, n:], cache.v[b, n:] = torch.nan, torch.inf
    else:
      cache.k.view(torch.uint8)[b, n:], cache.v.view(torch.uint8)[b, n:] = 0x7f, 0xff
      cache.k_scale[b, :, n:], cache.v_scale[b, :, n:] = torch.inf, torch.nan
  got, lse = ops.attn_cache(q, cache, ints(lens), return_lse=True)
  assert same(got, clean) and same(lse, clean_lse)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("fmt", [None] + FORMATS, ids=str)
@pytest.mark.parametrize("Sq, group", [(1, 4), (30, 2)])
def test_rows_that_are_not_finite_stay_in_their_sequence(ops, Sq, group, fmt, dtype):
  # a NaN in one sequence's seen rows: NaN there as without a cache, nothing elsewhere
  cache = make_cache(3, 200, 2, fmt or dtype, 15, dtype)
  q = q_of(3, Sq, 2 * group, dtype, 16)
  clean = ops.attn_cache(q, cache)
  if fmt is None:
    cache.k[1, 20, 1, 5] = torch.nan
  else:
    cache.k_scale[1, 1, 20] = torch.nan
  got = ops.attn_cache(q, cache)
  assert torch.isnan(got[1, :, group:]).all()
  got[1, :, group:] = clean[1, :, group:]
  assert same(got, clean)


@pytest.mark.parametrize("fmt", [None] + FORMATS, ids=str)
@pytest.mark.parametrize("n, Sq", [(2, 1), (30, 1), (2, 40)])
def test_a_prefix_of_nothing_but_nan(ops, n, Sq, fmt):
  # (every part of it has no maximum; the sum still has to say so)
  prefix, cache = make_cache(2, 300, 2, fmt or torch.float16, 150), make_cache(2 * n, 50, 2, fmt or torch.float16, 151)
  q = q_of(2 * n, Sq, 4, torch.float16, 152)
  clean = ops.attn_prefix(q, prefix, cache)
  (prefix.k if fmt is None else prefix.k_scale)[1].fill_(torch.nan)
  got = ops.attn_prefix(q, prefix, cache)
  assert torch.isnan(got[n:]).all() and same(got[:n], clean[:n])


@pytest.mark.parametrize("fmt", FORMATS, ids=str)
@pytest.mark.parametrize("Sq, group", [(1, 4), (30, 2)])
@pytest.mark.parametrize("spread", [2.0 ** -20, 1.0, 30.0])
def test_scales_that_differ_by_many_powers_of_two(ops, fmt, Sq, group, spread):
  # values 2^-30 to 2^10 times the others' size, in bf16's range but not in f16's
  cache = make_cache(1, 300, 2, fmt, 17, torch.bfloat16, spread)
  cache.v_scale *= torch.exp2(torch.randint(-30, 11, cache.v_scale.shape, generator=gen(18), device="cuda").float())
  q = q_of(1, Sq, 2 * group, torch.bfloat16, 19, min(1 / spread, 64.0))
  check_attention(*ops.attn_cache(q, cache, return_lse=True), _attention(q, cache))


@pytest.mark.parametrize("fmt", [None] + FORMATS, ids=str)
@pytest.mark.parametrize("rows", [(1, 4), (40, 4)], ids=str)
@pytest.mark.parametrize("direction", [1, -1])
def test_logits_that_keep_growing_or_shrinking(ops, fmt, rows, direction):
  # the running maximum moves at every tile, or never after the first
  Sq, group = rows
  cache = make_cache(1, 1500, 1, torch.bfloat16, 20, torch.bfloat16)
  ramp = torch.linspace(-40, 40, 1500, device="cuda") * direction
  k = cache.k + ramp[None, :, None, None] / 8
  c16 = ft().KVCache(k.bfloat16().contiguous(), cache.v)
  if fmt is not None:
    c8 = ft().KVCache.empty(1, 1500, 1, dtype=fmt)
    c8.write(c16.k, c16.v)
    c16 = c8
  q = (q_of(1, Sq, group, torch.bfloat16, 21) * 0.05 + 0.5).bfloat16()
  check_attention(*ops.attn_cache(q, c16, return_lse=True), _attention(q, c16))


@pytest.mark.parametrize("fmt", [torch.bfloat16] + FORMATS, ids=str)
@pytest.mark.parametrize("Sq", [1, 20])
def test_strides_and_layouts(ops, fmt, Sq):
  # token-major rows, a slice of a larger cache's heads and rows, q and out as slices of wider tensors
  B, S, Hkv, group = 2, 220, 2, 4
  big = make_cache(B + 1, S + 9, Hkv + 2, fmt, 22, torch.bfloat16, token_major=True)
  at = lambda t: t[1:, 4:4 + S, 1:1 + Hkv]
  sc = lambda t: None if t is None else t[1:, 1:1 + Hkv, 4:4 + S]
  part = ft().KVCache(at(big.k), at(big.v), sc(big.k_scale), sc(big.v_scale))
  wide = q_of(B, Sq, Hkv * group + 3, torch.bfloat16, 23)
  q = wide[:, :, 3:]
  room = torch.full((B, Sq + 2, Hkv * group + 1, D), 9.0, dtype=torch.bfloat16, device="cuda")
  got = ops.attn_cache(q, part, ints([S, 101]), out=room[:, 1:1 + Sq, 1:])
  check_attention(got, None, _attention(q, part, [S, 101]))
  assert (room[:, 0] == 9).all() and (room[:, 1 + Sq:] == 9).all() and (room[:, :, 0] == 9).all()
  dense = ft().KVCache(*(None if t is None else t.contiguous() for t in (part.k, part.v, part.k_scale, part.v_scale)))
  assert same(ops.attn_cache(q.contiguous(), dense, ints([S, 101])), got)


def test_caches_longer_than_32_bit_offsets(ops):
  # the second sequence's rows lie beyond 2^32 elements
  S, H = 1_300_000, 14
  cache = ft().KVCache(*[torch.zeros(2, S, H, D, dtype=torch.int8, device="cuda") for _ in range(2)],
                       *[torch.zeros(2, H, S, device="cuda") for _ in range(2)])
  g = gen(24)
  n = 130
  k, v = (torch.randn(2, n, H, D, generator=g, device="cuda").half() for _ in range(2))
  far = S - n
  cache.write(k, v, start=ints([far, far]))
  code, _ = codes_of(k, torch.int8)
  assert same(cache.k[:, far:], code)
  tail = ft().KVCache(cache.k[:, far:], cache.v[:, far:],
                      *[torch.nn.functional.pad(t[..., far:], (0, 2))[..., :n] for t in (cache.k_scale, cache.v_scale)])
  back = cache.read(torch.float16, idx=torch.arange(far, S, dtype=torch.int32, device="cuda").expand(2, H, n).contiguous())
  assert same(back[0], tail.read(torch.float16)[0])
  # (the rows in front are zeros and their scales too: logits 0 and values 0, weight S - n of them)
  for Sq in (1, 20):
    q = q_of(2, Sq, H, torch.float16, 25)
    out, lse = ops.attn_cache(q, tail, causal=False, return_lse=True)
    got, far_lse = ops.attn_cache(q, cache, causal=False, return_lse=True)
    want = out.double() * torch.exp2(lse.double() - torch.logaddexp2(lse.double(), torch.tensor(far, device="cuda").double().log2())).transpose(1, 2)[..., None]
    scale = want.abs().amax()
    assert (got.double() - want).abs().max() <= scale * 2.0 ** -8 + 2.0 ** -24  # (f16 weights 2^-11 here, there and in `out`; subnormal outputs)
  del cache, tail
  torch.cuda.empty_cache()


PREFIXES = [  # G, n (sequences to a prefix), Sq, H, Hkv, P, prefix lengths, capacity
    (1, 1, 1, 2, 1, 1, [1], 1),
    (1, 4, 1, 8, 2, 300, [300], 40),
    (1, 16, 1, 4, 4, 1000, [999], 65),
    (1, 5, 1, 16, 4, 513, [513], 130),
    (2, 3, 2, 8, 4, 257, [257, 100], 33),
    (3, 2, 1, 5, 1, 700, [700, 0, 1], 64),
    (1, 70, 1, 4, 1, 1200, [1111], 20),
    (2, 33, 1, 10, 2, 400, [399, 385], 70),
    (1, 3, 140, 2, 1, 600, [600], 150),
    (2, 40, 4, 8, 8, 260, [260, 129], 12),
    (1, 130, 1, 2, 1, 4000, [4000], 300),
]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("fmts", [(None, None), (torch.int8, torch.int8), (torch.float8_e4m3fn, torch.float8_e4m3fn),
                                  (None, torch.int8), (torch.float8_e4m3fn, None)], ids=str)
@pytest.mark.parametrize("shape", PREFIXES, ids=str)
def test_attention_over_shared_prefixes(ops, shape, fmts, dtype):
  G, n, Sq, H, Hkv, P, plens, cap = shape
  B = G * n
  prefix = make_cache(G, P, Hkv, fmts[0] or dtype, 30, dtype)
  cache = make_cache(B, cap, Hkv, fmts[1] or dtype, 31, dtype)
  lens = [max(min(Sq, cap), cap - 7 * i % cap) for i in range(B)]
  q = q_of(B, Sq, H, dtype, 32, 1.5)
  for causal in (True, False):
    got, lse = ops.attn_prefix(q, prefix, cache, ints(lens), ints(plens), causal=causal, return_lse=True)
    check_attention(got, lse, _attention(q, cache, lens, causal, prefix, plens), f"causal={causal}")
  assert same(ft().PrefixAttn(Hkv, H).forward(q, prefix, cache, ints(lens), ints(plens)),
              ops.attn_prefix(q, prefix, cache, ints(lens), ints(plens)))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("fmt", [None] + FORMATS, ids=str)
@pytest.mark.parametrize("n", [3, 50])
def test_prefix_garbage_and_empty_parts(ops, n, fmt, dtype):
  # nothing of a sequence's own, nothing of the prefix, nothing at all, and garbage behind either
  G, H, Hkv, P, cap = 2, 4, 2, 333, 50
  prefix, cache = make_cache(G, P, Hkv, fmt or dtype, 33, dtype), make_cache(G * n, cap, Hkv, fmt or dtype, 34, dtype)
  plens, lens = [200, 0], [0 if i % 3 == 0 else 10 + i % 30 for i in range(G * n)]
  q = q_of(G * n, 1, H, dtype, 35)
  clean, lse = ops.attn_prefix(q, prefix, cache, ints(lens), ints(plens), return_lse=True)
  want = _attention(q, cache, lens, True, prefix, plens)
  check_attention(clean, lse, want)
  assert torch.isinf(want[1]).any()
  for c, ls in ((prefix, plens), (cache, lens)):
    for b, m in enumerate(ls):
      if fmt is None:
        c.k[b, m:], c.v[b, m:] = torch.inf, torch.nan
      else:
        c.k.view(torch.uint8)[b, m:], c.v.view(torch.uint8)[b, m:] = 0xff, 0x7f
        c.k_scale[b, :, m:], c.v_scale[b, :, m:] = torch.nan, torch.inf
  got, lse2 = ops.attn_prefix(q, prefix, cache, ints(lens), ints(plens), return_lse=True)
  assert same(got, clean) and same(lse2, lse)


# ------------------------------------------------------------------------------------------
# calls as a program makes them
# ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", [torch.bfloat16] + FORMATS, ids=str)
def test_same_bits_on_every_call_and_on_another_stream(ops, fmt):
  prefix, cache = make_cache(1, 2000, 2, fmt, 40, torch.bfloat16), make_cache(24, 200, 2, fmt, 41, torch.bfloat16)
  q, chunk = q_of(24, 1, 8, torch.bfloat16, 42), q_of(24, 21, 8, torch.bfloat16, 43)
  n = ints([200 - 5 * i for i in range(24)])
  first = [ops.attn_prefix(q, prefix, cache, n), ops.attn_cache(q, cache, n), ops.attn_cache(chunk, cache, n)]
  side = torch.cuda.Stream()
  for _ in range(5):
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
      other = [ops.attn_prefix(q, prefix, cache, n), ops.attn_cache(q, cache, n), ops.attn_cache(chunk, cache, n)]
    here = [ops.attn_prefix(q, prefix, cache, n), ops.attn_cache(q, cache, n), ops.attn_cache(chunk, cache, n)]
    side.synchronize()
    for a, b, c in zip(first, here, other):
      assert same(a, b) and same(a, c)


@pytest.mark.parametrize("fmt", FORMATS, ids=str)
def test_graphs_replay_with_new_contents_and_lengths(ops, fmt):
  # two captured steps (write, attention) over one cache, replayed in turn as a generation would, rows and lengths
  # changed between replays
  B, H, Hkv, cap = 3, 8, 2, 90
  prefix = make_cache(1, 300, Hkv, fmt, 44)
  caches = [ft().KVCache.empty(B, cap, Hkv, dtype=fmt) for _ in range(2)]
  plain = [ft().KVCache.empty(B, cap, Hkv, dtype=fmt) for _ in range(2)]
  for c in caches + plain:  # (rows that no step writes are seen too)
    for t in (c.k.view(torch.uint8), c.v.view(torch.uint8), c.k_scale, c.v_scale):
      t.zero_()
  k, v, q = (torch.zeros(B, 1, h, D, dtype=torch.float16, device="cuda") for h in (Hkv, Hkv, H))
  start, n = ints([0, 0, 0]), ints([1, 1, 1])

  def step(c):
    c.write(k, v, start=start)
    return ops.attn_cache(q, c, n), ops.attn_prefix(q, prefix, c, n)

  for c in caches:
    step(c)
  torch.cuda.synchronize()
  graphs = []
  for c in caches:
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
      out = step(c)
    graphs.append((g, out))
  for t in range(12):
    for x, seed in ((k, 1), (v, 2), (q, 3)):
      x.copy_(torch.randn(x.shape, generator=gen(100 * t + seed), device="cuda"))
    start.copy_(ints([t, 2 * t, 5 * t + 3])), n.copy_(start + 1)
    for (g, _) in graphs:
      g.replay()
    for (_, out), c in zip(graphs, plain):
      for a, b in zip(out, step(c)):
        assert same(a, b)


def test_graphed_calls_of_the_cases_over_caches(ops):
  # a call recorded for a cache, its scales and lengths by their addresses; an absent length is another call than a present one
  from flashtensor_b200.host import GraphedCall
  q, n, cache = q_of(3, 1, 8, torch.float16, 170), ints([70, 1, 33]), make_cache(3, 70, 2, torch.int8, 171)
  prefix, wide = make_cache(1, 200, 2, torch.float16, 172), make_cache(3, 70, 2, torch.float16, 173)
  for model, calls in ((ft().CacheAttn(2, 8), [(q, cache, n), (q, cache), (q, cache, None), (q, wide, n)]),
                       (ft().PrefixAttn(2, 8), [(q, prefix, cache, n), (q, prefix, cache, None, ints([150])), (q, prefix, wide, n)])):
    graphed = GraphedCall(model)
    for _ in range(2):
      for args in calls:
        assert same(graphed(*args), model(*args))
    n.copy_(ints([20, 68, 4]))
    for args in calls:
      assert same(graphed(*args), model(*args))
  assert len(graphed.cache) == 3


@pytest.mark.parametrize("fmt", [None] + FORMATS, ids=str)
@pytest.mark.parametrize("shape", [(1, 1, 8, 2, 900, 0), (160, 1, 4, 1, 60, 0), (30, 20, 8, 4, 300, 0), (2, 90, 8, 2, 700, 0),
                                   (40, 1, 8, 2, 50, 400), (4, 1, 8, 2, 90, 600)], ids=str)
def test_the_output_may_take_the_place_of_q(ops, shape, fmt):
  B, Sq, H, Hkv, cap, P = shape
  cache = make_cache(B, cap, Hkv, fmt or torch.bfloat16, 180, torch.bfloat16)
  q = q_of(B, Sq, H, torch.bfloat16, 181)
  if P:
    prefix = make_cache(1, P, Hkv, fmt or torch.bfloat16, 182, torch.bfloat16)
    call = lambda x, out: ops.attn_prefix(x, prefix, cache, out=out)
  else:
    call = lambda x, out: ops.attn_cache(x, cache, out=out)
  want, x = call(q, None), q.clone()
  assert call(x, x).data_ptr() == x.data_ptr() and same(x, want)


def test_no_store_lands_outside_outputs_or_workspace(ops):
  from test_parity_gpu import _Banded
  from flashtensor_b200 import _lib
  lib = _lib.load()
  for shape in ((1, 3, 1, 8, 2, 300, 77), (2, 20, 1, 10, 2, 700, 65), (1, 1, 45, 6, 2, 900, 333), (1, 1, 1, 4, 1, 5000, 900)):
    G, n, Sq, H, Hkv, P, cap = shape
    for fmt in (torch.bfloat16, *FORMATS):
      mem = _Banded(96 << 20)
      prefix, cache = make_cache(G, P, Hkv, fmt, 50, torch.bfloat16), make_cache(G * n, cap, Hkv, fmt, 51, torch.bfloat16)
      q = q_of(G * n, Sq, H, torch.bfloat16, 52)
      for pre in (None, prefix):
        out, lse = mem.take(q.shape, torch.bfloat16), mem.take((G * n, H, Sq), torch.float32)
        c = lambda x: _lib.KvCache(*(ops._desc(t) for t in ((None,) * 4 if x is None else (x.k, x.v, x.k_scale, x.v_scale))))
        p = _lib.AttnCacheParams(ops._desc(q), ops._desc(out), ops._desc(lse), c(cache), _lib.Tensor(), c(pre), _lib.Tensor(),
                                 0.0, 1, None, 0)
        need = ctypes.c_size_t(0)
        assert lib.asuka_b200_attn_cache_workspace_bytes(ctypes.byref(p), ctypes.byref(need)) == 0
        ws = mem.take((max(need.value, 256),), torch.uint8)
        assert ws.data_ptr() % 256 == 0
        p.workspace, p.workspace_bytes = ws.data_ptr(), need.value
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        assert lib.asuka_b200_attn_cache(ctypes.byref(p), stream) == 0
        torch.cuda.synchronize()
        assert mem.bands_untouched()
        ref = ops.attn_cache(q, cache) if pre is None else ops.attn_prefix(q, pre, cache)
        assert same(out, ref)
        if need.value > 0:
          p.workspace_bytes = need.value - 1
          assert lib.asuka_b200_attn_cache(ctypes.byref(p), stream) == -6
          p.workspace, p.workspace_bytes = ws.data_ptr() + 16, need.value
          assert lib.asuka_b200_attn_cache(ctypes.byref(p), stream) == -5
          p.workspace = None
          assert lib.asuka_b200_attn_cache(ctypes.byref(p), stream) == -1
      if fmt in FORMATS:
        rows = [mem.take((G * n, Hkv, cap, D), torch.uint8).view(fmt).transpose(1, 2) for _ in range(2)]
        scales = [mem.take((G * n, Hkv, (cap + 3) // 4 * 4), torch.float32) for _ in range(2)]
        to = ft().KVCache(*rows, *(t[..., :cap] for t in scales))
        new = torch.randn(G * n, 45, Hkv, D, device="cuda").bfloat16()
        for start in (-40, 0, cap - 3, cap, 2 ** 31 - 1):
          to.write(new, new, start=ints([start] * (G * n)))
        torch.cuda.synchronize()
        assert mem.bands_untouched()
        for t in scales:
          assert (t[..., cap:].contiguous().view(torch.uint8) == 0xa5).all()


@pytest.mark.parametrize("fmt", FORMATS, ids=str)
def test_a_generation_behind_a_selection(ops, fmt):
  # H2O's prefill and selection, its keys compacted into an 8-bit cache, then steps that write their own row and
  # attend to all of them; four samples go on from a second, whole prompt as their shared prefix
  H, S, keep, recent, steps = 4, 600, 100, 50, 5
  g = gen(60)
  rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").half()
  q, k, v = rnd(1, S, H, D), rnd(1, S, H, D), rnd(1, S, H, D)
  _, _, idx = ft().H2O(H, H).select(q, k, v, keep, recent)
  n0 = keep + recent
  cache = ft().KVCache.empty(1, n0 + steps, H, dtype=fmt).write(k, v, idx=idx)
  kept = idx.long().transpose(1, 2)[..., None].expand(-1, -1, -1, D)
  rows = [[codes_of(x.gather(1, kept), fmt)] for x in (k, v)]
  model = ft().CacheAttn(H, H)
  filled = ints([n0])
  for t in range(steps):
    new = rnd(1, 1, H, D), rnd(1, 1, H, D), rnd(1, 1, H, D)
    cache.write(new[1], new[2], start=filled)
    filled += 1
    got = model(new[0], cache, filled)
    for r, x in zip(rows, new[1:]):
      r.append(codes_of(x, fmt))
    ref = ft().KVCache(*[torch.cat([c.view(torch.uint8) for c, _ in r], 1).view(fmt) for r in rows],
                       *[torch.cat([s for _, s in r], 1).transpose(1, 2) for r in rows])
    check_attention(got, None, _attention(new[0], ref))
  prompt = ft().KVCache.empty(1, S, H, dtype=fmt).write(k, v)
  own = ft().KVCache.empty(4, steps, H, dtype=fmt)
  model = ft().PrefixAttn(H, H)
  for t in range(steps):
    new = rnd(4, 1, H, D), rnd(4, 1, H, D), rnd(4, 1, H, D)
    own.write(new[1], new[2], start=ints([t] * 4))
    got = model(new[0], prompt, own, ints([t + 1] * 4))
    check_attention(got, None, _attention(new[0], own, [t + 1] * 4, True, prompt))
  # what the cache holds reads back within half a code's step of what was written
  back = prompt.read(torch.float16)[0].double()
  step = 0.5 / 127 if fmt == torch.int8 else 2.0 ** -4
  size = k.double().abs().amax(-1, keepdim=True) if fmt == torch.int8 else k.double().abs() + 2.0 ** -9 * k.double().abs().amax(-1, keepdim=True)
  assert ((back - k.double()).abs() <= size * step * 1.001 + back.abs() * 2.0 ** -11).all()


def test_refusals_on_the_device(ops):
  from flashtensor_b200 import _lib
  cache = ft().KVCache.empty(2, 64, 2)
  q = torch.zeros(2, 1, 4, D, dtype=torch.float16, device="cuda")
  bad = [
      ("BAD_DTYPE", lambda: ops.attn_cache(q.float(), cache)),
      ("BAD_DTYPE", lambda: ops.attn_cache(q, ft().KVCache.empty(2, 64, 2, dtype=torch.bfloat16))),
      ("BAD_DTYPE", lambda: ops.attn_cache(q, cache, torch.tensor([1.0, 2.0], device="cuda"))),
      ("BAD_SHAPE", lambda: ops.attn_cache(q, cache, ints([1]))),
      ("BAD_SHAPE", lambda: ops.attn_cache(q[:1], cache)),
      ("BAD_SHAPE", lambda: ops.attn_cache(q[:, :, :3], cache)),
      ("BAD_SHAPE", lambda: ops.attn_prefix(q, ft().KVCache.empty(3, 64, 2), cache)),
      ("BAD_SHAPE", lambda: ops.attn_prefix(q, ft().KVCache.empty(1, 64, 4), cache)),
      ("NULL_POINTER", lambda: ops.attn_cache(q, ft().KVCache(cache.k, cache.v))),
      ("BAD_ARGUMENT", lambda: ops.attn_cache(q, ft().KVCache(q, q, cache.k_scale, cache.v_scale))),
      ("BAD_ARGUMENT", lambda: ops.attn_cache(q, cache, softmax_scale=float("inf"))),
      ("BAD_SHAPE", lambda: ops.quant_kv(q, q, cache)),
      ("BAD_DTYPE", lambda: ops.quant_kv(q[:, :, :2], q[:, :, :2], ft().KVCache(q[:, :, :2], q[:, :, :2]))),
      ("BAD_SHAPE", lambda: ops.quant_kv(q[:, :, :2], q[:, :, :2], cache, idx=torch.zeros(2, 3, 4, dtype=torch.int32, device="cuda"))),
      ("BAD_DTYPE", lambda: ops.dequant_kv(cache, torch.float32)),
      ("BAD_SHAPE", lambda: ops.dequant_kv(cache, length=65)),
      ("BAD_SHAPE", lambda: ops.dequant_kv(cache, length=1 << 45)),  # (refused ahead of the allocation)
      ("BAD_ARGUMENT", lambda: ops.dequant_kv(cache, length=-2)),
      ("BAD_ARGUMENT", lambda: ops.dequant_kv(cache, length=3, idx=torch.zeros(2, 2, 4, dtype=torch.int32, device="cuda"))),
  ]
  for code, call in bad:
    with pytest.raises(_lib.AsukaError, match=code):
      call()
  for call in (lambda: ops.attn_cache(q, cache, torch.tensor([1, 2], dtype=torch.int32)),
               lambda: ops.quant_kv(q[:, :, :2].cpu(), q[:, :, :2], cache)):
    with pytest.raises(RuntimeError, match="no CPU path"):
      call()
  with pytest.raises(RuntimeError, match="key/value heads"):
    ft().CacheAttn(4, 4).forward(q, cache)
  with pytest.raises(TypeError):
    ops.dequant_kv(cache, "bfloat16")


# ------------------------------------------------------------------------------------------
# the ends of the range
# ------------------------------------------------------------------------------------------
# streamed (a cluster to a unit, dealt out), one query tile of many rows, two: B, Sq, group
FORMS = [(1, 1, 4), (50, 1, 4), (2, 20, 2), (2, 100, 2)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("fmt", [None] + FORMATS, ids=str)
@pytest.mark.parametrize("n", [1, 129, 296, 352, 384])
@pytest.mark.parametrize("B, Sq, group", FORMS)
def test_query_rows_of_zeros_and_tiny_ones(ops, B, Sq, group, n, fmt, dtype):
  # logits of 0 or nearly: the mean of what the row sees, whatever lies behind the sequence or the mask (there are keys of zeros too)
  cache = make_cache(B, 400, 2, fmt or dtype, 190, dtype)
  cache.k[:, 300:] = 0
  if fmt is not None:
    cache.k_scale[:, :, 300:] = 2.0 ** -100
  q = q_of(B, Sq, 2 * group, dtype, 191)
  q[0] = 0
  q[-1, :, ::2] *= 0 if dtype == torch.float16 else 2.0 ** -90
  q[-1, Sq // 2:, 1::2] *= 2.0 ** -20
  prefix = make_cache(1, 330, 2, fmt or dtype, 192, dtype)
  lens = [n] * B
  for causal in (True, False):
    check_attention(*ops.attn_cache(q, cache, ints(lens), causal=causal, return_lse=True), _attention(q, cache, lens, causal), f"causal={causal}")
    check_attention(*ops.attn_prefix(q, prefix, cache, ints(lens), causal=causal, return_lse=True),
                    _attention(q, cache, lens, causal, prefix), f"prefix, causal={causal}")


def test_empty_indices_lengths_and_counts_are_refused(ops):
  # a tensor of no elements has no address, which is how an absent one is told: a selection of nothing would write every row
  from flashtensor_b200 import _lib
  cache = ft().KVCache.empty(2, 64, 2)
  for t in (cache.k, cache.v):
    t.view(torch.uint8).fill_(0x5a)
  q, new = (torch.ones(2, 3, h, D, dtype=torch.float16, device="cuda") for h in (4, 2))
  none, no_idx = ints([]), torch.empty(2, 2, 0, dtype=torch.int32, device="cuda")
  for call in (lambda: cache.write(new, new, idx=no_idx), lambda: cache.write(new, new, start=none), lambda: cache.write(new, new, count=none),
               lambda: cache.read(torch.float16, idx=no_idx), lambda: cache.read(torch.float16, kv_len=none), lambda: ops.attn_cache(q, cache, none),
               lambda: ops.attn_prefix(q, cache, cache, None, none), lambda: ops.attn_prefix(q, cache, cache, none)):
    with pytest.raises(_lib.AsukaError):
      call()
  assert (cache.k.contiguous().view(torch.uint8) == 0x5a).all() and (cache.v.contiguous().view(torch.uint8) == 0x5a).all()


def test_graphed_calls_whose_first_input_is_a_cache_or_absent(ops):
  from flashtensor_b200.host import GraphedCall
  cache, q, n = make_cache(2, 60, 2, torch.int8, 200), q_of(2, 1, 8, torch.float16, 201), ints([60, 7])
  attend = GraphedCall(lambda c, x, m: ops.attn_cache(x, c, m))
  last = GraphedCall(lambda m, x, c: ops.attn_cache(x, c, m))
  for _ in range(2):
    assert same(attend(cache, q, n), ops.attn_cache(q, cache, n))
    assert same(last(None, q, cache), ops.attn_cache(q, cache))
  # a write, whose rows and place change between replays
  k, v = (torch.zeros(2, 1, 2, D, dtype=torch.float16, device="cuda") for _ in range(2))
  write = GraphedCall(lambda c, *rest: c.write(*rest).k)
  plain = ft().KVCache(*[t.clone(memory_format=torch.preserve_format) for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)])
  for t in range(3):
    for x, seed in ((k, 202), (v, 203)):
      x.copy_(torch.randn(x.shape, generator=gen(seed + 10 * t), device="cuda"))
    n.copy_(ints([3 * t, 50 + t]))
    write(cache, k, v, n)
    plain.write(k, v, start=n)
    assert same(cache.k, plain.k) and same(cache.v, plain.v) and torch.equal(cache.v_scale, plain.v_scale)


# 2^125: values up to 2^127 of bf16's largest 2^128, scales 2^120; 2^-60: scales down to 2^-69
@pytest.mark.parametrize("fmt", FORMATS, ids=str)
@pytest.mark.parametrize("order", ["large", "small", "large first", "small first", "mixed", "mixed by 32", "zeros"])
@pytest.mark.parametrize("B, Sq, group", [*FORMS, (3, 4, 4)])
def test_values_at_the_ends_of_the_range(ops, B, Sq, group, order, fmt):
  # what the weights' sum holds may not depend on the size of the values, which is in the exponentials' reference
  S, P = 1100, 700
  def sized(c):
    n = c.k.shape[1]
    size = torch.full(c.v_scale.shape, 2.0 ** 125, device="cuda")
    j, g = torch.arange(n, device="cuda"), gen(210)
    if order == "small":
      size[:] = 2.0 ** -60
    elif order == "large first":
      size[..., 400:] = 1.0
    elif order == "small first":
      size[..., :400] = 2.0 ** -60
    elif order == "mixed":
      size = torch.exp2(125.0 * torch.randint(0, 2, size.shape, generator=g, device="cuda"))
    elif order == "mixed by 32":
      size = torch.exp2(torch.tensor([125.0, 0.0, -60.0], device="cuda")[(j // 32) % 3]).expand_as(size)
    elif order == "zeros":  # (rows of zeros have the smallest scale there is)
      size[..., 100:] = 1e30
      c.v.view(torch.uint8)[:, 200:] = 0
      c.v_scale[..., 200:], size[..., 200:] = 2.0 ** -100, 1.0
    c.v_scale *= size
    return c
  prefix, cache = sized(make_cache(1, P, 2, fmt, 211, torch.bfloat16)), sized(make_cache(B, S, 2, fmt, 212, torch.bfloat16))
  q, lens = q_of(B, Sq, 2 * group, torch.bfloat16, 213, 2.0), [S - 31 * i % 500 for i in range(B)]
  check_attention(*ops.attn_cache(q, cache, ints(lens), return_lse=True), _attention(q, cache, lens))
  check_attention(*ops.attn_prefix(q, prefix, cache, ints(lens), return_lse=True), _attention(q, cache, lens, True, prefix), "prefix")
  plain = make_cache(1, P, 2, torch.bfloat16, 214, torch.bfloat16)  # (values of ordinary size, without scales, ahead of them)
  check_attention(*ops.attn_prefix(q, plain, cache, ints(lens), return_lse=True), _attention(q, cache, lens, True, plain), "16-bit prefix")


@pytest.mark.parametrize("fmt", [None] + FORMATS, ids=str)
@pytest.mark.parametrize("B, S, group", [(1, 1000, 1), (3, 900, 2), (1, 1500, 4)])
def test_a_whole_prompt_and_its_keys_that_no_row_of_a_block_sees(ops, B, S, group, fmt):
  # a value that is not finite makes NaN of what sees it, and (with a weight of 0) may of rows of its block of query tiles; rows of the
  # blocks ahead do not touch it
  cache = make_cache(B, S, 2, fmt or torch.float16, 220)
  q = q_of(B, S, 2 * group, torch.float16, 221)
  clean, lse = ops.attn_cache(q, cache, return_lse=True)
  check_attention(clean, lse, _attention(q, cache))
  at = S - 20
  if fmt is None:
    cache.v[:, at] = torch.nan
  else:
    cache.v_scale[:, :, at] = torch.nan
  got, got_lse = ops.attn_cache(q, cache, return_lse=True)
  assert torch.isnan(got[:, at:]).all()
  ahead = at - 256 // group - 128   # (a block is 256 rows of a key/value head, a tile of keys 128)
  assert same(got[:, :ahead], clean[:, :ahead]) and same(got_lse, lse)


# The 2-norm of an f16 output's error over its own.  A rounding to a step of 2^-10 of values evenly spread over a power of two is off by
# 2^-10 / sqrt(12) against sqrt(7 / 3): 2^-10 / sqrt(28) = 1.85e-4 in the mean square, and with weights of that error and values that are
# independent of each other an output's is as large.  So: the weights and the output; where codes times scales are rounded (two query
# tiles over 8 bits), the values too, and the keys, whose error in a logit is 1.85e-4 |q| |k| of a component each, 1 with normal ones.
# A fifth more than the root of the sum of squares.
@pytest.mark.parametrize("fmt", [None] + FORMATS, ids=str)
@pytest.mark.parametrize("B, Sq, group, tiles", [(1, 1, 4, 0), (50, 1, 4, 0), (3, 2, 8, 0), (8, 20, 2, 1), (3, 100, 1, 1), (2, 100, 2, 2), (1, 300, 2, 2)])
def test_f16_outputs_are_as_near_as_their_roundings(ops, B, Sq, group, tiles, fmt):
  cache = make_cache(B, 2000, 2, fmt or torch.float16, 230)
  q, lens = q_of(B, Sq, 2 * group, torch.float16, 231), [2000 - 17 * i for i in range(B)]
  got = ops.attn_cache(q, cache, ints(lens)).double()
  want = _attention(q, cache, lens)[0]
  roundings = 2 if fmt is None or tiles < 2 else 4
  assert (got - want).norm() <= 1.2 * (roundings / 28) ** 0.5 * 2.0 ** -10 * want.norm()
