"""CPU: what the cache's entry points refuse before anything is launched, and the classes above them."""
import ctypes

import pytest
import torch

import flashtensor_b200 as ft
from flashtensor_b200 import _lib
from test_host_logic import _t

I8, E4M3, F32, I32, BF16 = _lib.I8, _lib.E4M3, _lib.F32, _lib.I32, _lib.BF16


def _cache(N=2, S=64, H=2, dtype=I8, **kw):
  rows = _t((N, S, H, 128), dtype=dtype)
  scale = _t((N, H, S), dtype=F32) if dtype in (I8, E4M3) else _lib.Tensor()
  return _lib.KvCache(kw.get("k", rows), kw.get("v", rows), kw.get("ks", scale), kw.get("vs", scale))


def _attn(lib, **kw):
  q = kw.get("q", _t((2, 1, 4, 128)))
  p = _lib.AttnCacheParams(q, kw.get("out", _t((2, 1, 4, 128))), kw.get("lse", _lib.Tensor()), kw.get("cache", _cache()),
                           kw.get("len", _lib.Tensor()), kw.get("prefix", _lib.KvCache()), kw.get("plen", _lib.Tensor()),
                           kw.get("scale", 0.0), 1, None, 0)
  return lib.asuka_b200_attn_cache(ctypes.byref(p), None)


def test_attention_refuses(built_lib):
  lib = _lib.load()
  assert lib.asuka_b200_attn_cache(None, None) == -1
  call = lambda **kw: _attn(lib, **kw)
  assert call(q=_t((2, 1, 4, 128), ptr=0)) == -1
  assert call(q=_t((2, 1, 4, 128), dtype=F32)) == -2
  assert call(q=_t((2, 1, 4, 64))) == -3
  assert call(q=_t((2, 1, 4, 128), ptr=0x1008)) == -5
  assert call(q=_t((2, 1, 4, 128), strides=(512, 512, 128, 2))) == -4
  assert call(q=_t((3, 1, 4, 128))) == -3                                   # sequences
  assert call(q=_t((2, 1, 3, 128))) == -3                                   # heads
  assert call(q=_t((2, 1, 2 * 129, 128)), out=_t((2, 1, 2 * 129, 128))) == -11
  assert call(q=_t((2, 0, 4, 128))) == -3
  assert call(cache=_cache(dtype=BF16)) == -2                               # 16 bits of another type than q
  assert call(cache=_cache(dtype=_lib.U8)) == -2
  assert call(cache=_cache(k=_t((2, 64, 2, 128), dtype=I8, ptr=0))) == -1
  assert call(cache=_cache(v=_t((2, 64, 2, 128), dtype=E4M3))) == -2
  assert call(cache=_cache(v=_t((2, 65, 2, 128), dtype=I8))) == -3
  assert call(cache=_cache(k=_t((2, 64, 2, 128), dtype=I8, strides=(16400, 264, 136, 1)))) == -4   # not 16-byte multiples
  assert call(cache=_cache(k=_t((2, 64, 2, 128), dtype=I8, strides=(1 << 40, 256, 128, 1)))) == -11
  assert call(cache=_cache(k=_t((2, 64, 2, 128), dtype=I8, strides=(-16384, 256, 128, 1)))) == -4
  assert call(cache=_cache(k=_t((2, 64, 2, 128), dtype=I8, strides=(0, 256, 128, 1)))) == -4
  assert call(cache=_cache(ks=_lib.Tensor())) == -1
  assert call(cache=_cache(vs=_t((2, 2, 64), dtype=I32))) == -2
  assert call(cache=_cache(vs=_t((2, 64, 2), dtype=F32))) == -3
  assert call(cache=_cache(vs=_t((2, 2, 64), dtype=F32, strides=(130, 65, 1)))) == -4
  assert call(cache=_cache(vs=_t((2, 2, 64), dtype=F32, strides=(2, 1, 4)))) == -4
  assert call(cache=_cache(vs=_t((2, 2, 64), dtype=F32, ptr=0x1004))) == -5
  assert call(cache=_cache(dtype=_lib.F16, ks=_t((2, 2, 64), dtype=F32))) == -10    # scales of 16 bits
  assert call(len=_t((3,), dtype=I32)) == -3
  assert call(len=_t((2,), dtype=F32)) == -2
  assert call(len=_t((2,), dtype=I32, strides=(2,))) == -4
  assert call(len=_t((2,), dtype=I32, ptr=0x1002)) == -5
  assert call(plen=_t((2,), dtype=I32)) == -10                              # lengths of no prefix
  assert call(prefix=_cache(N=3)) == -3
  assert call(prefix=_cache(N=4)) == -3                                     # more prefixes than sequences
  assert call(prefix=_cache(H=1)) == -3
  assert call(prefix=_cache(N=1), plen=_t((2,), dtype=I32)) == -3
  assert call(scale=float("nan")) == -10
  assert call(out=_t((2, 1, 2, 128))) == -3
  assert call(out=_t((2, 1, 4, 128), dtype=BF16)) == -2
  assert call(out=_t((2, 1, 4, 128), ptr=0)) == -1
  assert call(lse=_t((2, 1, 4), dtype=F32)) == -3
  need = ctypes.c_size_t(0)
  assert lib.asuka_b200_attn_cache_workspace_bytes(None, ctypes.byref(need)) == -1
  p = _lib.AttnCacheParams()
  assert lib.asuka_b200_attn_cache_workspace_bytes(ctypes.byref(p), None) == -1
  assert lib.asuka_b200_attn_cache_workspace_bytes(ctypes.byref(p), ctypes.byref(need)) == -1


def test_write_and_read_refuse(built_lib):
  lib = _lib.load()
  x = _t((2, 5, 2, 128))
  no = _lib.Tensor()
  put = lambda **kw: lib.asuka_b200_quant_kv(ctypes.byref(_lib.QuantKvParams(
      kw.get("k", x), kw.get("v", x), kw.get("idx", no), kw.get("start", no), kw.get("count", no), kw.get("cache", _cache()))), None)
  assert lib.asuka_b200_quant_kv(None, None) == -1
  assert put(k=_t((2, 5, 2, 128), ptr=0)) == -1
  assert put(k=_t((2, 5, 2, 128), dtype=F32)) == -2
  assert put(v=_t((2, 5, 2, 128), dtype=BF16)) == -2
  assert put(v=_t((2, 6, 2, 128))) == -3
  assert put(k=_t((2, 5, 2, 128), ptr=0x1004)) == -5
  assert put(k=_t((2, 0, 2, 128)), v=_t((2, 0, 2, 128))) == -3
  assert put(cache=_cache(dtype=_lib.F16)) == -2
  assert put(cache=_cache(N=3)) == -3
  assert put(cache=_cache(H=4)) == -3
  assert put(idx=_t((2, 3, 4), dtype=I32)) == -3
  assert put(idx=_t((2, 2, 4), dtype=F32)) == -2
  assert put(idx=_t((2, 2, 4), dtype=I32, strides=(16, 8, 1))) == -4
  assert put(start=_t((1,), dtype=I32)) == -3
  assert put(count=_t((2, 1), dtype=I32)) == -3
  out = _t((2, 64, 2, 128))
  get = lambda **kw: lib.asuka_b200_dequant_kv(ctypes.byref(_lib.DequantKvParams(
      kw.get("cache", _cache()), kw.get("idx", no), kw.get("len", no), kw.get("ko", out), kw.get("vo", out))), None)
  assert lib.asuka_b200_dequant_kv(None, None) == -1
  assert get(cache=_cache(dtype=BF16)) == -2
  assert get(ko=_t((2, 64, 2, 128), dtype=F32)) == -2
  assert get(vo=_t((2, 64, 2, 128), dtype=BF16)) == -2
  assert get(ko=_t((2, 65, 2, 128)), vo=_t((2, 65, 2, 128))) == -3          # more rows than there are
  assert get(ko=_t((1, 64, 2, 128))) == -3
  assert get(vo=_t((2, 63, 2, 128))) == -3
  assert get(idx=_t((2, 2, 9), dtype=I32)) == -3                            # nine indices, 64 rows
  assert get(len=_t((3,), dtype=I32)) == -3


def test_a_tensor_of_no_elements_is_not_an_absent_one(built_lib):
  # (it has no address either)
  lib = _lib.load()
  x, no, none, no_idx = _t((2, 5, 2, 128)), _lib.Tensor(), _t((0,), dtype=I32, ptr=0), _t((2, 2, 0), dtype=I32, ptr=0)
  for idx, start, count in ((no_idx, no, no), (no, none, no), (no, no, none)):
    assert lib.asuka_b200_quant_kv(ctypes.byref(_lib.QuantKvParams(x, x, idx, start, count, _cache())), None) == -3
  out = _t((2, 64, 2, 128))
  for idx, n in ((no_idx, no), (no, none)):
    assert lib.asuka_b200_dequant_kv(ctypes.byref(_lib.DequantKvParams(_cache(), idx, n, out, out)), None) == -3
  assert _attn(lib, len=none) == -3
  assert _attn(lib, prefix=_cache(N=1), plen=none) == -3


def test_operators_refuse_tensors_on_the_host(built_lib):
  from flashtensor_b200 import ops
  cache = ft.KVCache.empty(1, 8, 2, device="cpu")
  q = torch.zeros(1, 1, 4, 128, dtype=torch.float16)
  for call in (lambda: ops.attn_cache(q, cache), lambda: ops.attn_prefix(q, cache, cache), lambda: cache.read(),
               lambda: cache.write(q[:, :, :2], q[:, :, :2])):
    with pytest.raises(RuntimeError, match="no CPU path"):
      call()
  with pytest.raises(TypeError):
    ops.attn_cache(q, ft.KVCache(None, None))


def test_an_empty_cache_has_the_layout_the_kernels_want():
  c = ft.KVCache.empty(3, 101, 4, dtype=torch.float8_e4m3fn, device="cpu")
  assert c.k.shape == c.v.shape == (3, 101, 4, 128) and c.k.dtype == torch.float8_e4m3fn and c.capacity == 101
  assert c.k.stride() == (4 * 101 * 128, 128, 101 * 128, 1)                 # a head's rows side by side
  assert c.k_scale.shape == (3, 4, 101) and c.k_scale.stride() == (416, 104, 1) and c.k_scale.dtype == torch.float32
  c = ft.KVCache.empty(1, 5, 1, dtype=torch.bfloat16, device="cpu")
  assert c.k_scale is None and c.v_scale is None and c.v.dtype == torch.bfloat16
  for bad in (dict(dtype=torch.float32), dict(head_dim=64), dict(capacity=0)):
    with pytest.raises(ValueError):
      ft.KVCache.empty(**{"batch_size": 1, "capacity": 4, "device": "cpu", **bad})


def test_cases_keep_their_bookkeeping():
  a, p = ft.CacheAttn(2, 8), ft.PrefixAttn(2, 8)
  assert a.input_names == ["q", "cache"] and p.input_names == ["q", "prefix", "cache"]
  ins = p.prepare(6, 1, 40, device="cpu")["input"]
  assert ins["q"].shape == (6, 1, 8, 128) and ins["prefix"].k.shape == (1, 40, 2, 128) and ins["cache"].k.shape == (6, 1, 2, 128)
  assert a.get_flops(6, 1, 40) == 4 * 6 * 8 * 40 * 128 and p.get_flops(6, 1, 40) == 4 * 6 * 8 * 41 * 128
  count = lambda x: x.q.numel() if hasattr(x, "q") else x.numel() if torch.is_tensor(x) else x.k.numel() + x.v.numel()
  assert p.get_mem_size(6, 1, 40) == sum(map(count, ins.values())) + ins["q"].numel()
  ins = a.prepare(6, 1, 40, device="cpu")["input"]
  assert a.get_mem_size(6, 1, 40) == sum(map(count, ins.values())) + ins["q"].numel()
  with pytest.raises(AssertionError):
    ft.CacheAttn(3, 8)


def test_the_factory_finds_the_cases_over_caches():
  a, p = ft.get_model("CacheAttn", kv_head_num=2, head_num=8, causal=False), ft.get_model("PrefixAttn", kv_head_num=2, head_num=8)
  assert type(a) is ft.CacheAttn and not a.causal and type(p) is ft.PrefixAttn and p.head_num == 8
  assert type(ft.get_model("Attn")) is ft.Attn
  with pytest.raises(KeyError):
    ft.get_model("KVCache")


def test_structures_match_the_header(tmp_path):
  import os
  import shutil
  import subprocess
  cc = shutil.which("gcc") or shutil.which("cc")
  if cc is None:
    pytest.skip("no C compiler")
  blocks = {
      "asuka_kv_cache": (_lib.KvCache, ["k", "v", "k_scale", "v_scale"]),
      "asuka_quant_kv_params": (_lib.QuantKvParams, ["idx", "start", "count", "cache"]),
      "asuka_dequant_kv_params": (_lib.DequantKvParams, ["cache", "idx", "len", "k_out", "v_out"]),
      "asuka_attn_cache_params": (_lib.AttnCacheParams, ["q", "lse", "cache", "len", "prefix", "prefix_len", "softmax_scale",
                                                        "causal", "workspace", "workspace_bytes"]),
  }
  root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
  lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "asuka_b200.h"', "int main(void) {"]
  for name, (_, fields) in blocks.items():
    lines.append(f'  printf("{name} %zu\\n", sizeof({name}));')
    lines += [f'  printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f in fields]
  (tmp_path / "layout.c").write_text("\n".join(lines + ["  return 0;", "}"]))
  subprocess.run([cc, "-I", os.path.join(root, "include"), str(tmp_path / "layout.c"), "-o", str(tmp_path / "layout")], check=True)
  got = dict(l.split() for l in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.splitlines())
  for name, (cls, fields) in blocks.items():
    assert int(got[name]) == ctypes.sizeof(cls), name
    for f in fields:
      assert int(got[f"{name}.{f}"]) == getattr(cls, f).offset, f"{name}.{f}"
