"""A generation's KV cache: the keys and values of B sequences, in 16 bits or quantised to 8.

The reference ends with the prefill, its scores and (here) a selection; this is where the kept or new rows go.
"""
import torch

from . import ops

FORMATS = (torch.int8, torch.float8_e4m3fn, torch.float16, torch.bfloat16)


class KVCache:
  """``k``, ``v`` [B, capacity, Hkv, 128] and, in 8 bits, ``k_scale``, ``v_scale`` [B, Hkv, capacity] f32: a row (a
  token's key or value of one head) stands for its codes times its scale.  The tensors may be any the kernels
  take (base and strides multiples of 16 bytes, unit stride along the last axis); ``empty`` makes them with the rows of a
  head side by side, so that a head is read as one stream.

  How many rows of each sequence are filled is the caller's to keep (int32 [B] on the device, one for all
  layers): ``write`` takes the row to start at, attention and ``read`` the number of rows.  Both are for 8 bits; the
  rows of a 16-bit cache are the values themselves, to be assigned to (``k[:, a:b] = ...``, ``k.scatter_``).
  """
  __slots__ = ("k", "v", "k_scale", "v_scale")

  def __init__(self, k, v, k_scale=None, v_scale=None):
    self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale

  @classmethod
  def empty(cls, batch_size, capacity, kv_head_num=32, head_dim=128, dtype=torch.int8, device=None):
    if head_dim != 128:
      raise ValueError("the sm_100a kernels are built for head_dim = 128")
    if dtype not in FORMATS:
      raise ValueError(f"a cache is one of {FORMATS}, not {dtype}")
    if min(batch_size, capacity, kv_head_num) < 1:
      raise ValueError("a cache has at least one sequence, row and head")
    device = torch.cuda.current_device() if device is None else device
    rows = [torch.empty((batch_size, kv_head_num, capacity, head_dim), dtype=dtype, device=device).transpose(1, 2)
            for _ in range(2)]
    if dtype.itemsize == 2:
      return cls(*rows)
    padded = (capacity + 3) // 4 * 4  # (a head's scales start on a 16-byte boundary)
    scales = [torch.empty((batch_size, kv_head_num, padded), dtype=torch.float32, device=device)[..., :capacity]
              for _ in range(2)]
    return cls(*rows, *scales)

  @property
  def capacity(self):
    return self.k.shape[1]

  def write(self, k, v, start=None, count=None, idx=None):
    """``ops.quant_kv`` into this (8-bit) cache."""
    ops.quant_kv(k, v, self, start=start, count=count, idx=idx)
    return self

  def read(self, dtype=torch.bfloat16, idx=None, kv_len=None, length=None):
    """``ops.dequant_kv`` of this (8-bit) cache: (k, v)."""
    return ops.dequant_kv(self, dtype, idx=idx, kv_len=kv_len, length=length)
