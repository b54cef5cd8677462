"""flashtensor_b200: hand-written sm_100a kernels for the fused attention programs of
FlashTensor/Asuka (plain causal attention and its Gemma-2 / SnapKV / CORM siblings, H2O, Keyformer,
RoCo, SimA, EA), behind the reference's per-case callables and back-end plug-in interface, and what a
generation needs behind them: a KV cache in 16 or 8 bits and attention over it and over shared prefixes.  The
CUDA library is mandatory: importing the operator layer without it raises."""
from . import _lib
from .builder import B200Builder, Builder
from .cache import KVCache
from .cases import (CASES, EA, Attn, CacheAttn, Corm, Gemma2, H2O, KeyFormer, PrefixAttn, RoCo, SimA, SnapKV,
                    get_model)

__all__ = ["KVCache", "CacheAttn", "PrefixAttn", "EA", "Attn", "Gemma2", "SnapKV", "Corm", "H2O", "KeyFormer", "RoCo", "SimA", "CASES", "get_model", "Builder",
           "B200Builder", "_lib"]
