"""MI355X-native paged KV-cache data path for PipeSwift.

Hand-written gfx950 HIP kernels behind a C ABI (include/pipeswift_kv.h,
libpipeswift_kv.so), with the reference's Python cache API on top:

  reshape_and_cache   reshape_and_cache_flash / _diffkv (+ the triton_* names)
  impl_utils          append_kv_cache / append_mla_kv_cache
  metadata            KVCacheInfo, prepare_kv_info (slot_mapping, page_table)
  cudagraph           static metadata for graph replay
  cache_ops           gather_cache, copy_blocks, evict_tokens, commit_draft_tokens, compute_kv_scales
  rotary              norm_rope, norm_rope_and_cache: head norms and rotation, with the append
  mxfp4_kv            the 4-bit cache: reshape_and_cache_mxfp4, gather_mxfp4
  attention           paged attention over FP8 (decode, prefill, drafted trees) and 4-bit caches, and the weights it gave
  copy_engine         CopyEngine / CopyHandle (DRAM L2 offload, swap_blocks)
  fp8_kv              FP8 constants, flag and scale helpers
"""

from .cache_ops import commit_draft_tokens, compute_kv_scales, copy_blocks, evict_tokens, gather_cache
from .impl_utils import append_kv_cache, append_mla_kv_cache
from .metadata import KVCacheInfo, prepare_kv_info
from .reshape_and_cache import (
    reshape_and_cache_flash,
    reshape_and_cache_flash_diffkv,
    triton_reshape_and_cache_flash,
    triton_reshape_and_cache_flash_diffkv,
)

__all__ = [
    "KVCacheInfo",
    "append_kv_cache",
    "append_mla_kv_cache",
    "commit_draft_tokens",
    "compute_kv_scales",
    "copy_blocks",
    "evict_tokens",
    "gather_cache",
    "prepare_kv_info",
    "reshape_and_cache_flash",
    "reshape_and_cache_flash_diffkv",
    "triton_reshape_and_cache_flash",
    "triton_reshape_and_cache_flash_diffkv",
]
