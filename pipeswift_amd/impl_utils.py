"""Thin callers of the append, as the attention layers use them.

Mirrors ``append_kv_cache`` / ``append_mla_kv_cache`` of
pipeswift/utils/impl_utils.py:303-325: early return on an empty batch, the
layer's K/V views of ``kv_cache_info.kv_cache`` (GQA) or the layer of
``mla_cache_tensor`` with a 1-head axis (MLA), and ``kv_cache_info.slot_mapping``.
The optional FP8 scales of ``KVCacheInfo`` (one element, or one per layer)
are passed through.  A uint8 ``mla_cache_tensor`` holds tile-scaled FP8 latent
entries (``mla_fp8``), which the append quantizes itself (no per-tensor scale), and
a uint8 ``kv_cache`` holds 4-bit rows (``mxfp4_kv``) likewise.
``norm_rope_append_kv_cache`` is the append with the layer's norms and rotation of q
and k in the same pass.
"""

from __future__ import annotations

import torch

from .metadata import KVCacheInfo, coalesced_to_cuda  # noqa: F401  (re-exported, impl_utils.py:340)
from .mla_fp8 import concat_and_cache_mla_fp8_tiles
from .mxfp4_kv import reshape_and_cache_mxfp4
from .reshape_and_cache import reshape_and_cache_flash, reshape_and_cache_flash_diffkv
from .rotary import norm_rope_and_cache


def _layer_scale(scale, layer_idx):
    if scale is None:
        return None
    return scale if scale.numel() == 1 else scale[layer_idx: layer_idx + 1]


def append_kv_cache(key, value, kv_cache_info: KVCacheInfo = None, layer_idx: int = 0):
    if key.shape[0] == 0:
        return
    k_cache, v_cache = kv_cache_info.kv_cache[0][layer_idx], kv_cache_info.kv_cache[1][layer_idx]
    if k_cache.dtype == torch.uint8:
        reshape_and_cache_mxfp4(key, value, k_cache, v_cache, kv_cache_info.slot_mapping)
        return
    reshape_and_cache_flash(
        key,
        value,
        k_cache,
        v_cache,
        kv_cache_info.slot_mapping,
        _layer_scale(kv_cache_info.k_scale, layer_idx),
        _layer_scale(kv_cache_info.v_scale, layer_idx),
    )


def norm_rope_append_kv_cache(query, key, value, positions, cos_sin, q_weight=None, k_weight=None, eps=1e-6, sections=None,
                              interleaved=False, kv_cache_info: KVCacheInfo = None, layer_idx: int = 0, q_out=None):
    """query [N, Hq, D] and key [N, Hkv, D] normed and rotated (``rotary.norm_rope``),
    key and value appended to the layer's cache, whatever its type; returns the query."""
    k_cache, v_cache = kv_cache_info.kv_cache[0][layer_idx], kv_cache_info.kv_cache[1][layer_idx]
    scales = None, None
    if k_cache.dtype != torch.uint8:  # (4-bit rows have their own)
        scales = _layer_scale(kv_cache_info.k_scale, layer_idx), _layer_scale(kv_cache_info.v_scale, layer_idx)
    return norm_rope_and_cache(
        query, key, value, k_cache, v_cache, kv_cache_info.slot_mapping, positions, cos_sin, q_weight, k_weight, eps,
        sections, interleaved, *scales, q_out)


def append_mla_kv_cache(ckv, kpe, kv_cache_info: KVCacheInfo = None, layer_idx: int = 0):
    if ckv.shape[0] == 0:
        return
    cache = kv_cache_info.mla_cache_tensor[layer_idx]
    if cache.dtype == torch.uint8:
        concat_and_cache_mla_fp8_tiles(ckv, kpe, cache, kv_cache_info.slot_mapping)
        return
    reshape_and_cache_flash_diffkv(
        ckv.unsqueeze(1),
        kpe.unsqueeze(1),
        kv_cache_info.mla_cache_tensor[layer_idx].unsqueeze(2),
        kv_cache_info.slot_mapping,
        _layer_scale(kv_cache_info.k_scale, layer_idx),
    )
