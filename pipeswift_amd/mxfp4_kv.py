"""A KV cache of 4 bits: rows in microscaled 4-bit floats, written and read back.

The reference's caches are bf16 or FP8 (pipeswift/utils/fp8_kv.py:24-25); this one
takes 4.25 bits an element.  It is a uint8 tensor in the GQA cache's layout with
the row of a head in place of its elements:

    [layers, num_blocks, 2, block_size, kv_heads, entry_bytes(head_dim)]

    [0, D/2)            E2M1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives),
                        element 2i in the low half of byte i, 2i + 1 in the high half
    [D/2, D/2 + D/32)   one scale byte for 32 elements: 2^(byte - 127)
    zeros up to a multiple of 4 bytes (68 bytes for D = 128, 36 for 64)

A group's scale is the smallest power of two s >= 2^-126 with max |x| < 7 s, so that
no value is clipped and each is off by at most half a step (a quarter of it, or s / 4
below s).  A group that holds a NaN or an infinity reads as NaN; zeros stay zeros.

Every operation that moves rows or pages takes it as it is: ``copy_blocks``,
``CopyEngine``, ``evict_tokens``, ``commit_draft_tokens``.
``impl_utils.append_kv_cache`` writes it where the cache is uint8,
``rotary.norm_rope_and_cache`` in the pass that norms and rotates the keys, and
``attention.paged_mxfp4_attention`` (``flash_attn_varlen_func`` with it) reads it.
Both functions here run on the caller's current stream and allocate nothing.
"""

from __future__ import annotations

import torch

from ._lib import check, dtype_code, i64_array, lib, on_device, ptr, stream_handle

GROUP = 32
_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def entry_bytes(head_dim: int) -> int:
    """Bytes of a row: head_dim / 2 codes and head_dim / 32 scales, rounded up to 4."""
    n = int(lib().psk_mxfp4_entry_bytes(int(head_dim)))
    check(n if n < 0 else 0, "mxfp4 entry size")
    return n


def check_cache(cache: torch.Tensor, num_heads: int, head_dim: int, name: str) -> None:
    assert cache.dtype == torch.uint8 and cache.ndim == 4, \
        f"{name} must be uint8 [num_blocks, block_size, kv_heads, entry_bytes]"
    entry = entry_bytes(head_dim)
    assert cache.shape[2] == num_heads and cache.shape[3] == entry, (
        f"{name} has rows {tuple(cache.shape[2:])}, want ({num_heads}, {entry}) for heads of {head_dim}"
    )
    assert cache.stride(3) == 1, f"{name} needs unit last stride"


def reshape_and_cache_mxfp4(
    key: torch.Tensor,
    value: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
) -> None:
    """key/value [N, H, D] (bf16, fp16 or fp32, unit last stride) quantized into
    key_cache/value_cache, uint8 [num_blocks, block_size, H, entry_bytes(D)]:
    ``reshape_and_cache_flash``'s counterpart for the 4-bit cache.  Token t goes to
    slot ``slot_mapping[t]`` (int64); negative and out-of-range slots are skipped."""
    assert key.ndim == 3 and value.ndim == 3
    assert key.is_cuda and value.is_cuda and slot_mapping.is_cuda
    heads, dim = key.shape[1], key.shape[2]
    assert value.shape[1:] == key.shape[1:] and value.dtype == key.dtype
    assert key.dtype in _TYPES, f"a 4-bit cache takes bf16, fp16 or fp32 rows, not {key.dtype}"
    assert (key.stride(2) == 1 and value.stride(2) == 1) or key.numel() == 0, "heads must have unit inner stride"
    check_cache(key_cache, heads, dim, "key_cache")
    check_cache(value_cache, heads, dim, "value_cache")
    assert value_cache.shape == key_cache.shape
    device = key_cache.device
    assert key.device == device and value.device == device and value_cache.device == device
    assert slot_mapping.dtype == torch.int64 and slot_mapping.ndim == 1 and slot_mapping.is_contiguous()
    assert slot_mapping.device == device, "slot_mapping must live on the cache's device"
    n = slot_mapping.shape[0]
    assert n <= min(key.shape[0], value.shape[0]), f"slot_mapping has {n} entries for {key.shape[0]} tokens"
    with on_device(device):
        st = lib().psk_reshape_and_cache_mxfp4(
            ptr(key), ptr(value), ptr(key_cache), ptr(value_cache), ptr(slot_mapping), n, heads, dim, key_cache.shape[1],
            key_cache.shape[0], i64_array(key.stride()), i64_array(value.stride()), i64_array(key_cache.stride()),
            i64_array(value_cache.stride()), dtype_code(key.dtype), stream_handle(device),
        )
    check(st, "reshape_and_cache_mxfp4")


def gather_mxfp4(
    src_cache: torch.Tensor,
    dst: torch.Tensor,
    block_table: torch.Tensor,
    cu_seq_lens: torch.Tensor,
    batch_size: int | None = None,
    seq_starts: torch.Tensor | None = None,
    src_cache_v: torch.Tensor | None = None,
    dst_v: torch.Tensor | None = None,
) -> None:
    """Read each sequence's 4-bit rows into contiguous ``dst`` rows [T, H, D] (bf16
    and fp32: the exact values; fp16: rounded): ``cache_ops.gather_cache``'s
    counterpart, with its arguments.  For t in [cu[b], cu[b+1]) and p = seq_starts[b]
    + t - cu[b], ``dst[t]`` is the row of ``block_table[b, p // block_size]``, ``p %
    block_size``; zeros where there is no such page.  Rows at or past
    cu[batch_size] stay as they were.  ``src_cache_v`` / ``dst_v`` read a second cache
    of the same geometry in the same launch."""
    assert src_cache.is_cuda and dst.is_cuda and block_table.is_cuda and cu_seq_lens.is_cuda
    device = src_cache.device
    assert dst.ndim == 3 and dst.dtype in _TYPES, "dst must be [T, H, D] in bf16, fp16 or fp32"
    heads, dim = dst.shape[1], dst.shape[2]
    check_cache(src_cache, heads, dim, "src_cache")
    assert (dst.stride(2) == 1 and (dst.stride(1) == dim or heads == 1)) or dst.numel() == 0, "dst rows must be contiguous"
    assert block_table.dtype == torch.int32 and block_table.ndim == 2
    assert block_table.stride(1) == 1 or block_table.shape[1] <= 1, "block_table needs unit last stride"
    assert cu_seq_lens.dtype == torch.int32 and cu_seq_lens.ndim == 1 and cu_seq_lens.is_contiguous()
    B = cu_seq_lens.shape[0] - 1 if batch_size is None else int(batch_size)
    assert 0 <= B <= cu_seq_lens.shape[0] - 1 and B <= block_table.shape[0]
    if seq_starts is not None:
        assert seq_starts.dtype == torch.int32 and seq_starts.is_contiguous() and seq_starts.shape[0] >= B
    assert (src_cache_v is None) == (dst_v is None), "a second cache needs a second destination"
    if src_cache_v is not None:
        assert src_cache_v.shape == src_cache.shape and src_cache_v.stride() == src_cache.stride()
        assert src_cache_v.dtype == src_cache.dtype
        assert dst_v.shape == dst.shape and dst_v.stride() == dst.stride() and dst_v.dtype == dst.dtype
    for t in (dst, block_table, cu_seq_lens, seq_starts, src_cache_v, dst_v):
        assert t is None or t.device == device, "all tensors must share the cache's device"
    T = dst.shape[0]
    with on_device(device):
        st = lib().psk_gather_mxfp4(
            ptr(src_cache), ptr(src_cache_v), ptr(dst), ptr(dst_v), ptr(block_table), ptr(cu_seq_lens), ptr(seq_starts), B,
            block_table.stride(0), block_table.shape[1], T, heads, dim, src_cache.shape[1], src_cache.shape[0],
            i64_array(src_cache.stride()), max(dst.stride(0), heads * dim) if T <= 1 else dst.stride(0),
            dtype_code(dst.dtype), stream_handle(device),
        )
    check(st, "gather_mxfp4")
