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

from ._lib import DTYPE_CODES, check, lib, on_device, pack_i64x3, pack_i64x10, ptr, stream_handle

GROUP = 32
_TYPES = (torch.bfloat16, torch.float16, torch.float32)
_entries: dict = {}  # bytes of a row, by head size


def entry_bytes(head_dim: int) -> int:
    """Bytes of a row: head_dim / 2 codes and head_dim / 32 scales, rounded up to 4."""
    n = _entries.get(head_dim)
    if n is None:
        n = int(lib().psk_mxfp4_entry_bytes(int(head_dim)))
        check(n if n < 0 else 0, "mxfp4 entry size")
        _entries[head_dim] = n
    return n


def check_cache(cache: torch.Tensor, num_heads: int, head_dim: int, name: str) -> None:
    shape = cache.shape
    assert cache.dtype == torch.uint8 and len(shape) == 4, \
        f"{name} must be uint8 [num_blocks, block_size, kv_heads, entry_bytes]"
    entry = _entries.get(head_dim) or entry_bytes(head_dim)
    assert shape[2] == num_heads and shape[3] == entry, (
        f"{name} has rows {tuple(shape[2:])}, want ({num_heads}, {entry}) for heads of {head_dim}"
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
    assert len(key.shape) == 3 and len(value.shape) == 3
    assert key.is_cuda, "key must be on a GPU"
    tokens, heads, dim = key.shape
    dtype, device = key.dtype, key.device
    assert value.shape[1:] == (heads, dim) and value.dtype == dtype
    assert dtype in _TYPES, f"a 4-bit cache takes bf16, fp16 or fp32 rows, not {dtype}"
    ks, vs = key.stride(), value.stride()
    assert (ks[2] == 1 and vs[2] == 1) or key.numel() == 0, "heads must have unit inner stride"
    check_cache(key_cache, heads, dim, "key_cache")
    check_cache(value_cache, heads, dim, "value_cache")
    blocks, page = key_cache.shape[:2]
    assert value_cache.shape == key_cache.shape
    for t in (value, key_cache, value_cache, slot_mapping):
        assert t.device == device, "all tensors must share the key's device"
    assert slot_mapping.dtype == torch.int64 and len(slot_mapping.shape) == 1, "slot_mapping must be int64 [tokens]"
    n = slot_mapping.shape[0]
    assert n <= 1 or slot_mapping.stride(0) == 1, "slot_mapping needs unit stride"
    assert n <= min(tokens, value.shape[0]), f"slot_mapping has {n} entries for {tokens} tokens"
    with on_device(device):
        st = lib().psk_reshape_and_cache_mxfp4(
            key.data_ptr(), value.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), slot_mapping.data_ptr(), n, heads,
            dim, page, blocks, pack_i64x10(*ks[:2], *vs[:2], *key_cache.stride()[:3], *value_cache.stride()[:3]),
            DTYPE_CODES[dtype], stream_handle(device),
        )
    if st:
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
    assert src_cache.is_cuda, "src_cache must be on a GPU"
    device, dtype = src_cache.device, dst.dtype
    assert len(dst.shape) == 3 and dtype in _TYPES, "dst must be [T, H, D] in bf16, fp16 or fp32"
    T, heads, dim = dst.shape
    check_cache(src_cache, heads, dim, "src_cache")
    blocks, page = src_cache.shape[:2]
    ds, cs = dst.stride(), src_cache.stride()
    assert (ds[2] == 1 and (ds[1] == dim or heads == 1)) or dst.numel() == 0, "dst rows must be contiguous"
    assert len(block_table.shape) == 2 and block_table.dtype == torch.int32, "block_table must be int32 [sequences, pages]"
    rows, width = block_table.shape
    assert width <= 1 or block_table.stride(1) == 1, "block_table needs unit last stride"
    assert cu_seq_lens.dtype == torch.int32 and len(cu_seq_lens.shape) == 1 and cu_seq_lens.is_contiguous()
    seqs = cu_seq_lens.shape[0] - 1
    B = seqs if batch_size is None else int(batch_size)
    assert 0 <= B <= seqs and B <= rows
    if seq_starts is not None:
        assert seq_starts.dtype == torch.int32 and seq_starts.is_contiguous() and seq_starts.shape[0] >= B
    assert (src_cache_v is None) == (dst_v is None), "a second cache needs a second destination"
    if src_cache_v is not None:
        assert src_cache_v.shape == src_cache.shape and src_cache_v.stride() == cs and src_cache_v.dtype == torch.uint8
        assert dst_v.shape == dst.shape and dst_v.stride() == ds and dst_v.dtype == dtype
    for t in (dst, block_table, cu_seq_lens, seq_starts, src_cache_v, dst_v):
        assert t is None or t.device == device, "all tensors must share the cache's device"
    with on_device(device):
        st = lib().psk_gather_mxfp4(
            src_cache.data_ptr(), ptr(src_cache_v), dst.data_ptr(), ptr(dst_v), block_table.data_ptr(), cu_seq_lens.data_ptr(),
            ptr(seq_starts), B, block_table.stride(0), width, T, heads, dim, page, blocks, pack_i64x3(*cs[:3]),
            max(ds[0], heads * dim) if T <= 1 else ds[0], DTYPE_CODES[dtype], stream_handle(device),
        )
    if st:
        check(st, "gather_mxfp4")
