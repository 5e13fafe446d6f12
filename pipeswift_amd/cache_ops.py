"""Block gather, copy_blocks, token eviction and draft commits, and the per-tensor
FP8 scale, on gfx950 HIP kernels.

None of these has a counterpart in the reference (wsjdsg/PipeSwift):
  * its attention kernels read the paged cache in place through the page table
    (pipeswift/llms/layers/attention.py:189-211), so there is no gather;
  * its prefix cache shares whole pages by refcount and remaps a duplicate page
    instead of copying it (pipeswift/engine/block_manager.py:723-780, 841-877),
    so there is no copy_blocks;
  * its FP8 KV cache uses a fixed scale of 1.0 (pipeswift/utils/fp8_kv.py:1-3).
They follow vLLM's conventions for the same operations and are pinned by the
closed forms in their docstrings.  Nor does it evict single tokens or verify
drafted trees: ``evict_tokens`` and ``commit_draft_tokens`` are this build's own.
"""

from __future__ import annotations

import math
import threading

import numpy as np
import torch

from ._lib import check, distinct, dtype_code, i64_array, lib, on_device, overlap, ptr, stream_handle

FP8_E4M3_MAX = 448.0


# --------------------------------------------------------------------------- #
# gather
# --------------------------------------------------------------------------- #


def _row_len(cache: torch.Tensor) -> int:
    """Elements per slot row; the row (dims 2..) must be contiguous."""
    row = 1
    expect = 1
    for dim in range(cache.ndim - 1, 1, -1):
        assert cache.stride(dim) == expect or cache.shape[dim] == 1, (
            f"cache rows must be contiguous beyond dim 1 (strides {cache.stride()})"
        )
        expect *= cache.shape[dim]
        row *= cache.shape[dim]
    return row


def gather_cache(
    src_cache: torch.Tensor,
    dst: torch.Tensor,
    block_table: torch.Tensor,
    cu_seq_lens: torch.Tensor,
    batch_size: int | None = None,
    seq_starts: torch.Tensor | None = None,
    scale: torch.Tensor | None = None,
    src_cache_v: torch.Tensor | None = None,
    dst_v: torch.Tensor | None = None,
) -> None:
    """Copy each sequence's paged rows into contiguous ``dst`` rows.

    src_cache [num_blocks, block_size, *row] (row contiguous; e.g. the K view
    [P, ps, H, D] of the fused [L, P, 2, ps, H, D] cache), dst [T, *row],
    block_table int32 [B, W], cu_seq_lens int32 [B + 1], seq_starts int32 [B]
    (optional first position gathered per sequence).  For t in
    [cu[b], cu[b+1]) and p = seq_starts[b] + t - cu[b]:
    ``dst[t] = src_cache[block_table[b, p // block_size], p % block_size]``.
    A block id outside the cache, or a p beyond the table row, gives a zero
    row.  With an fp8 cache and a bf16/fp16/fp32 ``dst`` each element is
    ``round(float(q) * scale)`` (scale 1.0 when None).  ``src_cache_v``/``dst_v``
    gather a second cache of the same geometry (V) in the same launch.
    """
    assert src_cache.is_cuda and dst.is_cuda and block_table.is_cuda and cu_seq_lens.is_cuda
    device = src_cache.device
    assert src_cache.ndim >= 3, "src_cache must be [num_blocks, block_size, ...]"
    row = _row_len(src_cache)
    assert dst.ndim >= 2 and math.prod(dst.shape[1:]) == row, "dst rows must match the cache rows"
    assert dst[0].is_contiguous() if dst.shape[0] else True, "dst rows must be contiguous"
    assert block_table.dtype == torch.int32 and block_table.ndim == 2 and block_table.is_contiguous()
    assert cu_seq_lens.dtype == torch.int32 and cu_seq_lens.is_contiguous()
    B = cu_seq_lens.shape[0] - 1 if batch_size is None else int(batch_size)
    assert 0 <= B <= cu_seq_lens.shape[0] - 1 and B <= block_table.shape[0]
    if seq_starts is not None:
        assert seq_starts.dtype == torch.int32 and seq_starts.is_contiguous() and seq_starts.shape[0] >= B
    is_dequant = src_cache.dtype != dst.dtype
    if is_dequant:
        assert src_cache.dtype == torch.float8_e4m3fn, "dtype change is only defined for an fp8 cache"
    else:
        assert scale is None, "scale only applies to an fp8 -> float gather"
    if scale is not None:
        assert scale.dtype == torch.float32 and scale.numel() == 1 and scale.device == device
    if src_cache_v is not None or dst_v is not None:
        assert src_cache_v is not None and dst_v is not None
        assert src_cache_v.shape == src_cache.shape and src_cache_v.stride() == src_cache.stride()
        assert src_cache_v.dtype == src_cache.dtype
        assert dst_v.shape == dst.shape and dst_v.stride() == dst.stride() and dst_v.dtype == dst.dtype
    for t in (dst, block_table, cu_seq_lens, seq_starts, scale, src_cache_v, dst_v):
        assert t is None or t.device == device, "all tensors must share the cache's device"

    status = lib().psk_gather_cache(
        ptr(src_cache), ptr(src_cache_v), ptr(dst), ptr(dst_v), ptr(block_table), ptr(cu_seq_lens),
        ptr(seq_starts), B, block_table.stride(0), dst.shape[0], row, src_cache.shape[1], src_cache.shape[0],
        src_cache.stride(0), src_cache.stride(1), dst.stride(0),
        dtype_code(src_cache.dtype), dtype_code(dst.dtype), ptr(scale), stream_handle(device),
    )
    check(status, "gather_cache")


# --------------------------------------------------------------------------- #
# copy_blocks
# --------------------------------------------------------------------------- #


def validate_block_mapping(mapping: np.ndarray, num_blocks: int) -> None:
    """Snapshot preconditions: ids in range, unique destinations, destinations
    disjoint from sources.  Raises AssertionError."""
    m = np.asarray(mapping, dtype=np.int64).reshape(-1, 2)
    if len(m) == 0:
        return
    bad = np.flatnonzero(((m < 0) | (m >= num_blocks)).any(axis=1))
    assert len(bad) == 0, f"block ids out of range [0, {num_blocks}): {m[bad[:8]].tolist()}"
    assert len(np.unique(m[:, 1])) == len(m), "duplicate destination block"
    clash = np.isin(m[:, 1], m[:, 0])
    assert not clash.any(), f"destination blocks that are also sources: {m[clash, 1][:8].tolist()}"


def _slab(cache: torch.Tensor):
    """(num_layers, layer_stride, block_stride, block_bytes) in bytes for a
    layered cache [L, P, ...] whose (layer, page) slab is contiguous."""
    assert cache.ndim >= 3, "caches for copy_blocks are layered: [num_layers, num_blocks, ...]"
    es = cache.element_size()
    expect = 1
    for dim in range(cache.ndim - 1, 1, -1):
        assert cache.stride(dim) == expect or cache.shape[dim] == 1, (
            f"each (layer, block) slab must be contiguous (strides {cache.stride()})"
        )
        expect *= cache.shape[dim]
    return cache.shape[0], cache.stride(0) * es, cache.stride(1) * es, expect * es


def copy_blocks(caches, block_mapping: torch.Tensor, validate: bool = True) -> None:
    """For every cache, layer l and pair (s, d): ``cache[l, d] = cache[l, s]``.

    ``caches`` is one tensor or a list of layered caches [L, num_blocks, ...]
    (pages on dim 1, the layout CopyEngine takes: the fused GQA cache
    [L, P, 2, ps, H, D] moves K and V together, MLA is [L, P, ps, 576]).
    ``block_mapping`` is int64 [n, 2] of (src, dst) on the host or the device.
    With ``validate`` (default) the mapping is checked on the host -- ids in
    range, unique destinations, no destination that is also a source -- which
    makes the copy a snapshot: every read sees the pre-call contents.  A
    device-resident mapping is then copied to the host for the check; pass
    ``validate=False`` to skip it (out-of-range pairs are still skipped by the
    kernel, overlapping ones race).
    """
    if isinstance(caches, torch.Tensor):
        caches = [caches]
    assert len(caches) > 0
    device = caches[0].device
    assert all(c.is_cuda and c.device == device for c in caches)
    assert block_mapping.dtype == torch.int64 and block_mapping.ndim == 2 and block_mapping.shape[1] == 2
    n = block_mapping.shape[0]
    if n == 0:
        return
    if validate:
        host = block_mapping if not block_mapping.is_cuda else block_mapping.cpu()
        for c in caches:
            validate_block_mapping(host.numpy(), c.shape[1])
    if block_mapping.is_cuda:
        assert block_mapping.device == device
        dev_map = block_mapping.contiguous()
    else:
        dev_map = block_mapping.contiguous().pin_memory().to(device, non_blocking=True)
    stream = stream_handle(device)
    for c in caches:
        layers, layer_stride, block_stride, block_bytes = _slab(c)
        status = lib().psk_copy_blocks(
            ptr(c), layers, layer_stride, block_stride, block_bytes, c.shape[1], ptr(dev_map), n, stream
        )
        check(status, "copy_blocks")
    if not block_mapping.is_cuda:
        # keep the staged copy alive until the kernels that read it have run
        dev_map.record_stream(torch.cuda.current_stream(device))


# --------------------------------------------------------------------------- #
# tokens: eviction to a budget, commit of a drafted path
# --------------------------------------------------------------------------- #


def _cache_pairs(caches, first_row_dim):
    """``caches`` as (cache, second cache of the same geometry or None) pairs, one
    launch each.  Rows are contiguous from ``first_row_dim`` on."""
    if isinstance(caches, torch.Tensor):
        caches = [caches]
    assert len(caches) > 0
    first = caches[0]
    device, outer = first.device, first.shape[:3]
    assert first.is_cuda, "all caches must be on one GPU"
    assert first.ndim < 6 or outer[2] != 2, "a fused [L, num_blocks, 2, block_size, ...] cache goes as its K and V views"
    pairs, i = [], 0
    while i < len(caches):
        a = caches[i]
        shape, strides = a.shape, a.stride()
        assert a.device == device, "all caches must be on one GPU"
        assert shape[:3] == outer, "all caches must have the same layers, pages and page size"
        expect = 1
        for dim in range(len(shape) - 1, first_row_dim - 1, -1):
            assert strides[dim] == expect or shape[dim] == 1, (
                f"cache rows must be contiguous beyond dim {first_row_dim - 1} (strides {strides})"
            )
            expect *= shape[dim]
        # (all that a launch would refuse of a cache, so that none follows one that has written)
        assert 1 <= expect * a.element_size() < 2 ** 31, f"cache rows of {expect} elements"
        b = caches[i + 1] if i + 1 < len(caches) else None
        if b is not None and b.device == device and b.shape == shape and b.stride() == strides and b.dtype == a.dtype:
            pairs.append((a, b))
            i += 2
        else:
            pairs.append((a, None))
            i += 1
    return pairs


def _i32(t, device, dims, rows, name):
    shape = t.shape
    assert t.dtype == torch.int32 and t.device == device, f"{name} must be int32 on the caches' device"
    assert len(shape) == dims and shape[0] >= rows, f"{name} has shape {tuple(shape)}, want {dims} dimensions and {rows} rows"
    assert shape[-1] <= 1 or t.stride(-1) == 1, f"{name} needs unit last stride"


def evict_tokens(
    caches,
    scores: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    dst_block_table: torch.Tensor,
    budget: int,
    sink: int = 0,
    recent: int = 0,
    scores_out: torch.Tensor | None = None,
):
    """Keep at most ``budget`` tokens of each sequence and layer, by their
    scores, in fresh pages.

    caches: one tensor or a list (K and V views), [L, num_blocks, block_size,
    H, *row] with contiguous head rows, or [L, num_blocks, block_size, row] for
    a latent cache (H = 1).  scores: float32 [L, B, H, width] (unit last
    stride), for instance the running sums of
    ``attention.accumulate_attention_weights``, or [L, B, 1, width] for one
    choice for all heads.  For each layer, sequence and head, of the n =
    seq_lens[b] tokens (at most ``width``):
      * all are kept if n <= budget;
      * else the first ``sink``, the last ``recent`` and, of those between, the
        budget - sink - recent of the highest scores; ties go to the lower
        position, a NaN score counts below every other.
    Kept token i, in position order, becomes row i of the pages
    ``dst_block_table[b]`` (int32 [B, W], rows for the budget or for ``width``
    tokens, whichever are fewer; entries outside the cache are skipped, a source
    row on a missing page reads as zeros).
    Those pages must be none that ``block_table`` names, each named once: prefix
    pages may be shared by sequences, so they are read and left as they are.
    ``scores_out`` (default: ``scores``, in place; else it shares no element with
    it) receives the kept tokens' scores, then zeros up to n.

    Returns (kept, new_lens): int32 [L, B, H or 1, budget], each kept token's old
    position (-1 past the last), and int32 [B], the new lengths.  One launch for
    the choice -- for scores of more than 16384 tokens four, five in place, and as
    many again for every 4096 parts of 16384 of all their rows -- and one for each
    pair of caches of one geometry; no synchronization.
    """
    first = caches if isinstance(caches, torch.Tensor) else caches[0]
    assert first.ndim >= 4, "caches are layered: [L, num_blocks, block_size, heads, ...] or [L, num_blocks, block_size, row]"
    heads = 1 if first.ndim == 4 else first.shape[3]
    pairs = _cache_pairs(caches, 3 if first.ndim == 4 else 4)
    device = first.device
    layers, num_blocks, page = first.shape[:3]
    for a, _ in pairs:
        assert a.ndim == first.ndim and (a.ndim == 4 or a.shape[3] == heads), "all caches must have the same heads"
    shape, strides = scores.shape, scores.stride()
    assert scores.dtype == torch.float32 and len(shape) == 4 and scores.device == device
    B, kept_heads, width = shape[1:]
    assert shape[0] == layers and kept_heads in (1, heads), \
        f"scores of shape {tuple(shape)} for {layers} layers of {heads} heads"
    assert strides[3] == 1 or width <= 1, "scores need unit last stride"
    out_strides, out_width = strides, width
    if scores_out is None:
        scores_out = scores
    else:
        out_strides, out_width = scores_out.stride(), scores_out.shape[-1]
        assert scores_out.dtype == torch.float32 and scores_out.device == device
        assert scores_out.dim() == 4 and scores_out.shape[:3] == shape[:3]
        assert out_strides[3] == 1 or out_width <= 1, "scores need unit last stride"
    in_place = scores_out is scores or (scores_out.data_ptr() == scores.data_ptr() and out_strides == strides)
    assert distinct(scores_out, max(width, out_width)) if in_place else distinct(scores_out) and not overlap(scores, scores_out), \
        "scores_out must be scores itself or share no element with it, and be no broadcast"
    budget, sink, recent = int(budget), int(sink), int(recent)
    assert budget >= 1 and sink >= 0 and recent >= 0 and sink + recent <= budget, \
        f"sink {sink} and recent {recent} do not fit a budget of {budget}"
    _i32(block_table, device, 2, B, "block_table")
    _i32(dst_block_table, device, 2, B, "dst_block_table")
    _i32(seq_lens, device, 1, B, "seq_lens")
    # (all that a launch would refuse, so that none follows one that has written)
    assert 1 <= layers <= 65535 and B <= 65535 and heads >= 1 and budget * heads < 2 ** 31, \
        f"{layers} layers, {B} sequences, a budget of {budget} for {heads} heads"
    assert num_blocks >= 1 and page >= 1 and (B == 0 or block_table.shape[1] >= 1 and dst_block_table.shape[1] >= 1), \
        "an empty cache or block table"
    assert dst_block_table.shape[1] * page >= min(budget, width), \
        f"{dst_block_table.shape[1]} pages of {page} cannot hold a budget of {budget}"
    assert block_table.data_ptr() != dst_block_table.data_ptr() or B == 0, "the kept tokens go to pages of their own"
    kept = torch.empty(layers, B, kept_heads, budget, dtype=torch.int32, device=device)
    new_lens = torch.empty(B, dtype=torch.int32, device=device)
    with on_device(device):
        stream = stream_handle(device)
        need = int(lib().psk_select_tokens_workspace_bytes(layers, B, kept_heads, width, budget))
        if need < 0:
            check(need, "evict_tokens workspace")
        workspace = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        status = lib().psk_select_tokens(
            ptr(scores), i64_array(strides[:3]), width, ptr(scores_out), i64_array(out_strides[:3]), out_width,
            ptr(seq_lens), layers, B, kept_heads, budget, sink, recent, ptr(kept), ptr(new_lens), ptr(workspace), need,
            stream,
        )
        check(status, "evict_tokens")
        for a, b in pairs if B else ():
            es, st = a.element_size(), a.stride()
            head = math.prod(a.shape[3 if a.ndim == 4 else 4:])
            status = lib().psk_move_kept_tokens(
                ptr(a), ptr(b), st[0] * es, st[1] * es, st[2] * es, 0 if a.ndim == 4 else st[3] * es, head * es, layers,
                heads, page, num_blocks, ptr(block_table),
                block_table.stride(0), block_table.shape[1], ptr(dst_block_table), dst_block_table.stride(0),
                dst_block_table.shape[1], ptr(kept), kept_heads, budget, B, stream,
            )
            check(status, "evict_tokens")
    return kept, new_lens


def commit_draft_tokens(
    caches,
    block_table: torch.Tensor,
    starts: torch.Tensor,
    path: torch.Tensor,
    path_lens: torch.Tensor,
) -> None:
    """Make the accepted path of each drafted tree the sequence's next tokens,
    in every layer.

    Sequence b's drafted tokens were appended in tree order from position
    ``starts[b]``; ``path[b, i]`` (int32 [B, M], M at most 256) is the i-th
    accepted one's index among them, for i < path_lens[b] (int32 [B]).  The row
    of position starts[b] + path[b, i] becomes the row of position starts[b] +
    i, as a snapshot: every row is read before any is written, whatever the
    order of ``path``.  The sequence then has starts[b] + path_lens[b] tokens.
    caches: one tensor or a list, [L, num_blocks, block_size, *row] with
    contiguous rows (K and V views of the fused cache, a latent cache; the fused
    [L, num_blocks, 2, block_size, ...] one itself is refused); two of one
    geometry move in one launch.  Negative indices and rows on missing pages
    are skipped.  The pages of drafted tokens are a sequence's own.
    """
    pairs = _cache_pairs(caches, 3)
    first = pairs[0][0]
    assert first.ndim >= 4, "caches are layered: [L, num_blocks, block_size, ...]"
    # (a launch moves what the one before it has left)
    assert len(pairs) == 1 or len({c.data_ptr() for c in caches}) == len(caches), "a cache is named twice"
    device = first.device
    layers, num_blocks, page = first.shape[:3]
    B = path.shape[0]
    _i32(path, device, 2, 0, "path")
    _i32(block_table, device, 2, B, "block_table")
    _i32(starts, device, 1, B, "starts")
    _i32(path_lens, device, 1, B, "path_lens")
    with on_device(device):
        for a, b in pairs:
            es, st = a.element_size(), a.stride()
            status = lib().psk_commit_draft_tokens(
                ptr(a), ptr(b), st[0] * es, st[1] * es, st[2] * es, math.prod(a.shape[3:]) * es, layers, page, num_blocks, ptr(block_table), block_table.stride(0), block_table.shape[1], ptr(starts),
                ptr(path), path.stride(0), path.shape[1], ptr(path_lens), B, stream_handle(device),
            )
            check(status, "commit_draft_tokens")


# --------------------------------------------------------------------------- #
# FP8 per-tensor scale
# --------------------------------------------------------------------------- #

_workspaces: dict = {}
_ws_lock = threading.Lock()


def amax_workspace(device) -> torch.Tensor:
    """Per-device uint32 workspace of the amax kernels (partial maxima).

    Allocate it (``warmup``) before any HIP graph capture; it needs no initial
    contents, so it is reusable inside graphs.  Calls that share it must be
    ordered on one stream (they run on the caller's stream).
    """
    device = torch.device(device)
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    ws = _workspaces.get(device)
    if ws is None:
        with _ws_lock:
            ws = _workspaces.get(device)
            if ws is None:
                assert not torch.cuda.is_current_stream_capturing(), (
                    "allocate the amax workspace (cache_ops.warmup) before graph capture"
                )
                n = int(lib().psk_kv_amax_workspace_len())
                ws = torch.zeros(n, dtype=torch.int32, device=device)
                _workspaces[device] = ws
    return ws


def warmup(device) -> None:
    amax_workspace(device)


def compute_kv_scales(
    key: torch.Tensor,
    value: torch.Tensor | None = None,
    qmax: float = FP8_E4M3_MAX,
    out: torch.Tensor | None = None,
    amax_out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Per-tensor scales ``amax / qmax`` (1.0 for an all-zero tensor) for key
    and value, in one launch; returns float32 [2] (or [1] without value).

    amax = max |x| over the tensor, NaN ignored.  Inputs are [N, ...] with
    contiguous rows (dims 1..), e.g. the strided K/V views of a qkv projection.
    """
    assert key.is_cuda
    device = key.device
    tensors = [key] if value is None else [key, value]
    for t in tensors:
        assert t.device == device and t.dtype in (torch.bfloat16, torch.float16, torch.float32)
        assert t.dtype == key.dtype and t.shape == key.shape
    rows = key.shape[0] if key.ndim else 1
    row_len = math.prod(key.shape[1:]) if key.ndim > 1 else 1
    strides = []
    for t in tensors:
        if t.ndim > 1:
            exp = 1
            for dim in range(t.ndim - 1, 0, -1):
                assert t.stride(dim) == exp or t.shape[dim] == 1, "rows must be contiguous"
                exp *= t.shape[dim]
        strides.append(t.stride(0) if t.ndim else 1)
    k = len(tensors)
    if out is None:
        assert not torch.cuda.is_current_stream_capturing(), "pass `out` when capturing"
        out = torch.empty(k, dtype=torch.float32, device=device)
    assert out.dtype == torch.float32 and out.numel() >= k and out.is_contiguous() and out.device == device
    if amax_out is not None:
        assert amax_out.dtype == torch.float32 and amax_out.numel() >= k and amax_out.device == device
    ws = amax_workspace(device)
    if k == 2 and rows * row_len == 0:
        # Empty tensors have NULL data, and a NULL second tensor means "key
        # only" to the C entry: one single-tensor call per output (scale 1.0).
        for j, t in enumerate(tensors):
            status = lib().psk_kv_amax_scale(
                ptr(t), None, rows, row_len, strides[j], strides[j], dtype_code(key.dtype), float(qmax),
                out.data_ptr() + 4 * j, None if amax_out is None else amax_out.data_ptr() + 4 * j,
                ptr(ws), ws.numel(), stream_handle(device),
            )
            check(status, "compute_kv_scales")
        return out
    status = lib().psk_kv_amax_scale(
        ptr(key), ptr(value), rows, row_len, strides[0], strides[-1], dtype_code(key.dtype), float(qmax),
        ptr(out), ptr(amax_out), ptr(ws), ws.numel(), stream_handle(device),
    )
    check(status, "compute_kv_scales")
    return out
