"""ctypes binding of libpipeswift_kv.so, the gfx950 C ABI of the KV-cache path.

The library is built in-tree (``__graft_entry__.build()`` or
``make -C pipeswift_amd/csrc``) next to this file.  There is no fallback: if the
library is missing every operation raises, so nothing can silently run a
non-HIP path.  Status codes follow include/pipeswift_kv.h: negative values are
precondition failures (AssertionError, matching the reference's Python
asserts), positive values are hipError_t (RuntimeError, matching the
reference's driver-failure path, copy_engine.py:454-457).
"""

from __future__ import annotations

import contextlib
import ctypes
import os
import struct
import threading

import numpy as np
import torch

LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libpipeswift_kv.so")

DTYPE_CODES = {
    torch.float32: 0,
    torch.float16: 1,
    torch.bfloat16: 2,
    torch.float8_e4m3fn: 3,
}
MXFP4_CODE = 4  # the rows of mxfp4_kv, held as uint8

SWAP_MEMCPY = 0
SWAP_BLIT = 2

_c_int64_p = ctypes.POINTER(ctypes.c_int64)
_c_uint64_p = ctypes.POINTER(ctypes.c_uint64)
_vp = ctypes.c_void_p
_i64 = ctypes.c_int64
_int = ctypes.c_int

# name -> (restype, argtypes)
_SIGNATURES = {
    "psk_last_error": (ctypes.c_char_p, []),
    "psk_abi_version": (_int, []),
    "psk_reshape_and_cache": (
        _int,
        [_vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _c_int64_p, _c_int64_p, _int, _int,
         _vp, _vp, _vp],
    ),
    "psk_concat_and_cache_mla": (
        _int,
        [_vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _int, _int, _vp, _vp],
    ),
    "psk_gather_cache": (
        _int,
        [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _int, _int,
         _vp, _vp],
    ),
    "psk_copy_blocks": (_int, [_vp, _i64, _i64, _i64, _i64, _i64, _vp, _i64, _vp]),
    "psk_swap_blocks": (
        _int,
        [_int, _c_uint64_p, _c_uint64_p, _c_uint64_p, _i64, _c_int64_p, _c_int64_p, _c_int64_p, _i64, _i64, _i64,
         _vp, _i64, _vp, _i64, _vp],
    ),
    "psk_swap_staging_bytes": (_i64, [_i64, _i64]),
    "psk_coalesce_runs": (_i64, [_c_int64_p, _c_int64_p, _i64, _c_int64_p, _c_int64_p, _c_int64_p]),
    "psk_kv_amax_scale": (
        _int,
        [_vp, _vp, _i64, _i64, _i64, _i64, _int, ctypes.c_float, _vp, _vp, _vp, _i64, _vp],
    ),
    "psk_kv_amax_workspace_len": (_i64, []),
    "psk_reshape_and_cache_amax": (
        _int,
        [_vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _c_int64_p, _c_int64_p, _int,
         ctypes.c_float, _vp, _vp, _vp, _i64, _vp],
    ),
    "psk_kv_amax_scale_noalloc": (
        _int,
        [_vp, _vp, _i64, _i64, _i64, _i64, _int, ctypes.c_float, _vp, _vp, _vp],
    ),
    "psk_build_kv_metadata": (
        _i64,
        [_i64, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _int, _i64, _vp, _vp, _vp, _vp, _vp, _i64],
    ),
    "psk_refresh_graph_metadata": (
        _int,
        [_vp, _i64, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _vp, _i64, _i64, _vp, _i64, _vp, _vp, _vp, _i64, _i64,
         ctypes.c_int32, _vp],
    ),
    "psk_build_next_decode_metadata": (
        _i64, [_i64, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _vp, _vp],
    ),
    "psk_host_alloc": (_int, [_i64, ctypes.POINTER(ctypes.c_void_p)]),
    "psk_host_free": (_int, [_vp]),
    "psk_keyed_hash": (_int, [_vp, _i64, ctypes.c_uint64, _int, _vp]),
    "psk_page_hash_chain": (_i64, [_vp, _i64, _i64, _i64, ctypes.c_uint64, _int, _vp, _i64]),
    "psk_paged_decode_attention": (
        _int,
        [_vp, _i64, _i64, _int, _vp, _vp, _c_int64_p, _c_int64_p, _vp, _i64, _i64, _vp, _i64, _i64, _i64, _i64, _i64,
         _i64, _i64, _i64, _i64, _vp, _int, ctypes.c_float, _vp, _vp, _vp, _c_int64_p, _vp, _i64, _i64, _int, _vp,
         _i64, _vp, _i64, _vp],
    ),
    "psk_paged_decode_workspace_len": (_i64, [_i64, _i64, _i64, _i64, _i64, _i64]),
    "psk_paged_prefill_attention": (
        _int,
        [_vp, _i64, _i64, _int, _vp, _vp, _c_int64_p, _c_int64_p, _vp, _i64, _i64, _vp, _i64, _i64, _i64, _i64, _i64,
         _i64, _i64, _i64, _vp, _int, ctypes.c_float, _vp, _vp, _vp, _c_int64_p, _vp, _i64, _i64, _int, _vp, _i64,
         _vp, _i64, _vp],
    ),
    "psk_paged_prefill_workspace_len": (_i64, [_i64]),
    "psk_paged_prefill_step_workspace_len": (_i64, [_i64] * 6),
    "psk_paged_tree_attention": (
        _int,
        [_vp, _i64, _i64, _int, _vp, _vp, _c_int64_p, _c_int64_p, _vp, _i64, _i64, _vp, _i64, _i64, _i64, _i64, _i64,
         _i64, _i64, _i64, _i64, _vp, _vp, _i64, _i64, ctypes.c_float, _vp, _vp, _vp, _c_int64_p, _vp, _i64, _i64,
         _int, _vp, _i64, _vp, _i64, _vp],
    ),
    "psk_paged_tree_workspace_len": (_i64, [_i64] * 6),
    "psk_accumulate_attention_weights": (
        _int,
        [_vp, _i64, _i64, _i64, _vp, _i64, _i64, _int, _vp, _c_int64_p, _vp, _i64, _vp, _i64, _i64, _vp, _i64, _i64,
         _i64, _i64, _i64, _i64, _i64, _i64, _i64, _vp, _int, ctypes.c_float, ctypes.c_float, _vp, _vp, _c_int64_p,
         _vp, _i64, _vp],
    ),
    "psk_attention_weights_workspace_bytes": (_i64, [_i64, _i64, _i64, _i64, _int]),
    "psk_select_tokens": (
        _int,
        [_vp, _c_int64_p, _i64, _vp, _c_int64_p, _i64, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _vp, _vp, _vp, _i64,
         _vp],
    ),
    "psk_select_tokens_workspace_bytes": (_i64, [_i64] * 5),
    "psk_move_kept_tokens": (
        _int,
        [_vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _vp, _i64, _i64, _vp, _i64, _i64, _vp, _i64,
         _i64, _i64, _vp],
    ),
    "psk_commit_draft_tokens": (
        _int,
        [_vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _vp, _i64, _i64, _vp, _vp, _i64, _i64, _vp, _i64, _vp],
    ),
    "psk_norm_rope": (
        _int,
        [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _int, _i64, _i64, _i64, _i64, _vp, _vp, _int, ctypes.c_float, _vp, _int,
         _i64, _i64, _vp, _vp, _i64, _i64, _i64, _int, _int, _vp, _i64, _i64, _vp, _vp, _vp],
    ),
    "psk_paged_mxfp4_attention": (
        _int,
        [_vp, _i64, _i64, _int, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _vp, _i64, _i64, _i64, _i64, _i64,
         _i64, _i64, _i64, _i64, _vp, _int, ctypes.c_float, _vp, _i64, _i64, _int, _vp, _i64, _vp, _i64, _vp],
    ),
    "psk_paged_mxfp4_workspace_len": (_i64, [_i64] * 6),
    "psk_mxfp4_entry_bytes": (_i64, [_i64]),
    "psk_reshape_and_cache_mxfp4": (
        _int,
        [_vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _vp, _int, _vp],
    ),
    "psk_gather_mxfp4": (
        _int,
        [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _vp, _i64, _int, _vp],
    ),
    "psk_mla_fp8_tile_entry_bytes": (_i64, [_i64, _i64]),
    "psk_concat_and_cache_mla_fp8_tiles": (
        _int, [_vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _int, _vp],
    ),
    "psk_gather_mla_fp8_tiles": (
        _int, [_vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _int, _vp],
    ),
}

EXPORTED_SYMBOLS = tuple(_SIGNATURES)

_lib = None
_lock = threading.Lock()


def lib() -> ctypes.CDLL:
    """Load the library once; raise ImportError with the build command if absent."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not os.path.exists(LIB_PATH):
                raise ImportError(
                    f"{LIB_PATH} is not built; run `python -c 'import __graft_entry__ as g; g.build()'` "
                    "from the repository root (hipcc --offload-arch=gfx950)"
                )
            handle = ctypes.CDLL(LIB_PATH)
            for name, (res, args) in _SIGNATURES.items():
                fn = getattr(handle, name)
                fn.restype = res
                fn.argtypes = args
            _lib = handle
    return _lib


def check(status: int, what: str) -> None:
    if status == 0:
        return
    msg = lib().psk_last_error().decode(errors="replace")
    if status < 0:
        raise AssertionError(f"{what}: {msg}")
    raise RuntimeError(f"{what}: {msg}")


def dtype_code(dtype: torch.dtype) -> int:
    try:
        return DTYPE_CODES[dtype]
    except KeyError:
        raise AssertionError(f"unsupported dtype {dtype}") from None


# torch's raw accessor of the current stream (what its generated kernels call):
# 0.05 us against 1.7 us for torch.cuda.current_stream(device).cuda_stream, which
# builds a Stream object per call.  The public call is the fallback.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream_handle(device: torch.device) -> int:
    if _raw_stream is not None:
        idx = device.index if device.index is not None else torch.cuda.current_device()
        return _raw_stream(idx)
    return torch.cuda.current_stream(device).cuda_stream


_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_HERE = contextlib.nullcontext()


def on_device(device: torch.device):
    """A context in which ``device`` is the current one: the library launches on
    the current device, and the stream has to be one of its own."""
    if device.index is None or device.index == _current_device():
        return _HERE
    return torch.cuda.device(device)


_I64x4 = ctypes.c_int64 * 4
_I64x3, _I64x6 = ctypes.c_int64 * 3, ctypes.c_int64 * 6


def i64_array(values) -> ctypes.Array:
    n = len(values)
    if n == 4:
        return _I64x4(*values)
    if n == 3:
        return _I64x3(*values)
    return (_I64x6 if n == 6 else ctypes.c_int64 * n)(*values)


# Packed int64 values, for the entries that take strides as one pointer: a bytes
# object is passed by its address, at a tenth of a ctypes array's cost.
pack_i64x3, pack_i64x10, pack_i64x16 = (struct.Struct(f"={n}q").pack for n in (3, 10, 16))


def _row_starts(t):
    """(first elements of a tensor's rows, sorted, by their places in memory; elements of a row).
    A row is the last dimension where its stride is one, else a single element."""
    shape, strides = list(t.shape), list(t.stride())
    width = shape.pop() if shape and strides[-1] == 1 else 1
    at = np.zeros(1, dtype=np.int64)
    for n, s in zip(shape, strides):
        at = (at[:, None] + np.arange(n, dtype=np.int64) * s).reshape(-1)
    return np.sort(at), width


def distinct(t, width: int = 0) -> bool:
    """Whether no two elements of a tensor lie in one place (a broadcast, rows that
    overlap); ``width``: with rows of at least as many elements."""
    if t.is_contiguous() and (not width or width <= t.shape[-1]):
        return True
    inner = 0  # places that the dimensions so far span, less one
    for s, n in sorted((s, n if s != 1 else max(n, width)) for s, n in zip(t.stride(), t.shape) if n > 1 or s == 1):
        if n > 1 and s <= inner:
            break
        inner += s * (n - 1)
    else:
        return True
    starts, own = _row_starts(t)
    return len(starts) < 2 or int(np.diff(starts).min()) >= max(own, width)


def overlap(a, b) -> bool:
    """Whether two tensors of one element size share an element."""
    apart = (b.data_ptr() - a.data_ptr()) // a.element_size()
    if a.is_contiguous() and b.is_contiguous():
        return -b.numel() < apart < a.numel() and 0 not in a.shape and 0 not in b.shape
    if 0 in a.shape or 0 in b.shape:
        return False
    ends = [sum(s * (n - 1) for s, n in zip(t.stride(), t.shape)) for t in (a, b)]
    if apart > ends[0] or apart + ends[1] < 0:
        return False
    (x, wx), (y, wy) = _row_starts(a), _row_starts(b)
    y = y + apart  # a row of b at y overlaps those of a at y - wx < x < y + wy
    return bool((np.searchsorted(x, y - wx, "right") < np.searchsorted(x, y + wy, "left")).any())


def ptr(t) -> int:
    return 0 if t is None else t.data_ptr()
