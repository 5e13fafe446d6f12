"""Norms of the query and key heads with the rotation of their positions, in one
pass, with the append of K and V where there is a cache.

The reference norms and rotates q and k as layers of their own and then calls
``append_kv_cache`` (pipeswift/utils/impl_utils.py:303-314); ``norm_rope_and_cache``
does the three in one launch of ``psk_norm_rope`` and leaves the cache bytes that
they would.

For a head x [D]: ``y = x * rsqrt(mean(x^2) + eps) * weight`` in float32 (no weight:
y = x); then pair i of the first ``rot`` elements, (y[i], y[i + rot/2]) or with
``interleaved`` (y[2i], y[2i+1]), turns by its position's angle:
(a c - b s, b c + a s).  ``cos_sin`` float32 [positions, rot] holds the cosines of the
rot/2 pairs, then their sines.  ``positions`` is [N], or [axes, N] for several axes
(time, height, width): then ``sections`` says how many pairs, in order, go by each.
A weight that counts from one (``1 + w``) is passed with the one added.
Results are rounded once, to the input's type.  A position outside the table turns
its head to NaN.
"""

from __future__ import annotations

from typing import Optional, Sequence

import torch

from . import _lib
from ._lib import check, distinct, dtype_code, i64_array, lib, on_device, overlap, ptr, stream_handle
from .mxfp4_kv import check_cache

_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def _span(t):
    """First and last byte address that a tensor covers (none: an empty span)."""
    if 0 in t.shape:
        return 0, -1
    last = sum(s * (n - 1) for s, n in zip(t.stride(), t.shape))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size() - 1


def _check_out(out, own, others, name):
    """An output is its input itself, or shares no element with any input."""
    assert out.shape == own.shape and out.dtype == own.dtype and out.device == own.device, \
        f"{name} must have the shape and type of its input"
    assert out.stride(2) == 1 or out.shape[2] <= 1, f"{name} needs unit last stride"
    assert distinct(out), f"{name} is a broadcast"
    in_place = out.data_ptr() == own.data_ptr() and out.stride() == own.stride()
    lo, hi = _span(out)
    for t in others if in_place else (own, *others):
        if t is None:
            continue
        a, b = _span(t)
        assert b < lo or hi < a or t.element_size() == out.element_size() and not overlap(out, t), \
            f"{name} must be its input itself or share no element with the inputs and outputs"


def _run(q, k, v, positions, cos_sin, q_weight, k_weight, eps, sections, interleaved, q_out, k_out, caches, slot_mapping,
         scales, what):
    device = q.device
    assert q.is_cuda and k.is_cuda, "q and k must be on a GPU"
    assert q.ndim == 3 and k.ndim == 3 and q.shape[0] == k.shape[0] and q.shape[2] == k.shape[2], \
        f"q {tuple(q.shape)} and k {tuple(k.shape)} must be [N, heads, D]"
    assert q.dtype in _TYPES and k.dtype == q.dtype, f"q and k are bf16, fp16 or fp32, not {q.dtype} and {k.dtype}"
    n, hq, dim = q.shape
    hkv = k.shape[1]
    for t in (q, k, v):
        assert t is None or t.stride(2) == 1 or t.numel() == 0, "heads must have unit inner stride"
    assert cos_sin.dtype == torch.float32 and cos_sin.ndim == 2 and cos_sin.stride(1) == 1, \
        "cos_sin must be float32 [positions, rot] with unit last stride"
    assert positions.dtype in (torch.int32, torch.int64) and positions.ndim in (1, 2) and positions.shape[-1] == n, \
        f"positions must be int32 or int64 [{n}] or [axes, {n}]"
    assert positions.stride(-1) == 1 or n <= 1, "positions need unit last stride"
    axes = positions.shape[0] if positions.ndim == 2 else 1
    if axes > 1 or sections is not None:
        assert sections is not None and len(sections) == axes, f"positions on {axes} axes need as many sections"
        assert sum(int(x) for x in sections) * 2 == cos_sin.shape[1], \
            f"sections {list(sections)} are not the {cos_sin.shape[1] // 2} pairs of the rotation"
    weight_dtype = q.dtype
    for w in (q_weight, k_weight):
        if w is not None:
            assert w.shape == (dim,) and w.is_contiguous() and w.dtype in (q.dtype, torch.float32), \
                f"a norm's weight is [{dim}] in {q.dtype} or float32"
            weight_dtype = w.dtype
    assert q_weight is None or k_weight is None or q_weight.dtype == k_weight.dtype, "the weights have one type"
    if q_out is None:
        q_out = torch.empty((n, hq, dim), dtype=q.dtype, device=device)
    else:
        _check_out(q_out, q, (k, v, k_out), "q_out")
    if k_out is not None:
        _check_out(k_out, k, (q, v), "k_out")
    elif caches is None:
        k_out = torch.empty((n, hkv, dim), dtype=q.dtype, device=device)
    kc = vc = kcs = vcs = slots = None
    code, page, blocks = 0, 1, 0
    if caches is not None:
        kc, vc = caches
        assert v.shape == k.shape and v.dtype == k.dtype, f"v {tuple(v.shape)} must be like k {tuple(k.shape)}"
        assert kc.ndim == 4 and vc.shape == kc.shape and vc.dtype == kc.dtype
        if kc.dtype == torch.uint8:
            check_cache(kc, hkv, dim, "key_cache")
            check_cache(vc, hkv, dim, "value_cache")
            code = _lib.MXFP4_CODE
        else:
            assert kc.dtype in (q.dtype, torch.float8_e4m3fn), f"kv cache dtype {kc.dtype} does not match {q.dtype}"
            assert kc.shape[2:] == (hkv, dim), f"cache rows {tuple(kc.shape[2:])} for keys ({hkv}, {dim})"
            assert kc.stride(3) == 1 and vc.stride(3) == 1, "cache rows need unit last stride"
            code = dtype_code(kc.dtype)
        slots = slot_mapping
        assert slots.dtype == torch.int64 and slots.shape == (n,) and slots.is_contiguous(), \
            f"slot_mapping must be contiguous int64 [{n}]"
        for s in scales:
            assert s is None or s.dtype == torch.float32 and s.numel() == 1 and kc.dtype == torch.float8_e4m3fn, \
                "scales are one float32 element each and only apply to an fp8 cache"
        page, blocks = kc.shape[1], kc.shape[0]
        kcs, vcs = i64_array(kc.stride()), i64_array(vc.stride())
    for t in (k, v, positions, cos_sin, q_weight, k_weight, kc, vc, slots, *scales):
        assert t is None or t.device == device, "all tensors must be on q's device"
    with on_device(device):
        st = lib().psk_norm_rope(
            ptr(q), i64_array(q.stride()), ptr(k), i64_array(k.stride()), ptr(v), None if v is None else i64_array(v.stride()),
            dtype_code(q.dtype), n, hq, hkv, dim, ptr(q_weight), ptr(k_weight), dtype_code(weight_dtype), float(eps),
            ptr(positions), positions.element_size(), positions.stride(0) if axes > 1 else 0, axes,
            i64_array([int(x) for x in sections]) if axes > 1 else None, ptr(cos_sin), max(cos_sin.stride(0), cos_sin.shape[1]),
            cos_sin.shape[0], cos_sin.shape[1], 1 if interleaved else 0, ptr(q_out), i64_array(q_out.stride()),
            ptr(k_out), None if k_out is None else i64_array(k_out.stride()), ptr(kc), ptr(vc), kcs, vcs, code, ptr(slots),
            page, blocks, ptr(scales[0]), ptr(scales[1]), stream_handle(device),
        )
    check(st, what)
    return q_out, k_out


def norm_rope(
    q: torch.Tensor,
    k: torch.Tensor,
    positions: torch.Tensor,
    cos_sin: torch.Tensor,
    q_weight: Optional[torch.Tensor] = None,
    k_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    sections: Optional[Sequence[int]] = None,
    interleaved: bool = False,
    q_out: Optional[torch.Tensor] = None,
    k_out: Optional[torch.Tensor] = None,
):
    """q [N, Hq, D] and k [N, Hkv, D] (bf16, fp16 or fp32; slices of a projection are
    fine, heads on 16-byte boundaries) normed and rotated.  ``q_out`` and ``k_out``
    may be q and k themselves.  D: a multiple of 8 up to 512; rot: a multiple of 16,
    or of 8 with ``interleaved``.  Returns (q_out, k_out)."""
    return _run(q, k, None, positions, cos_sin, q_weight, k_weight, eps, sections, interleaved, q_out, k_out, None, None,
                (None, None), "norm_rope")


def norm_rope_and_cache(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
    positions: torch.Tensor,
    cos_sin: torch.Tensor,
    q_weight: Optional[torch.Tensor] = None,
    k_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    sections: Optional[Sequence[int]] = None,
    interleaved: bool = False,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
    q_out: Optional[torch.Tensor] = None,
    k_out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``norm_rope`` and the append of its keys and of ``v`` [N, Hkv, D] at
    ``slot_mapping`` (int64 [N]; negative and out-of-range slots are skipped, their
    queries computed all the same): the bytes of ``reshape_and_cache_flash`` for a
    cache of k's type or FP8 (with ``k_scale`` / ``v_scale``), of
    ``mxfp4_kv.reshape_and_cache_mxfp4`` for a uint8 one.  The keys are rounded to
    their type first, as there.  ``k_out`` receives them too if given.  Returns q_out."""
    return _run(q, k, v, positions, cos_sin, q_weight, k_weight, eps, sections, interleaved, q_out, k_out,
                (key_cache, value_cache), slot_mapping, (k_scale, v_scale), "norm_rope_and_cache")[0]
