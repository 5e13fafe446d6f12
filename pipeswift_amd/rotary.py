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
the pairs that go by it to NaN, and no other element.
"""

from __future__ import annotations

from typing import Optional, Sequence

import torch

from . import _lib
from ._lib import check, distinct, i64_array, lib, on_device, overlap, pack_i64x16, ptr, stream_handle
from .mxfp4_kv import check_cache

_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def _span(t):
    """First and last byte address that a tensor covers (none: an empty span)."""
    if 0 in t.shape:
        return 0, -1
    last = sum(s * (n - 1) for s, n in zip(t.stride(), t.shape))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size() - 1


def _side_by_side(a, b):
    """Whether [N, heads, D] tensors of one type and token stride are columns of a projection that do not
    meet (False where it takes ``overlap`` to say)."""
    s, size = a.stride(0), a.element_size()
    off, rest = divmod(b.data_ptr() - a.data_ptr(), size)
    if rest or s <= 0 or b.dim() != 3 or b.stride(0) != s:
        return False
    at = off % s
    return at >= (a.shape[1] - 1) * a.stride(1) + a.shape[2] and at + (b.shape[1] - 1) * b.stride(1) + b.shape[2] <= s


def _check_out(out, own, others, name):
    """An output is its input itself, or shares no element with any input, other output or cache."""
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
        assert b < lo or hi < a or t.element_size() == out.element_size() and (_side_by_side(out, t) or not overlap(out, t)), \
            f"{name} must be its input itself or share no element with the inputs, outputs and caches"


def _sections(sections, axes, pairs):
    assert sections is not None and len(sections) == axes, f"positions on {axes} axes need as many sections"
    sections = [int(x) for x in sections]
    assert sum(sections) == pairs, f"sections {sections} are not the {pairs} pairs of the rotation"
    return i64_array(sections) if axes > 1 else None


def _run(q, k, v, positions, cos_sin, q_weight, k_weight, eps, sections, interleaved, q_out, k_out, kc, vc, slots, k_scale,
         v_scale, what):
    device, dtype = q.device, q.dtype
    assert q.is_cuda, "q must be on a GPU"
    assert len(q.shape) == 3 and len(k.shape) == 3, f"q {tuple(q.shape)} and k {tuple(k.shape)} must be [N, heads, D]"
    n, hq, dim = q.shape
    hkv = k.shape[1]
    assert k.shape[0] == n and k.shape[2] == dim, f"q {tuple(q.shape)} and k {tuple(k.shape)} must be [N, heads, D]"
    assert dtype in _TYPES and k.dtype == dtype, f"q and k are bf16, fp16 or fp32, not {dtype} and {k.dtype}"
    qs, ks = q.stride(), k.stride()
    assert (qs[2] == 1 or q.numel() == 0) and (ks[2] == 1 or k.numel() == 0), "heads must have unit inner stride"
    assert len(cos_sin.shape) == 2, "cos_sin must be [positions, rot]"
    known, rot = cos_sin.shape
    table = cos_sin.stride()
    assert cos_sin.dtype == torch.float32 and table[1] == 1, "cos_sin must be float32 [positions, rot] with unit last stride"
    assert table[0] >= rot or known <= 1, f"cos_sin has rows of {rot} that are {table[0]} apart"
    dims = len(positions.shape)
    ps = positions.stride()
    assert dims in (1, 2) and positions.shape[-1] == n and (ps[-1] == 1 or n <= 1), \
        f"positions must be [{n}] or [axes, {n}] with unit last stride"
    assert positions.dtype in (torch.int64, torch.int32), f"positions are int32 or int64, not {positions.dtype}"
    axes = positions.shape[0] if dims == 2 else 1
    if axes != 1 or sections is not None:
        sections = _sections(sections, axes, rot // 2)
    weight_dtype = dtype
    for w in (q_weight, k_weight):
        if w is not None:
            assert w.shape == (dim,) and (w.dtype == dtype or w.dtype == torch.float32) and w.is_contiguous(), \
                f"a norm's weight is [{dim}] in {dtype} or float32"
            weight_dtype = w.dtype
    assert q_weight is None or k_weight is None or q_weight.dtype == k_weight.dtype, "the weights have one type"
    if q_out is None:
        q_out = torch.empty((n, hq, dim), dtype=dtype, device=device)
    else:
        _check_out(q_out, q, (k, v, k_out, kc, vc), "q_out")
    if k_out is not None:
        _check_out(k_out, k, (q, v, kc, vc), "k_out")
    elif kc is None:
        k_out = torch.empty((n, hkv, dim), dtype=dtype, device=device)
    vs = os = kcs = vcs = (0, 0, 0)
    code, page, blocks = 0, 1, 0
    if k_out is not None:
        os = k_out.stride()
    if kc is not None:
        assert v.shape == k.shape and v.dtype == dtype, f"v {tuple(v.shape)} must be like k {tuple(k.shape)}"
        vs = v.stride()
        assert vs[2] == 1 or v.numel() == 0, "heads must have unit inner stride"
        shape, ctype = kc.shape, kc.dtype
        assert len(shape) == 4 and vc.shape == shape and vc.dtype == ctype
        if ctype == torch.uint8:
            check_cache(kc, hkv, dim, "key_cache")
            check_cache(vc, hkv, dim, "value_cache")
            code = _lib.MXFP4_CODE
        else:
            assert ctype == dtype or ctype == torch.float8_e4m3fn, f"kv cache dtype {ctype} does not match {dtype}"
            assert shape[2] == hkv and shape[3] == dim, f"cache rows {tuple(shape[2:])} for keys ({hkv}, {dim})"
            assert kc.stride(3) == 1 and vc.stride(3) == 1, "cache rows need unit last stride"
            code = _lib.DTYPE_CODES[ctype]
        kcs, vcs = kc.stride(), vc.stride()
        assert slots.dtype == torch.int64 and slots.shape == (n,) and (n <= 1 or slots.stride(0) == 1), \
            f"slot_mapping must be contiguous int64 [{n}]"
        for s in (k_scale, v_scale):
            assert s is None or s.dtype == torch.float32 and s.numel() == 1 and ctype == torch.float8_e4m3fn, \
                "scales are one float32 element each and only apply to an fp8 cache"
        blocks, page = shape[:2]
    for t in (k, v, positions, cos_sin, q_weight, k_weight, kc, vc, slots, k_scale, v_scale):
        assert t is None or t.device == device, "all tensors must be on q's device"
    with on_device(device):
        st = lib().psk_norm_rope(
            q.data_ptr(), k.data_ptr(), ptr(v), q_out.data_ptr(), ptr(k_out), ptr(kc), ptr(vc),
            pack_i64x16(*qs[:2], *ks[:2], *vs[:2], *q_out.stride()[:2], *os[:2], *kcs[:3], *vcs[:3]), _lib.DTYPE_CODES[dtype],
            n, hq, hkv, dim, ptr(q_weight), ptr(k_weight), _lib.DTYPE_CODES[weight_dtype], float(eps), positions.data_ptr(),
            8 if positions.dtype == torch.int64 else 4, ps[0] if axes > 1 else 0, axes, sections, cos_sin.data_ptr(),
            table[0] if known > 1 else rot, known, rot, 1 if interleaved else 0, code, ptr(slots), page, blocks, ptr(k_scale),
            ptr(v_scale), stream_handle(device),
        )
    if st:
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
                None, None, None, "norm_rope")


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
    assert v is not None and key_cache is not None and value_cache is not None and slot_mapping is not None, \
        "the append needs v, both caches and slot_mapping"
    return _run(q, k, v, positions, cos_sin, q_weight, k_weight, eps, sections, interleaved, q_out, k_out, key_cache,
                value_cache, slot_mapping, k_scale, v_scale, "norm_rope_and_cache")[0]
