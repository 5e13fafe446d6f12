"""CPU oracle of the 4-bit KV cache, its attention, and the norms with rotation, in
float64 and integers from the definitions.

A 4-bit row of D elements: D/2 bytes of E2M1 codes (the even element low), D/32 scale
bytes, zeros to a multiple of 4.  The scale of 32 elements is the smallest power of
two s >= 2^-126 with max |x| < 7 s (1 for zeros), the codes x / s to nearest even; a
group with a NaN or an infinity has scale 0xFF and codes 0.
"""

from __future__ import annotations

import numpy as np

GROUP = 32
_VALUES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
# the border between code i and i + 1 belongs to the even one
_BORDERS = (_VALUES[:-1] + _VALUES[1:]) / 2


def entry_bytes(dim: int) -> int:
    return (dim // 2 + dim // GROUP + 3) // 4 * 4


def quantize(x: np.ndarray) -> np.ndarray:
    """uint8 [.., entry] of float64 values [.., D]."""
    x = np.asarray(x, dtype=np.float64)
    d = x.shape[-1]
    g = x.reshape(x.shape[:-1] + (d // GROUP, GROUP))
    bad = ~np.isfinite(g).all(-1)
    a = np.where(bad[..., None], 0.0, np.abs(g))
    top = a.max(-1)
    m, e = np.frexp(top)  # top = m 2^e, 1/2 <= m < 1: top < 7 2^k from k = e - 3 on where m < 7/8
    k = np.where(top == 0, 0, np.maximum(np.where(m < 0.875, e - 3, e - 2), -126))
    r = np.ldexp(a, -k[..., None])
    code = np.zeros(r.shape, dtype=np.uint8)
    for i, border in enumerate(_BORDERS):
        code = np.where((r > border) if i % 2 == 0 else (r >= border), i + 1, code).astype(np.uint8)
    code |= np.where(np.signbit(g), 8, 0).astype(np.uint8)
    code = np.where(bad[..., None], 0, code).astype(np.uint8).reshape(x.shape)
    out = np.zeros(x.shape[:-1] + (entry_bytes(d),), dtype=np.uint8)
    out[..., :d // 2] = code[..., ::2] | (code[..., 1::2] << 4)
    out[..., d // 2:d // 2 + d // GROUP] = np.where(bad, 255, k + 127)
    return out


def dequantize(rows: np.ndarray, dim: int) -> np.ndarray:
    """float64 [.., D] of rows (NaN in groups of scale 0xFF)."""
    code = np.stack([rows[..., :dim // 2] & 15, rows[..., :dim // 2] >> 4], -1).reshape(rows.shape[:-1] + (dim,))
    v = np.where(code & 8, -_VALUES[code & 7], _VALUES[code & 7])
    e = rows[..., dim // 2:dim // 2 + dim // GROUP].astype(np.int64)
    s = np.where(e == 255, np.nan, np.ldexp(1.0, e - 127))
    return v * np.repeat(s, GROUP, -1)


def append(key, value, key_cache, value_cache, slots) -> None:
    """float64 rows [N, H, D] into uint8 caches [P, ps, H, entry]."""
    ps, n = key_cache.shape[1], key_cache.shape[0] * key_cache.shape[1]
    for cache, rows in ((key_cache, quantize(key)), (value_cache, quantize(value))):
        for t, s in enumerate(slots):
            if 0 <= s < n:
                cache[s // ps, s % ps] = rows[t]


def rows_of(cache, table_row, positions):
    """uint8 [n, H, entry]; rows without a page are zeros (of scale 1)."""
    P, ps = cache.shape[:2]
    out = np.zeros((len(positions),) + cache.shape[2:], dtype=np.uint8)
    for i, p in enumerate(positions):
        page = p // ps
        if 0 <= p and page < len(table_row) and 0 <= table_row[page] < P:
            out[i] = cache[table_row[page], p % ps]
    return out


def attention(q, k_cache, v_cache, block_table, seq_lens, cu_q, scale, causal=True):
    """(out float64 [T, Hq, D], lse float64 [T, Hq], largest sum |q K| scaled) of
    float64 queries; rows that see no key: zeros and -inf."""
    T, hq, d = q.shape
    hkv = k_cache.shape[2]
    out, lse, most = np.zeros((T, hq, d)), np.full((T, hq), -np.inf), 0.0
    for b, L in enumerate(seq_lens):
        L = max(int(L), 0)
        first, n = int(cu_q[b]), int(cu_q[b + 1] - cu_q[b])
        if n <= 0:
            continue
        keys = dequantize(rows_of(k_cache, block_table[b], range(L)), d)
        vals = dequantize(rows_of(v_cache, block_table[b], range(L)), d)
        for i in range(n):
            see = max(0, min(L, L - n + 1 + i)) if causal else L
            if see == 0:
                continue
            for h in range(hq):
                kh = keys[:see, h // (hq // hkv)]
                s = kh @ q[first + i, h] * scale
                most = max(most, float(np.nanmax(np.abs(kh) @ np.abs(q[first + i, h])) * abs(scale)) if see else 0.0)
                m = s.max()
                p = np.exp(s - m)
                out[first + i, h] = (p / p.sum()) @ vals[:see, h // (hq // hkv)]
                lse[first + i, h] = m + np.log(p.sum())
    return out, lse, most


def norm_rope(x, positions, cos_sin, weight=None, eps=1e-6, sections=None, interleaved=False):
    """(float64 [N, H, D], the sum of the magnitudes that make each element)."""
    x = np.asarray(x, dtype=np.float64)
    rot = cos_sin.shape[1]
    half = rot // 2
    y = x
    if weight is not None:
        y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(weight, dtype=np.float64)
    positions = np.asarray(positions).reshape(-1, x.shape[0])
    axis = np.repeat(np.arange(len(positions)), sections if sections is not None else [half])
    p = positions[axis].T  # [N, half]
    known = (p >= 0) & (p < cos_sin.shape[0])
    i = np.arange(half)
    t = cos_sin.astype(np.float64)
    at = np.where(known, p, 0)
    c, s = np.where(known, t[at, i], np.nan)[:, None], np.where(known, t[at, half + i], np.nan)[:, None]
    out, size = y.copy(), np.abs(y)
    lo, hi = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, half), slice(half, rot))
    a, b = y[..., lo], y[..., hi]
    out[..., lo], out[..., hi] = a * c - b * s, b * c + a * s
    size[..., lo], size[..., hi] = np.abs(a * c) + np.abs(b * s), np.abs(b * c) + np.abs(a * s)
    return out, size
