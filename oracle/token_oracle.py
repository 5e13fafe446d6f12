"""CPU oracle of the operators on single cached tokens -- TEST INFRASTRUCTURE ONLY.

Tree attention and the accumulated attention weights in float64, the choice of
an eviction and the moves of kept and committed rows, each restated from its
definition with plain loops over sequences.  Pinned in tests/test_token_oracle.py
against torch's masked softmax, the causal oracle and literal tiny cases.
"""

from __future__ import annotations

import numpy as np

from .kv_oracle import e4m3fn_to_f32, quantize_e4m3, to_f32


def _cached(cache, pages_row, count, head):
    """float64 [count, D] of a sequence's first rows; rows on missing pages are zeros."""
    P, ps = cache.shape[:2]
    j = np.arange(count)
    pages = np.full(count, -1, dtype=np.int64)
    inside = j // ps < len(pages_row)
    pages[inside] = np.asarray(pages_row, dtype=np.int64)[j[inside] // ps]
    ok = (pages >= 0) & (pages < P)
    rows = np.zeros((count, cache.shape[3]), dtype=np.float64)
    rows[ok] = e4m3fn_to_f32(cache[pages[ok], (j % ps)[ok], head]).astype(np.float64)
    return rows


def _queries(q, q_dtype, qd):
    if q_dtype == "fp8":
        return e4m3fn_to_f32(q).astype(np.float64)
    return e4m3fn_to_f32(quantize_e4m3(to_f32(q, q_dtype), qd)).astype(np.float64)


def _descales(d, B, Hkv):
    return np.ones((B, Hkv), np.float32) if d is None else np.asarray(d, dtype=np.float32)


def tree_visible(mask_rows, n, length):
    """bool [n, length]: drafted token i sees the keys before the n drafted ones
    and drafted key t where bit t % 64 of word t // 64 of its mask is set."""
    see = np.zeros((n, length), dtype=bool)
    for i in range(n):
        for p in range(length):
            t = p - (length - n)
            see[i, p] = t < 0 or bool((int(mask_rows[i, t // 64]) >> (t % 64)) & 1)
    return see


def causal_visible(n, length, causal=True):
    p, i = np.arange(length)[None, :], np.arange(n)[:, None]
    return p <= length - n + i if causal else np.ones((n, length), dtype=bool)


def _sequences(q, q_dtype, k_cache, block_table, seq_lens, cu, scale, qd_all, kd_all):
    """Per sequence and kv head: (b, h, first row, n, s [n, G, L] in float64, its
    absolute-value bound sum |q~ K| scale, descaled)."""
    Hkv, G = k_cache.shape[2], q.shape[1] // k_cache.shape[2]
    for b in range(len(cu) - 1):
        c0, n, L = int(cu[b]), int(cu[b + 1] - cu[b]), int(seq_lens[b])
        for h in range(Hkv):
            qd, kd = float(qd_all[b, h]), float(kd_all[b, h])
            K = _cached(k_cache, block_table[b], L, h)
            qq = _queries(q[c0:c0 + n, h * G:(h + 1) * G], q_dtype, qd)
            f = float(np.float32(scale)) * qd * kd
            with np.errstate(invalid="ignore"):
                yield b, h, c0, n, (qq @ K.T) * f, float((np.abs(qq) @ np.abs(K).T).max(initial=0.0)) * abs(f)


def tree_attention(q, q_dtype, k_cache, v_cache, block_table, seq_lens, mask, cu, scale, q_descale=None, k_descale=None,
                   v_descale=None):
    """(out [TQ, Hq, D], lse [TQ, Hq], bound) in float64 of paged_tree_attention;
    mask: int64 [TQ, words].  bound: the largest sum |q~ K| of a score, scaled.
    Rows that see no key, or that no sequence owns: zeros and -inf."""
    TQ, Hq, D = q.shape
    Hkv, G, B = k_cache.shape[2], Hq // k_cache.shape[2], len(cu) - 1
    qd, kd, vd = (_descales(d, B, Hkv) for d in (q_descale, k_descale, v_descale))
    out, lse, bound = np.zeros((TQ, Hq, D)), np.full((TQ, Hq), -np.inf), 0.0
    for b, h, c0, n, s, most in _sequences(q, q_dtype, k_cache, block_table, seq_lens, cu, scale, qd, kd):
        bound = max(bound, most)
        L = s.shape[2]
        see = tree_visible(np.asarray(mask)[c0:c0 + n], n, L)
        V = _cached(v_cache, block_table[b], L, h)
        for i in range(n):
            if not see[i].any():
                continue
            x = s[i][:, see[i]]
            m = x.max(axis=1, keepdims=True)
            p = np.exp(x - m)
            den = p.sum(axis=1, keepdims=True)
            out[c0 + i, h * G:(h + 1) * G] = (p @ V[see[i]]) / den * float(vd[b, h])
            lse[c0 + i, h * G:(h + 1) * G] = (m + np.log(den))[:, 0]
    return out, lse, bound


def attention_weights(scores, q, q_dtype, k_cache, lse, block_table, seq_lens, cu, scale, q_descale=None,
                      k_descale=None, causal=True, decay=1.0):
    """(new scores [S, Hkv, width] in float64, bound, largest |s|) of
    accumulate_attention_weights; lse: float32 [Hq, TQ]."""
    Hkv, G, B = k_cache.shape[2], q.shape[1] // k_cache.shape[2], len(cu) - 1
    qd, kd = (_descales(d, B, Hkv) for d in (q_descale, k_descale))
    new, bound, most_s = np.asarray(scores, dtype=np.float64).copy(), 0.0, 0.0
    for b, h, c0, n, s, most in _sequences(q, q_dtype, k_cache, block_table, seq_lens, cu, scale, qd, kd):
        bound = max(bound, most)
        L = min(s.shape[2], new.shape[2])
        if s.size:
            most_s = max(most_s, float(np.abs(s).max()))
        see = causal_visible(n, s.shape[2], causal)
        ls = np.asarray(lse, dtype=np.float64)[h * G:(h + 1) * G, c0:c0 + n].T  # [n, G]
        w = np.where(see[:, None, :], np.exp(s - ls[:, :, None]), 0.0).sum((0, 1))[:L]
        old = 0.0 if decay == 0.0 else new[b, h, :L] * float(np.float32(decay))
        new[b, h, :L] = old + w
    return new, bound, most_s


def select_tokens(scores, seq_lens, budget, sink, recent):
    """(kept [L, B, H, budget] with -1 past the last, new_lens [B], list of the
    kept positions) of evict_tokens."""
    layers, B, H, width = scores.shape
    kept = np.full((layers, B, H, budget), -1, dtype=np.int32)
    new_lens = np.array([min(max(int(seq_lens[b]), 0), width, budget) for b in range(B)], dtype=np.int32)
    for layer in range(layers):
        for b in range(B):
            n = min(max(int(seq_lens[b]), 0), width)
            for h in range(H):
                if n <= budget:
                    keep = list(range(n))
                else:
                    free = range(sink, n - recent)
                    x = scores[layer, b, h]
                    # NaN below every number; larger first, then the lower position
                    order = sorted(free, key=lambda i: (1, 0.0, i) if np.isnan(x[i]) else (0, -float(x[i]), i))
                    keep = sorted(list(range(sink)) + order[:budget - sink - recent] + list(range(n - recent, n)))
                kept[layer, b, h, :len(keep)] = keep
    return kept, new_lens


def evict_tokens(caches, scores, block_table, seq_lens, dst_block_table, budget, sink, recent):
    """evict_tokens on host copies: moves rows of ``caches`` ([L, P, ps, H, ...],
    in place) and returns (kept, new_lens, scores_out)."""
    kept, new_lens = select_tokens(scores, seq_lens, budget, sink, recent)
    out = np.array(scores, copy=True)
    layers, B, H, width = scores.shape
    for layer in range(layers):
        for b in range(B):
            n = min(max(int(seq_lens[b]), 0), width)
            for h in range(H):
                k = kept[layer, b, h][kept[layer, b, h] >= 0]
                out[layer, b, h, :n] = 0.0
                out[layer, b, h, :len(k)] = scores[layer, b, h, k]
    for cache in caches:
        old = cache.copy()
        P, ps, heads = cache.shape[1:4]
        for layer in range(layers):
            for b in range(B):
                for h in range(heads):
                    for i, p in enumerate(kept[layer, b, h if H > 1 else 0]):
                        to = int(dst_block_table[b, i // ps]) if p >= 0 else -1
                        if not 0 <= to < P:
                            continue
                        page = int(block_table[b, p // ps]) if p // ps < block_table.shape[1] else -1
                        cache[layer, to, i % ps, h] = old[layer, page, p % ps, h] if 0 <= page < P else 0
    return kept, new_lens, out


def commit_draft_tokens(cache, block_table, starts, path, path_lens):
    """commit_draft_tokens on a host copy [L, P, ps, ...], in place."""
    old = cache.copy()
    P, ps = cache.shape[1:3]

    def at(b, p):
        page = int(block_table[b, p // ps]) if p // ps < block_table.shape[1] else -1
        return (page, p % ps) if 0 <= page < P else None

    for b in range(len(starts)):
        for i in range(min(int(path_lens[b]), path.shape[1])):
            t = int(path[b, i])
            if t < 0 or starts[b] < 0:
                continue
            src, dst = at(b, int(starts[b]) + t), at(b, int(starts[b]) + i)
            if src and dst:
                cache[:, dst[0], dst[1]] = old[:, src[0], src[1]]
