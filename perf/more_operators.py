"""Norms with rotation, and a KV cache held in 4 bits, as timed cases.

What a layer does between its projections and its attention's output, over a
paged cache: ``rotary.norm_rope`` and ``rotary.norm_rope_and_cache`` (RMS norm of
every query and key head, the position rotation, and the append in the same
pass), ``mxfp4_kv.reshape_and_cache_mxfp4`` with ``mxfp4_kv.gather_mxfp4`` (the
cache quantized to microscaled 4-bit floats as it is written, and read back) and
``attention.paged_mxfp4_attention`` (decode, a few drafted tokens, prefill).
With ``own`` false every case runs in elementary torch operations in 32 bits.

A 4-bit row is a token's head: D / 2 bytes of two E2M1 codes each (the even
element in the low half), then a scale byte 2^(e - 127) for each 32 elements, and
padding to 4 bytes.

Model shapes: 32 query heads over 8 or 4 kv heads of 128 and their
tensor-parallel shards.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
GROUP = 32
D_ATT = 128


# --------------------------------------------------------------------------- #
# the cases
# --------------------------------------------------------------------------- #


def _rope(tokens, hq, hkv, dim, rot, norm, axes, interleaved, dtype, cache, page, mix=1):
    return {"kind": "rope", "tokens": tokens, "hq": hq, "hkv": hkv, "dim": dim, "rot": rot, "norm": norm, "axes": axes,
            "interleaved": interleaved, "dtype": dtype, "cache": cache, "page": page, "mix": mix}


def _kv4(seqs, new_lo, new_hi, ctx_lo, ctx_hi, heads, dim, page, dtype, mix=1):
    return {"kind": "kv4", "seqs": seqs, "n_lo": new_lo, "n_hi": new_hi, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi,
            "heads": heads, "dim": dim, "page": page, "dtype": dtype, "mix": mix}


def _attn(seqs, n_lo, n_hi, ctx_lo, ctx_hi, hq, hkv, page, mix=1, lse=False):
    return {"kind": "attn", "seqs": seqs, "n_lo": n_lo, "n_hi": n_hi, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi, "hq": hq,
            "hkv": hkv, "page": page, "mix": mix, "lse": lse}


def listed():
    return [
        # A decode batch of one layer: every head normed and rotated, K and V appended.
        {"name": "rope_decode"} | _rope(64, 32, 8, 128, 128, True, 1, False, "bf16", True, 16),
        # A prompt of one layer.
        {"name": "rope_prompt"} | _rope(8192, 32, 8, 128, 128, True, 1, False, "bf16", True, 16, mix=2),
        # Images and video beside text: three axes of positions, no norm, a tensor-parallel shard, fp16.
        {"name": "rope_axes"} | _rope(20011, 8, 2, 128, 128, False, 3, False, "f16", False, 16, mix=3),
        # One short request extends its 4-bit cache by a few tokens and reads it back: latency.
        {"name": "kv4_short"} | _kv4(1, 17, 17, 600, 600, 8, 128, 16, "bf16"),
        # A chunk of two long prompts written, their whole contexts read back.
        {"name": "kv4_chunk"} | _kv4(2, 2048, 2048, 14000, 43000, 8, 128, 16, "bf16", mix=4),
        # Many short requests, heads of 64 (whose rows are padded), pages of 24.
        {"name": "kv4_ragged"} | _kv4(100, 1, 40, 1, 700, 5, 64, 24, "f16", mix=5),
        # One request decodes alone over a short context: latency.
        {"name": "attn_alone"} | _attn(1, 1, 1, 1000, 1000, 32, 8, 16),
        # A decode batch over mixed contexts.
        {"name": "attn_decode"} | _attn(64, 1, 1, 512, 32768, 32, 8, 16, mix=2),
        # Two very long contexts, 8 query heads a kv head, pages of 64.
        {"name": "attn_long"} | _attn(2, 1, 1, 150000, 200000, 32, 4, 64, mix=3),
        # Drafted tokens of many requests on a tensor-parallel shard, contexts down to a few tokens, pages of 24.
        {"name": "attn_drafts"} | _attn(48, 1, 4, 3, 6000, 8, 1, 24, mix=9, lse=True),
        # A chunk of a long prompt over its cached prefix.
        {"name": "attn_chunk"} | _attn(1, 2048, 2048, 30000, 30000, 32, 8, 16),
        # Fresh prompts of mixed lengths, packed.
        {"name": "attn_prompts"} | _attn(8, 100, 4000, 0, 0, 32, 8, 16, mix=6),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    case = _draw(rng)
    while work(case)["flops"] > 1.0e12 or work(case)["bytes"] > 3.0e8:
        for k in ("tokens", "ctx_lo", "ctx_hi", "n_hi"):
            if k in case:
                case[k] = max(case.get("n_lo", 1) if k == "n_hi" else 1, case[k] * 3 // 4)
        if "n_lo" in case:
            case["n_lo"] = min(case["n_lo"], max(1, case["n_hi"] * 3 // 4))
    return case


def _draw(rng):
    kind = rng.choice(["rope", "kv4", "attn", "attn"])
    page = rng.choice([16, 16, 16, 32, 64, 24])
    mix = rng.randrange(1, 1 << 20)
    if kind == "rope":
        hq, hkv, dim = rng.choice([(32, 8, 128), (32, 4, 128), (8, 1, 128), (16, 2, 128), (12, 4, 64), (8, 2, 256)])
        axes = rng.choice([1, 1, 3])
        return _rope(_log_int(rng, 1, 20000), hq, hkv, dim, rng.choice([dim, dim, dim // 2]), rng.random() < 0.6, axes,
                     rng.random() < 0.3, rng.choice(["bf16", "bf16", "f16"]), rng.random() < 0.6, page, mix)
    if kind == "kv4":
        seqs, hi = _log_int(rng, 1, 100), _log_int(rng, 1, 45000)
        n_hi = _log_int(rng, 1, 2000)
        return _kv4(seqs, rng.choice([1, n_hi]), n_hi, max(1, hi // rng.choice([1, 4, 32])), hi, rng.choice([1, 2, 4, 5, 8]),
                    rng.choice([128, 128, 64, 96]), page, rng.choice(["bf16", "bf16", "f16", "f32"]), mix)
    hq, hkv = rng.choice([(32, 8), (32, 8), (32, 4), (16, 4), (8, 2), (8, 1), (16, 2), (4, 4), (12, 6), (40, 10)])
    form = rng.choice(["decode", "decode", "drafts", "chunk", "prompts"])
    if form == "prompts":
        seqs = _log_int(rng, 1, 16)
        n_hi = _log_int(rng, 5, 4000)
        return _attn(seqs, max(1, n_hi // rng.choice([1, 8, 64])), n_hi, 0, 0, hq, hkv, page, mix, rng.random() < 0.5)
    seqs = _log_int(rng, 1, 64)
    n_hi = {"decode": 1, "drafts": _log_int(rng, 2, 16), "chunk": _log_int(rng, 17, 2048)}[form]
    hi = min(_log_int(rng, 16, 200000), 1200000 // seqs)
    return _attn(seqs, rng.choice([1, n_hi, n_hi]), n_hi, max(1, hi // rng.choice([1, 4, 32])), hi, hq, hkv, page, mix,
                 rng.random() < 0.5)


# --------------------------------------------------------------------------- #
# shapes that follow from a case alone
# --------------------------------------------------------------------------- #


def _counts(case):
    """(new tokens, cached tokens with them) of each sequence."""
    r = random.Random(case["mix"])
    lo, hi = case["ctx_lo"], case["ctx_hi"]
    ctx = [hi] * case["seqs"] if hi <= lo else [
        int(math.exp(r.uniform(math.log(max(lo, 1)), math.log(hi)))) for _ in range(case["seqs"])]
    n = [r.randint(case["n_lo"], case["n_hi"]) for _ in range(case["seqs"])]
    return n, [c + k for c, k in zip(ctx, n)]


def _entry(dim):
    return (dim // 2 + dim // GROUP + 3) // 4 * 4


def _sections(case):
    """Pairs of the rotation that go by each axis (time, height, width: 1/4, 3/8, 3/8)."""
    half = case["rot"] // 2
    if case["axes"] == 1:
        return [half]
    return [half // 4, half * 3 // 8, half - half // 4 - half * 3 // 8]


# --------------------------------------------------------------------------- #
# prepare
# --------------------------------------------------------------------------- #

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_MAX_POS = 40960


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _cumulative(values):
    out = [0]
    for v in values:
        out.append(out[-1] + v)
    return out


def _tables(g, lens, page):
    """A random page table over the lengths (page 0 is none of theirs), and the page after them."""
    need = [-(-n // page) for n in lens]
    perm = (torch.randperm(sum(need), generator=g, device=DEV) + 1).to(torch.int32)
    table = torch.zeros(len(lens), max(need + [1]), dtype=torch.int32, device=DEV)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = perm[at:at + k]
        at += k
    return table, 1 + sum(need)


def _cos_sin(rot):
    """[positions, rot] float32: cosines, then sines, of the angles in 64 bits."""
    freq = 1.0e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)
    angle = torch.arange(_MAX_POS, dtype=torch.float64, device=DEV)[:, None] * freq
    return torch.cat([torch.cos(angle), torch.sin(angle)], 1).float()


def _prepare_rope(case, seed):
    g = _gen(seed)
    n, hq, hkv, d, page = case["tokens"], case["hq"], case["hkv"], case["dim"], case["page"]
    qkv = (torch.randn(n, (hq + 2 * hkv) * d, generator=g, device=DEV) * 1.5).to(_TYPES[case["dtype"]])
    q, k, v = qkv.split([hq * d, hkv * d, hkv * d], 1)
    pos = torch.randint(0, _MAX_POS, (case["axes"], n), generator=g, device=DEV)
    s = {"kind": "rope", "q": q.view(n, hq, d), "k": k.view(n, hkv, d), "v": v.view(n, hkv, d),
         "pos": pos[0].contiguous() if case["axes"] == 1 else pos, "table": _cos_sin(case["rot"]),
         "sections": _sections(case) if case["axes"] > 1 else None, "interleaved": case["interleaved"], "qw": None,
         "kw": None, "cache": None}
    if case["norm"]:
        s["qw"] = (1.0 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(q.dtype)
        s["kw"] = (1.0 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(q.dtype)
    if case["cache"]:
        pages = -(-n // page) + 2
        s["cache"] = torch.randn(pages, 2, page, hkv, d, generator=g, device=DEV).to(q.dtype)
        s["slots"] = torch.randperm(pages * page, generator=g, device=DEV)[:n]
        s["slots"][5::37] = -1  # a graph's padding
    return s


def _random_rows(g, pages, page, heads, dim):
    """A cache of 4-bit rows of values ~N(0, 1)."""
    cache = torch.empty(pages, 2, page, heads, _entry(dim), dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 25) // (2 * page * heads * dim))
    for i in range(0, pages, step):
        part = cache[i:i + step]
        part.copy_(_pack(torch.randn(part.shape[:-1] + (dim,), generator=g, device=DEV)))
    return cache


def _prepare_kv4(case, seed):
    g = _gen(seed)
    n, lens = _counts(case)
    heads, d, page = case["heads"], case["dim"], case["page"]
    table, pages = _tables(g, lens, page)
    cache = _random_rows(g, pages, page, heads, d)
    dtype = _TYPES[case["dtype"]]
    # heads of different sizes, as keys have them
    size = torch.exp(torch.randn(heads, d, generator=g, device=DEV) * 0.7)
    k = (torch.randn(sum(n), heads, d, generator=g, device=DEV) * size).to(dtype)
    v = (torch.randn(sum(n), heads, d, generator=g, device=DEV) * 0.3).to(dtype)
    slots = []
    for b, (m, L) in enumerate(zip(n, lens)):
        pos = torch.arange(L - m, L, device=DEV)
        slots.append(table[b, pos // page].long() * page + pos % page)
    return {"kind": "kv4", "k": k, "v": v, "slots": torch.cat(slots), "kc": cache[:, 0], "vc": cache[:, 1], "table": table,
            "cu": _i32(_cumulative(lens)), "lens": lens, "out": (sum(lens), heads, d), "dtype": dtype}


def _prepare_attn(case, seed):
    g = _gen(seed)
    n, lens = _counts(case)
    table, pages = _tables(g, lens, case["page"])
    cache = _random_rows(g, pages, case["page"], case["hkv"], D_ATT)
    # logits of standard deviation 2
    q = (torch.randn(sum(n), case["hq"], D_ATT, generator=g, device=DEV) * 2.0).to(torch.bfloat16)
    return {"kind": "attn", "q": q, "kc": cache[:, 0], "vc": cache[:, 1], "table": table, "seq_lens": _i32(lens),
            "cu": _i32(_cumulative(n)), "n": n, "lens": lens, "max_q": max(n), "max_k": max(lens),
            "scale": D_ATT ** -0.5, "lse": case["lse"]}


def prepare(case, seed):
    return {"rope": _prepare_rope, "kv4": _prepare_kv4, "attn": _prepare_attn}[case["kind"]](case, seed)


# --------------------------------------------------------------------------- #
# run
# --------------------------------------------------------------------------- #


def run(s):
    if not own:
        return {"rope": _plain_rope, "kv4": _plain_kv4, "attn": _plain_attn}[s["kind"]](s)
    from pipeswift_amd import attention, mxfp4_kv, rotary
    if s["kind"] == "rope":
        if s["cache"] is None:
            return rotary.norm_rope(s["q"], s["k"], s["pos"], s["table"], q_weight=s["qw"], k_weight=s["kw"],
                                    sections=s["sections"], interleaved=s["interleaved"])
        q = rotary.norm_rope_and_cache(
            s["q"], s["k"], s["v"], s["cache"][:, 0], s["cache"][:, 1], s["slots"], s["pos"], s["table"],
            q_weight=s["qw"], k_weight=s["kw"], sections=s["sections"], interleaved=s["interleaved"])
        return q, s["cache"]
    if s["kind"] == "kv4":
        mxfp4_kv.reshape_and_cache_mxfp4(s["k"], s["v"], s["kc"], s["vc"], s["slots"])
        k = torch.empty(s["out"], dtype=s["dtype"], device=DEV)
        v = torch.empty_like(k)
        mxfp4_kv.gather_mxfp4(s["kc"], k, s["table"], s["cu"], src_cache_v=s["vc"], dst_v=v)
        return k, v
    return attention.paged_mxfp4_attention(
        s["q"], s["kc"], s["vc"], s["table"], s["seq_lens"], s["cu"], s["max_q"], softmax_scale=s["scale"],
        return_softmax_lse=s["lse"], max_seq_len=s["max_k"])


def _rotated(x, w, s):
    """float32 of a tensor's heads, normed and rotated."""
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.float()
    rot = s["table"].shape[1]
    half = rot // 2
    if s["sections"] is None:
        cs = s["table"][s["pos"]]
        cos, sin = cs[:, :half], cs[:, half:]
    else:
        axis = torch.cat([torch.full((m,), a) for a, m in enumerate(s["sections"])]).to(DEV)
        i = torch.arange(half, device=DEV)
        at = s["pos"][axis].t()  # [N, half]
        cos, sin = s["table"][at, i], s["table"][at, half + i]
    cos, sin = cos[:, None], sin[:, None]
    a, b = (x[..., :rot:2], x[..., 1:rot:2]) if s["interleaved"] else (x[..., :half], x[..., half:rot])
    y = x.clone()
    if s["interleaved"]:
        y[..., :rot:2], y[..., 1:rot:2] = a * cos - b * sin, b * cos + a * sin
    else:
        y[..., :half], y[..., half:rot] = a * cos - b * sin, b * cos + a * sin
    return y


def _plain_rope(s):
    q = _rotated(s["q"], s["qw"], s).to(s["q"].dtype)
    k = _rotated(s["k"], s["kw"], s).to(s["k"].dtype)
    if s["cache"] is None:
        return q, k
    cache, page = s["cache"], s["cache"].shape[2]
    live = (s["slots"] >= 0)[:, None, None]
    # rows without a slot repeat the first row's write (its slot is one)
    at = torch.where(s["slots"] >= 0, s["slots"], s["slots"][:1])
    for half, rows in ((0, k), (1, s["v"])):
        cache[at // page, half, at % page] = torch.where(live, rows, rows[:1])
    return q, cache


def _power(e):
    """float32 2^e of integers, -126 <= e <= 127."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _pack(x):
    """The 4-bit rows [.., entry] of float32 [.., D]."""
    d = x.shape[-1]
    g = x.unflatten(-1, (d // GROUP, GROUP))
    m, e = torch.frexp(g.abs().amax(-1))
    # the smallest power of two s with max |x| < 7 s (1 for a group of zeros)
    e = torch.where(m == 0, 0, torch.where(m < 0.875, e - 3, e - 2).clamp(min=-126))
    a = g.abs() / _power(e)[..., None]
    two, four = a >= 2.0, a >= 4.0
    step = torch.where(four, 2.0, torch.where(two, 1.0, 0.5))
    code = torch.round(a / step).to(torch.uint8) + 2 * two.to(torch.uint8) + 2 * four.to(torch.uint8)
    code = (code | (torch.signbit(g).to(torch.uint8) << 3)).flatten(-2)
    out = torch.zeros(x.shape[:-1] + (_entry(d),), dtype=torch.uint8, device=x.device)
    out[..., :d // 2] = code[..., ::2] | (code[..., 1::2] << 4)
    out[..., d // 2:d // 2 + d // GROUP] = (e + 127).to(torch.uint8)
    return out


def _unpack(rows, d):
    """float32 [.., D] of 4-bit rows."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=rows.device)
    table = torch.cat([table, -table])
    raw = rows[..., :d // 2]
    x = torch.stack([table[(raw & 15).long()], table[(raw >> 4).long()]], -1).flatten(-2)
    scale = _power(rows[..., d // 2:d // 2 + d // GROUP].to(torch.int32) - 127)
    return (x.unflatten(-1, (d // GROUP, GROUP)) * scale[..., None]).flatten(-2)


def _cached(cache, table_row, count, dim):
    """float32 [count, H, D] of a sequence's first rows."""
    pos = torch.arange(count, device=DEV)
    return _unpack(cache[table_row[pos // cache.shape[1]].long(), pos % cache.shape[1]], dim)


def _plain_kv4(s):
    page, d = s["kc"].shape[1], s["k"].shape[2]
    for cache, x in ((s["kc"], s["k"]), (s["vc"], s["v"])):
        cache[s["slots"] // page, s["slots"] % page] = _pack(x.float())
    return tuple(torch.cat([_cached(c, s["table"][b], L, d).to(s["dtype"]) for b, L in enumerate(s["lens"])])
                 for c in (s["kc"], s["vc"]))


def _plain_attn(s):
    hq, hkv = s["q"].shape[1], s["kc"].shape[2]
    out = torch.empty_like(s["q"])
    lse = torch.empty(hq, s["q"].shape[0], device=DEV)
    at = 0
    for b, (n, L) in enumerate(zip(s["n"], s["lens"])):
        keys = _cached(s["kc"], s["table"][b], L, D_ATT).permute(1, 2, 0).contiguous()  # [Hkv, D, L]
        vals = _cached(s["vc"], s["table"][b], L, D_ATT).permute(1, 0, 2).contiguous()  # [Hkv, L, D]
        q = s["q"][at:at + n].float().view(n, hkv, hq // hkv, D_ATT).permute(1, 2, 0, 3).reshape(hkv, -1, D_ATT)
        x = torch.bmm(q, keys) * s["scale"]
        last = (L - n + torch.arange(n, device=DEV)).repeat(hq // hkv)  # of each row [G, n]
        x.masked_fill_(torch.arange(L, device=DEV)[None] > last[:, None], float("-inf"))
        top = x.amax(-1, keepdim=True)
        p = torch.exp(x.sub_(top))
        total = p.sum(-1, keepdim=True)
        o = torch.bmm(p, vals) / total
        out[at:at + n] = o.view(hkv, -1, n, D_ATT).permute(2, 0, 1, 3).reshape(n, hq, D_ATT).to(out.dtype)
        lse[:, at:at + n] = (top + torch.log(total)).view(hq, n)
        at += n
    return (out, lse) if s["lse"] else out


# --------------------------------------------------------------------------- #
# work
# --------------------------------------------------------------------------- #


def work(case):
    if case["kind"] == "rope":
        n, d = case["tokens"], case["dim"]
        rows = case["hq"] + (2 if case["cache"] else 1) * case["hkv"]
        return {"bytes": n * (2 * rows * d * 2 + 4 * case["rot"] + 8 * case["axes"] + (8 if case["cache"] else 0)),
                "flops": n * (case["hq"] + case["hkv"]) * (3 * case["rot"] + (4 * d if case["norm"] else 0))}
    n, lens = _counts(case)
    pages = sum(-(-L // case["page"]) for L in lens)
    if case["kind"] == "kv4":
        size = 4 if case["dtype"] == "f32" else 2
        row, entry = case["dim"] * size, _entry(case["dim"])
        # the new rows quantized and written, every row read and expanded
        return {"bytes": 2 * case["heads"] * (sum(n) * (row + entry) + sum(lens) * (entry + row)) + 8 * sum(n) + 4 * pages,
                "flops": 0}
    pairs = sum(k * (L - k) + k * (k + 1) // 2 for k, L in zip(n, lens))
    return {"bytes": sum(lens) * case["hkv"] * 2 * _entry(D_ATT) + sum(n) * case["hq"] * (4 * D_ATT + (4 if case["lse"] else 0))
            + 4 * pages, "flops": 4 * D_ATT * case["hq"] * pairs}


# --------------------------------------------------------------------------- #
# exact: from the definitions, in 64 bits
# --------------------------------------------------------------------------- #


def _exact_rope(case, s):
    def turn(x, w):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt(torch.mean(x ** 2, -1, keepdim=True) + 1e-6) * w.double()
        rot = case["rot"]
        pos = s["pos"][None] if case["axes"] == 1 else s["pos"]
        y = x.clone()
        i = 0
        for a, count in enumerate(_sections(case)):
            for _ in range(count):
                c, z = s["table"][pos[a], i].double()[:, None], s["table"][pos[a], rot // 2 + i].double()[:, None]
                u, w2 = (2 * i, 2 * i + 1) if case["interleaved"] else (i, rot // 2 + i)
                y[:, :, u] = x[:, :, u] * c - x[:, :, w2] * z
                y[:, :, w2] = x[:, :, w2] * c + x[:, :, u] * z
                i += 1
        return y

    q, k = turn(s["q"], s["qw"]), turn(s["k"], s["kw"])
    if not case["cache"]:
        return q, k
    cache = s["cache"].double()
    live = s["slots"] >= 0
    at = s["slots"][live]
    cache[at // case["page"], 0, at % case["page"]] = k[live]
    cache[at // case["page"], 1, at % case["page"]] = s["v"][live].double()
    return q, cache


def _exact_power(e):
    """float64 2^e of int64."""
    return ((e + 1023) << 52).view(torch.float64)


def _exact_values(rows, d):
    """float64 values of 4-bit rows, from the fields of their codes."""
    raw = rows[..., :d // 2].long()
    code = torch.empty(rows.shape[:-1] + (d,), dtype=torch.int64, device=rows.device)
    code[..., 0::2], code[..., 1::2] = raw % 16, raw // 16
    sign, exponent, fraction = code // 8, code // 2 % 4, code % 2
    size = torch.where(exponent == 0, 0.5 * fraction.double(), (1.0 + 0.5 * fraction) * _exact_power(exponent - 1))
    scale = _exact_power(rows[..., d // 2:d // 2 + d // GROUP].long() - 127)
    return torch.where(sign == 1, -size, size) * scale.repeat_interleave(GROUP, -1)


def _exact_quantized(x):
    """float64 x as the 4-bit row holds it, by the borders between its values."""
    g = x.double().unflatten(-1, (-1, GROUP))
    top = g.abs().amax(-1, keepdim=True)
    size = _exact_power((torch.where(top > 0, top, 4.0).contiguous().view(torch.int64) >> 52) - 1023)  # 2^floor(log2 top)
    scale = torch.where(top < 1.75 * size, size / 4.0, size / 2.0).clamp(min=2.0 ** -126)
    a = g.abs() / scale
    v = torch.zeros_like(a)
    for value, border, inside in ((0.5, 0.25, False), (1.0, 0.75, True), (1.5, 1.25, False), (2.0, 1.75, True),
                                  (3.0, 2.5, False), (4.0, 3.5, True), (6.0, 5.0, False)):
        v = torch.where(a >= border if inside else a > border, value, v)
    return (torch.sign(g) * v * scale).flatten(-2)


def _exact_kv4(case, s):
    n, lens = _counts(case)
    outs = []
    for cache, x in ((s["kc"], s["k"]), (s["vc"], s["v"])):
        new, parts, at = _exact_quantized(x), [], 0
        for b, (m, L) in enumerate(zip(n, lens)):
            pos = torch.arange(L - m, device=DEV)
            rows = cache[s["table"][b, pos // case["page"]].long(), pos % case["page"]]
            parts += [_exact_values(rows, case["dim"]), new[at:at + m]]
            at += m
        outs.append(torch.cat(parts))
    return tuple(outs)


def _exact_attn(case, s):
    n, lens = _counts(case)
    hq, hkv, page = case["hq"], case["hkv"], case["page"]
    out = torch.empty(sum(n), hq, D_ATT, dtype=torch.float64, device=DEV)
    lse = torch.empty(hq, sum(n), dtype=torch.float64, device=DEV)
    at = 0
    for b, (k, L) in enumerate(zip(n, lens)):
        pos = torch.arange(L, device=DEV)
        slot = s["table"][b, pos // page].long(), pos % page
        hidden = pos[None] > (L - k + torch.arange(k, device=DEV))[:, None]
        for h in range(hkv):
            keys, vals = (_exact_values(c[slot[0], slot[1], h], D_ATT) for c in (s["kc"], s["vc"]))
            for hh in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                x = (s["q"][at:at + k, hh].double() @ keys.t() * s["scale"]).masked_fill(hidden, float("-inf"))
                norm = torch.logsumexp(x, 1)
                out[at:at + k, hh] = torch.exp(x - norm[:, None]) @ vals
                lse[hh, at:at + k] = norm
        at += k
    return (out, lse) if case["lse"] else out


def exact(case, seed):
    return {"rope": _exact_rope, "kv4": _exact_kv4, "attn": _exact_attn}[case["kind"]](case, prepare(case, seed))
