"""Tree attention, attention-weight eviction and draft commits over the paged KV cache, as timed cases.

The operators a serving engine calls beside the append and the readers:
``attention.paged_tree_attention`` (verification of a drafted tree),
``attention.accumulate_attention_weights`` with ``cache_ops.evict_tokens``
(a cache kept to a budget by the weights its tokens receive) and
``cache_ops.commit_draft_tokens`` (the accepted path becomes the sequence).
With ``own`` false every case runs in elementary torch operations in 32 bits.

Model shapes: 32 query heads over 8 or 4 kv heads of 128, their
tensor-parallel shards, and the 576-element latent row.
"""

from __future__ import annotations

import math
import random

import torch

own = False

D = 128
LATENT = 576
DEV = "cuda"


# --------------------------------------------------------------------------- #
# the cases
# --------------------------------------------------------------------------- #


def _tree(seqs, n_lo, n_hi, ctx_lo, ctx_hi, hq, hkv, page, q="bf16", mix=1, lse=False):
    return {"kind": "tree", "seqs": seqs, "n_lo": n_lo, "n_hi": n_hi, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi, "hq": hq,
            "hkv": hkv, "page": page, "q": q, "mix": mix, "lse": lse}


def _weights(seqs, n_lo, n_hi, ctx_lo, ctx_hi, hq, hkv, page, q="bf16", mix=1, decay=1.0):
    return {"kind": "weights", "seqs": seqs, "n_lo": n_lo, "n_hi": n_hi, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi, "hq": hq,
            "hkv": hkv, "page": page, "q": q, "mix": mix, "decay": decay}


def _evict(layers, seqs, lo, hi, budget, sink, recent, heads, shared, page, cache, mix=1):
    return {"kind": "evict", "layers": layers, "seqs": seqs, "ctx_lo": lo, "ctx_hi": hi, "budget": budget, "sink": sink,
            "recent": recent, "heads": heads, "shared": shared, "page": page, "cache": cache, "mix": mix}


def _commit(layers, seqs, n, depth, heads, page, cache, mix=1):
    return {"kind": "commit", "layers": layers, "seqs": seqs, "n": n, "depth": depth, "heads": heads, "page": page,
            "cache": cache, "mix": mix}


def listed():
    return [
        # One request alone verifies a small tree over a short context: latency.
        {"name": "tree_alone"} | _tree(1, 8, 8, 1000, 1000, 32, 8, 16),
        # A decode batch, 16 drafted tokens each over mixed contexts.
        {"name": "tree_batch"} | _tree(32, 16, 16, 512, 16384, 32, 8, 16, q="fp8", mix=5),
        # Few long contexts with wide trees, 8 query heads a kv head: the most rows per key.
        {"name": "tree_wide"} | _tree(4, 61, 61, 20000, 60000, 32, 4, 64, mix=3),
        # A tensor-parallel shard, trees of 1 to 33 tokens over contexts down to a few tokens, pages of 24.
        {"name": "tree_ragged"} | _tree(48, 1, 33, 3, 6000, 8, 1, 24, mix=9, lse=True),
        # After a decode step: one query token a sequence adds its weights to the running sums.
        {"name": "weights_decode"} | _weights(64, 1, 1, 128, 32768, 32, 8, 16, mix=2),
        # After a prompt: the last 64 queries of each sequence score its whole context.
        {"name": "weights_window"} | _weights(4, 64, 64, 8000, 32000, 32, 4, 16, mix=4, decay=0.0),
        # A whole prompt scores itself, causally.
        {"name": "weights_prompt"} | _weights(1, 2000, 2000, 0, 0, 32, 8, 16, q="fp8"),
        # One layer of a single short sequence passes its budget: latency.
        {"name": "evict_alone"} | _evict(1, 1, 1100, 1100, 1024, 4, 64, 8, False, 16, "fp8"),
        # Long prompts compressed in every layer, each kv head its own tokens.
        {"name": "evict_prompts"} | _evict(32, 2, 9000, 16000, 2048, 4, 128, 8, False, 16, "fp8", mix=6),
        # One very long context, bf16 cache, one choice for all heads.
        {"name": "evict_long"} | _evict(4, 1, 131072, 131072, 8192, 16, 1024, 4, True, 64, "bf16"),
        # The accepted paths of a verified batch, every layer of a GQA stack.
        {"name": "commit_batch"} | _commit(32, 32, 16, 6, 8, 16, "fp8", mix=7),
        # The same for a latent cache of 61 layers.
        {"name": "commit_latent"} | _commit(61, 8, 48, 9, 0, 64, "bf16", mix=8),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    case = _draw(rng)
    while work(case)["flops"] > 1.3e11 or work(case)["bytes"] > 6e8:
        for k in ("ctx_lo", "ctx_hi"):
            case[k] = max(1, case[k] * 3 // 4)
        for k in ("budget", "sink", "recent"):
            if k in case:
                case[k] = case[k] * 3 // 4
    return case


def _draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "weights", "weights", "evict", "evict", "commit"])
    hq, hkv = rng.choice([(32, 8), (32, 8), (32, 4), (16, 4), (8, 2), (8, 1), (16, 2), (4, 4)])
    page = rng.choice([16, 16, 16, 32, 64, 24])
    mix = rng.randrange(1, 1 << 20)
    if kind == "tree":
        seqs = _log_int(rng, 1, 64)
        n_hi = _log_int(rng, 2, 64)
        hi = min(_log_int(rng, 16, 60000), 500000 // seqs)
        return _tree(seqs, rng.choice([1, n_hi, n_hi]), n_hi, max(1, hi // rng.choice([1, 4, 32])), hi, hq, hkv, page,
                     rng.choice(["bf16", "fp8", "f16"]), mix, rng.random() < 0.5)
    if kind == "weights":
        if rng.random() < 0.3:  # a prompt over itself
            n = _log_int(rng, 50, 2000)
            return _weights(1, n, n, 0, 0, hq, hkv, page, rng.choice(["bf16", "fp8"]), mix, 0.0)
        seqs = _log_int(rng, 1, 64)
        n_hi = rng.choice([1, 1, _log_int(rng, 2, 64)])
        hi = min(_log_int(rng, 100, 60000), 1000000 // seqs)
        return _weights(seqs, rng.choice([1, n_hi, n_hi]), n_hi, max(1, hi // rng.choice([1, 4, 32])), hi, hq, hkv, page,
                        rng.choice(["bf16", "fp8", "f32"]), mix, rng.choice([1.0, 1.0, 0.0, 0.75]))
    if kind == "evict":
        layers, seqs, heads = _log_int(rng, 1, 32), _log_int(rng, 1, 16), rng.choice([1, 2, 4, 8])
        hi = min(_log_int(rng, 200, 131072), 900000 * 8 // (layers * seqs * heads))
        budget = max(8, int(hi * rng.uniform(0.05, 0.95)))
        sink = rng.choice([0, 4, budget // 10])
        return _evict(layers, seqs, max(8, hi // rng.choice([1, 2, 8])), hi, budget, sink,
                      rng.choice([0, budget // 4, budget - sink]), heads, rng.random() < 0.4, page,
                      rng.choice(["fp8", "fp8", "bf16"]), mix)
    n = _log_int(rng, 2, 64)
    return _commit(_log_int(rng, 1, 61), _log_int(rng, 1, 32), n, rng.randint(1, min(n, 12)), rng.choice([0, 1, 4, 8]),
                   page, rng.choice(["fp8", "bf16"]), mix)


# --------------------------------------------------------------------------- #
# shapes that follow from a case alone
# --------------------------------------------------------------------------- #


def _contexts(case):
    r = random.Random(case["mix"])
    lo, hi = case["ctx_lo"], case["ctx_hi"]
    if hi <= lo:
        return [hi] * case["seqs"]
    a = math.log(max(lo, 1))
    return [int(math.exp(r.uniform(a, math.log(hi)))) for _ in range(case["seqs"])]


def _counts(case):
    """(query tokens, cached tokens with them) of each sequence."""
    r = random.Random(case["mix"] + 1)
    n = [r.randint(case["n_lo"], case["n_hi"]) for _ in range(case["seqs"])]
    return n, [c + k for c, k in zip(_contexts(case), n)]


def _parents(case, n):
    """A drafted tree for each sequence: the parent of each token (-1: the context)."""
    r = random.Random(case["mix"] + 2)
    return [[r.randrange(-1, i) if r.random() < 0.4 else i - 1 for i in range(k)] for k in n]


def _ancestors(parents):
    seen = []
    for i, p in enumerate(parents):
        seen.append((seen[p] if p >= 0 else 0) | (1 << i))
    return seen


def _paths(case):
    """(accepted length, path of drafted indices) of each sequence, parents before children."""
    r = random.Random(case["mix"] + 3)
    got = []
    for _ in range(case["seqs"]):
        k = r.randint(0, case["depth"])
        got.append((k, sorted(r.sample(range(case["n"]), k)) + [0] * (case["depth"] - k)))
    return got


def _starts(case):
    r = random.Random(case["mix"] + 4)
    return [r.randrange(20, 400) for _ in range(case["seqs"])]


# --------------------------------------------------------------------------- #
# prepare
# --------------------------------------------------------------------------- #


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


def _cache(g, shape, dtype):
    """Values ~N(0, 1) in the cache's type."""
    cache = torch.empty(shape, dtype=dtype, device=DEV)
    flat = cache.view(-1)
    step = 1 << 26
    for i in range(0, flat.numel(), step):
        n = min(step, flat.numel() - i)
        flat[i:i + n] = torch.randn(n, generator=g, device=DEV).to(dtype)
    return cache


def _tables(g, lens, page, first=1):
    """A random page table over the lengths, of pages from ``first`` on, and the page after them."""
    need = [-(-n // page) for n in lens]
    pages = sum(need)
    perm = (torch.randperm(pages, generator=g, device=DEV) + first).to(torch.int32)
    table = torch.zeros(len(lens), max(need + [1]), dtype=torch.int32, device=DEV)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = perm[at:at + k]
        at += k
    return table, first + pages


_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "fp8": torch.float8_e4m3fn}


def _prepare_queries(case, seed):
    g = _gen(seed)
    n, lens = _counts(case)
    hq, hkv, page = case["hq"], case["hkv"], case["page"]
    table, pages = _tables(g, lens, page)
    cache = _cache(g, (pages, 2, page, hkv, D), torch.float8_e4m3fn)
    # logits of standard deviation 2 after the descale of the keys
    q = (torch.randn(sum(n), hq, D, generator=g, device=DEV) * 40.0).to(_TYPES[case["q"]])
    s = {"kind": case["kind"], "q": q, "k": cache[:, 0], "v": cache[:, 1], "max_q": max(n), "table": table,
         "cu": _i32(_cumulative(n)), "lens": _i32(lens), "scale": D ** -0.5,
         "kd": torch.tensor([0.0500488], device=DEV), "vd": torch.tensor([0.0437012], device=DEV)}
    return g, s, n, lens


def _prepare_tree(case, seed):
    g, s, n, lens = _prepare_queries(case, seed)
    bits = [a for p in _parents(case, n) for a in _ancestors(p)]
    s["mask"] = torch.tensor([b - (1 << 64) if b >> 63 else b for b in bits], dtype=torch.int64, device=DEV).view(-1, 1)
    s["lse"] = case["lse"]
    s["max_k"] = max(lens)
    return s


def _prepare_weights(case, seed):
    g, s, n, lens = _prepare_queries(case, seed)
    hq, hkv = case["hq"], case["hkv"]
    # what the attention of this step returned
    s["lse"] = torch.empty(hq, sum(n), dtype=torch.float32, device=DEV)
    at = 0
    for b, (k, L) in enumerate(zip(n, lens)):
        pos = torch.arange(L, device=DEV)
        slot = s["table"][b, pos // case["page"]].long(), pos % case["page"]
        keys = s["k"].view(torch.uint8)[slot].view(torch.float8_e4m3fn).float().permute(1, 2, 0)  # [Hkv, D, L]
        qs = s["q"][at:at + k].float().clamp(-448, 448).to(torch.float8_e4m3fn).float()
        qs = qs.view(k, hkv, hq // hkv, D).permute(1, 2, 0, 3).reshape(hkv, -1, D)
        x = torch.bmm(qs, keys.contiguous()) * (s["scale"] * s["kd"])
        see = pos[None] <= L - k + torch.arange(k, device=DEV)[:, None]
        x = x.view(hkv, hq // hkv, k, L).masked_fill(~see, float("-inf"))
        s["lse"][:, at:at + k] = torch.logsumexp(x, -1).reshape(hq, k)
        at += k
        del x, keys
    s["max_k"] = max(lens)
    # earlier sums of the size of this step's, so that neither hides the other
    s["scores"] = torch.rand(len(n), hkv, s["table"].shape[1] * case["page"], generator=g, device=DEV) * 0.01
    s["decay"] = case["decay"]
    return s


def _prepare_evict(case, seed):
    g = _gen(seed)
    lens = _contexts(case)
    page, heads, layers, budget = case["page"], case["heads"], case["layers"], case["budget"]
    table, first = _tables(g, lens, page)
    dst, end = _tables(g, [min(n, budget) for n in lens], page, first)
    cache = _cache(g, (layers, end, 2, page, heads, D), _TYPES[case["cache"]])
    # running sums of weights: a heavy tail, and tokens that never received any
    shape = (layers, len(lens), 1 if case["shared"] else heads, max(lens))
    scores = torch.rand(shape, generator=g, device=DEV) ** 6 * 8.0
    scores = torch.where(torch.rand(shape, generator=g, device=DEV) < 0.05, torch.zeros_like(scores), scores)
    return {"kind": "evict", "k": cache[:, :, 0], "v": cache[:, :, 1], "fresh": cache[:, first:], "scores": scores,
            "table": table, "lens": _i32(lens), "dst": dst, "budget": budget, "sink": case["sink"],
            "recent": case["recent"], "scores_out": torch.zeros_like(scores)}


def _prepare_commit(case, seed):
    g = _gen(seed)
    starts = _starts(case)
    table, pages = _tables(g, [s + case["n"] for s in starts], case["page"])
    head = (case["layers"], pages)
    if case["heads"]:
        cache = _cache(g, head + (2, case["page"], case["heads"], D), _TYPES[case["cache"]])
        caches = [cache[:, :, 0], cache[:, :, 1]]
    else:
        cache = _cache(g, head + (case["page"], LATENT), _TYPES[case["cache"]])
        caches = [cache]
    paths = _paths(case)
    return {"kind": "commit", "caches": caches, "cache": cache, "table": table, "starts": _i32(starts),
            "path": _i32([p for _, p in paths]), "path_lens": _i32([k for k, _ in paths])}


def prepare(case, seed):
    return {"tree": _prepare_tree, "weights": _prepare_weights, "evict": _prepare_evict,
            "commit": _prepare_commit}[case["kind"]](case, seed)


# --------------------------------------------------------------------------- #
# run
# --------------------------------------------------------------------------- #


def run(s):
    kind = s["kind"]
    if own:
        from pipeswift_amd import attention, cache_ops
        if kind == "tree":
            return attention.paged_tree_attention(
                s["q"], s["k"], s["v"], s["table"], s["lens"], s["mask"], s["cu"], s["max_q"],
                softmax_scale=s["scale"], k_descale=s["kd"], v_descale=s["vd"], return_softmax_lse=s["lse"],
                max_seq_len=s["max_k"])
        if kind == "weights":
            return attention.accumulate_attention_weights(
                s["scores"], s["q"], s["k"], s["lse"], s["table"], s["lens"], s["cu"], s["max_q"],
                softmax_scale=s["scale"], k_descale=s["kd"], decay=s["decay"], max_seq_len=s["max_k"])
        if kind == "evict":
            kept, lens = cache_ops.evict_tokens(
                [s["k"], s["v"]], s["scores"], s["table"], s["lens"], s["dst"], s["budget"], sink=s["sink"],
                recent=s["recent"], scores_out=s["scores_out"])
            return {"kept": kept, "lens": lens, "scores": s["scores_out"], "pages": s["fresh"]}
        cache_ops.commit_draft_tokens(s["caches"], s["table"], s["starts"], s["path"], s["path_lens"])
        return s["cache"]
    if kind == "tree":
        return _plain_tree(s)
    if kind == "weights":
        return _plain_weights(s)
    if kind == "evict":
        return _plain_evict(s)
    return _plain_commit(s)


def _slots(table, page, positions):
    """(page, row) of positions [B, n] of each sequence."""
    return torch.gather(table.long(), 1, positions // page), positions % page


def _as_bytes(cache):
    return cache.view(torch.uint8) if cache.dtype == torch.float8_e4m3fn else cache


def _padded_keys(s, name):
    """[B, Hkv, Lmax, D] float32 of a cache."""
    cache = s[name]
    pos = torch.arange(s["max_k"], device=DEV).expand(s["table"].shape[0], -1)
    rows = _as_bytes(cache)[_slots(s["table"], cache.shape[1], pos)].view(cache.dtype)
    return rows.permute(0, 2, 1, 3).float()


def _padded_queries(s):
    """[B, Hkv, n G, D] float32 of the quantized query, and the row of each padded (sequence, token)."""
    first, n = s["cu"][:-1].long(), (s["cu"][1:] - s["cu"][:-1]).long()
    at = first[:, None] + torch.minimum(torch.arange(s["max_q"], device=DEV), (n - 1).clamp(min=0)[:, None])
    q = s["q"].float().clamp(-448, 448).to(torch.float8_e4m3fn).float()
    hq, hkv = q.shape[1], s["k"].shape[2]
    q = q[at].view(at.shape[0], -1, hkv, hq // hkv, D).permute(0, 2, 1, 3, 4)
    return q.reshape(at.shape[0], hkv, -1, D), n, at


def _plain_scores(s):
    q, n, at = _padded_queries(s)
    b, hkv, _, _ = q.shape
    keys = _padded_keys(s, "k").reshape(b * hkv, -1, D)
    x = torch.bmm(q.reshape(b * hkv, -1, D), keys.transpose(1, 2)) * (s["scale"] * s["kd"])
    return x.view(b, hkv, s["max_q"], -1, x.shape[-1]), n, at  # [B, Hkv, n, G, L]


def _plain_tree(s):
    x, n, at = _plain_scores(s)
    pos = torch.arange(x.shape[-1], device=DEV)
    drafted = pos[None] - (s["lens"].long() - n)[:, None]  # [B, L]: the drafted index of a key, negative before it
    mask = s["mask"][:, 0][at]  # [B, n]
    bit = (mask[:, :, None] >> drafted.clamp(0, 63)[:, None]) & 1
    see = (drafted[:, None] < 0) | ((bit == 1) & (drafted < n[:, None])[:, None])
    x.masked_fill_(~see[:, None, :, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    b, hkv = x.shape[:2]
    v = _padded_keys(s, "v").reshape(b * hkv, -1, D)
    o = torch.bmm(p.view(b * hkv, -1, p.shape[-1]), v).view(b, hkv, s["max_q"], -1, D) / total * s["vd"]
    live = torch.arange(s["max_q"], device=DEV) < n[:, None]
    out = torch.empty(s["q"].shape, dtype=torch.bfloat16, device=DEV)
    rows = o.permute(0, 2, 1, 3, 4).reshape(b, s["max_q"], -1, D)
    out[at[live]] = rows[live].to(out.dtype)
    if not s["lse"]:
        return out
    lse = torch.empty(s["q"].shape[1], s["q"].shape[0], device=DEV)
    lse.t()[at[live]] = (top + torch.log(total))[..., 0].permute(0, 2, 1, 3).reshape(b, s["max_q"], -1)[live]
    return out, lse


def _plain_weights(s):
    x, n, at = _plain_scores(s)
    b, hkv, m, g, L = x.shape
    lse = s["lse"].view(hkv, g, -1)[:, :, at].permute(2, 0, 3, 1)  # [B, Hkv, n, G]
    pos = torch.arange(L, device=DEV)
    i = torch.arange(m, device=DEV)
    see = pos[None, None] <= ((s["lens"].long() - n)[:, None] + i)[:, :, None]
    see &= (i < n[:, None])[:, :, None] & (pos < s["lens"][:, None])[:, None]
    w = torch.where(see[:, None, :, None], torch.exp(x - lse[..., None]), torch.zeros((), device=DEV)).sum((2, 3))
    old = s["scores"][:, :, :L]
    new = w if s["decay"] == 0.0 else old * s["decay"] + w
    old.copy_(torch.where((pos < s["lens"][:, None])[:, None], new, old))
    return s["scores"]


def _plain_evict(s):
    scores, budget, lens = s["scores"], s["budget"], s["lens"].long()
    L = scores.shape[-1]
    pos = torch.arange(L, device=DEV)
    count = lens.clamp(max=budget)
    end = (lens - s["recent"])[:, None]
    key = torch.where(((pos < s["sink"]) | (pos >= end))[:, None], float("inf"), scores)
    key = torch.where((pos < lens[:, None])[:, None], key, float("-inf"))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :budget]
    i = torch.arange(order.shape[-1], device=DEV)
    live = (i < count[:, None])[:, None]
    kept = torch.where(live, order, L).sort(-1).values
    live = live.expand(kept.shape)
    picked = torch.where(live, scores.gather(-1, kept.clamp(max=L - 1)), torch.zeros((), device=DEV))
    out = torch.where((pos < lens[:, None])[:, None], torch.zeros((), device=DEV), s["scores_out"])
    out[..., :picked.shape[-1]] = torch.where(live, picked, out[..., :picked.shape[-1]])
    s["scores_out"].copy_(out)
    # the kept rows, for every kv head; places past a sequence's count repeat its first
    heads, page = s["k"].shape[3], s["k"].shape[2]
    src = torch.where(live, kept, kept[..., :1]).expand(-1, -1, heads, -1)
    dst = torch.where(live, i, torch.zeros_like(i)).expand(-1, -1, heads, -1)
    layer = torch.arange(src.shape[0], device=DEV)[:, None, None, None]
    seq = torch.arange(src.shape[1], device=DEV)[None, :, None, None]
    head = torch.arange(heads, device=DEV)[None, None, :, None]
    for cache in (_as_bytes(s["k"]), _as_bytes(s["v"])):
        rows = cache[layer, s["table"].long()[seq, src // page], src % page, head]
        cache[layer, s["dst"].long()[seq, dst // page], dst % page, head] = rows
    full = torch.full(kept.shape[:-1] + (budget,), -1, dtype=torch.int32, device=DEV)
    full[..., :kept.shape[-1]] = torch.where(live, kept, -1).to(torch.int32)
    return {"kept": full, "lens": count.to(torch.int32), "scores": s["scores_out"], "pages": s["fresh"]}


def _plain_commit(s):
    n = s["path_lens"].long()[:, None]
    i = torch.arange(s["path"].shape[1], device=DEV).expand(s["path"].shape)
    path = torch.where(n > 0, s["path"].long(), 0)
    src = s["starts"].long()[:, None] + torch.where(i < n, path, path[:, :1])
    dst = s["starts"].long()[:, None] + torch.where(i < n, i, 0)
    for cache in s["caches"]:
        cache, page = _as_bytes(cache), cache.shape[2]
        (a, x), (b, y) = _slots(s["table"], page, src), _slots(s["table"], page, dst)
        cache[:, b, y] = cache[:, a, x]
    return s["cache"]


# --------------------------------------------------------------------------- #
# work
# --------------------------------------------------------------------------- #


def work(case):
    kind = case["kind"]
    if kind in ("tree", "weights"):
        n, lens = _counts(case)
        hq, hkv = case["hq"], case["hkv"]
        rows = sum(n) * hq
        esz = {"fp8": 1, "f32": 4}.get(case["q"], 2)
        pages = sum(-(-k // case["page"]) for k in lens)
        if kind == "tree":
            pairs = sum(k * (L - k) for k, L in zip(n, lens))
            pairs += sum(bin(a).count("1") for p in _parents(case, n) for a in _ancestors(p))
            return {"bytes": sum(lens) * hkv * D * 2 + rows * D * (esz + 2) + 8 * sum(n) + 4 * pages
                    + (4 * rows if case["lse"] else 0), "flops": 4 * D * hq * pairs}
        pairs = sum(k * (L - k) + k * (k + 1) // 2 for k, L in zip(n, lens))
        return {"bytes": sum(lens) * hkv * (D + (4 if case["decay"] == 0.0 else 8)) + rows * (D * esz + 4) + 4 * pages,
                "flops": 2 * D * hq * pairs}
    if kind == "evict":
        lens = _contexts(case)
        each = case["layers"] * (1 if case["shared"] else case["heads"])
        kept = sum(min(n, case["budget"]) for n in lens)
        row = 2 * D * (1 if case["cache"] == "fp8" else 2)
        # the scores read and written over the old length, the kept positions, and every kept row moved
        return {"bytes": each * (8 * sum(lens) + 4 * len(lens) * case["budget"])
                + 2 * case["layers"] * case["heads"] * row * kept, "flops": 0}
    row = (2 * D * case["heads"] or LATENT) * (1 if case["cache"] == "fp8" else 2)
    moved = sum(1 for k, p in _paths(case) for i in range(k) if p[i] != i)
    return {"bytes": 2 * case["layers"] * row * moved + 4 * case["seqs"] * (case["depth"] + 2), "flops": 0}


# --------------------------------------------------------------------------- #
# exact: from the definitions, in 64 bits, sequence by sequence
# --------------------------------------------------------------------------- #


def _e4m3(x):
    """The nearest e4m3 value of float64 x, ties to even, saturating."""
    a = x.abs().clamp(max=448.0)
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
    return torch.sign(x) * (torch.round(a / step) * step).clamp(max=448.0)


def _values(cache, table_row, count, head):
    """float64 [count, D] of one head of a sequence's first rows."""
    page = cache.shape[1]
    pos = torch.arange(count, device=DEV)
    raw = cache.view(torch.uint8)[table_row[pos // page].long(), pos % page, head]
    return raw.view(torch.float8_e4m3fn).double()


def _exact_tree(case, s):
    n, lens = _counts(case)
    hq, hkv = case["hq"], case["hkv"]
    group = hq // hkv
    out = torch.empty(sum(n), hq, D, dtype=torch.float64, device=DEV)
    lse = torch.empty(hq, sum(n), dtype=torch.float64, device=DEV)
    q = _e4m3(s["q"].double())
    at = 0
    for b, (k, L, parents) in enumerate(zip(n, lens, _parents(case, n))):
        see = torch.zeros(k, L, dtype=torch.bool)
        see[:, :L - k] = True
        for i in range(k):
            j = i
            while j >= 0:
                see[i, L - k + j] = True
                j = parents[j]
        see = see.to(DEV)
        for h in range(hkv):
            keys, vals = _values(s["k"], s["table"][b], L, h), _values(s["v"], s["table"][b], L, h)
            for g in range(group):
                x = q[at:at + k, h * group + g] @ keys.t() * (s["scale"] * s["kd"].double())
                x = x.masked_fill(~see, float("-inf"))
                norm = torch.logsumexp(x, 1)
                out[at:at + k, h * group + g] = torch.exp(x - norm[:, None]) @ vals * s["vd"].double()
                lse[h * group + g, at:at + k] = norm
        at += k
    return (out, lse) if case["lse"] else out


def _exact_weights(case, s):
    n, lens = _counts(case)
    hq, hkv = case["hq"], case["hkv"]
    group = hq // hkv
    q = _e4m3(s["q"].double())
    total = s["scores"].double()
    at = 0
    for b, (k, L) in enumerate(zip(n, lens)):
        last = L - k + torch.arange(k, device=DEV)
        hidden = torch.arange(L, device=DEV)[None] > last[:, None]
        for h in range(hkv):
            keys = _values(s["k"], s["table"][b], L, h)
            got = torch.zeros(L, dtype=torch.float64, device=DEV)
            for hh in range(h * group, h * group + group):
                x = q[at:at + k, hh] @ keys.t() * (s["scale"] * s["kd"].double())
                got += torch.exp(x - s["lse"][hh, at:at + k].double()[:, None]).masked_fill(hidden, 0.0).sum(0)
            total[b, h, :L] = total[b, h, :L] * case["decay"] + got
        at += k
    return total


def exact(case, seed):
    if case["kind"] == "tree":
        return _exact_tree(case, prepare(case, seed))
    if case["kind"] == "weights":
        return _exact_weights(case, prepare(case, seed))
    # the others copy: the plain form's values are the definition's
    return None
