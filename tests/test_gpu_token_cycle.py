"""The operators together, as a serving step uses them: a prompt's attention, the
weights of its last queries, an eviction to a budget in fresh pages, a drafted
tree appended and attended to, its accepted path committed, and a decode step on
what is left -- against the float64 oracle on the tokens that remain."""

import numpy as np
import pytest
import torch

from oracle import kv_oracle as O
from oracle import token_oracle as T
from pipeswift_amd import attention, cache_ops, reshape_and_cache

pytestmark = pytest.mark.gpu

HQ, HKV, PS, LAYERS = 16, 4, 16, 2


def test_prompt_evict_tree_commit_decode(dev):
    g = torch.Generator().manual_seed(5)
    lens, budget, sink, recent, window = [213, 150, 96], 96, 4, 32, 16
    drafts, B = [7, 1, 12], 3
    P = 120
    perm = torch.randperm(P - 1, generator=g).to(torch.int32) + 1
    W = 15
    bt = perm[:B * W].view(B, W).to(dev)
    fresh = perm[B * W:B * W + B * 8].view(B, 8).to(dev)
    cache = torch.zeros(LAYERS, P, 2, PS, HKV, 128, dtype=torch.float8_e4m3fn, device=dev)
    kv = [cache[:, :, 0], cache[:, :, 1]]
    lens_d = torch.tensor(lens, dtype=torch.int32, device=dev)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=dev)

    def slots(table, first, count):
        rows = []
        for b in range(B):
            p = torch.arange(first[b], first[b] + count[b], device=dev)
            rows.append(table[b, p // PS].long() * PS + p % PS)
        return torch.cat(rows)

    def randn(n, h):
        return (torch.randn(n, h, 128, generator=g) * 2).to(torch.bfloat16).to(dev)

    scores = torch.zeros(LAYERS, B, HKV, 256, device=dev)
    scale = 128 ** -0.5
    for layer in range(LAYERS):
        reshape_and_cache.reshape_and_cache_flash(randn(sum(lens), HKV), randn(sum(lens), HKV), kv[0][layer],
                                                  kv[1][layer], slots(bt, [0] * B, lens))
        q = randn(sum(lens), HQ)
        _, lse = attention.flash_attn_varlen_func(q, kv[0][layer], kv[1][layer], max(lens), cu, None, lens_d, bt,
                                                  softmax_scale=scale, causal=True, return_softmax_lse=True)
        # the last queries of each prompt, gathered
        last = torch.cat([torch.arange(int(cu[b + 1]) - window, int(cu[b + 1]), device=dev) for b in range(B)])
        attention.accumulate_attention_weights(scores[layer], q[last], kv[0][layer], lse[:, last], bt, lens_d,
                                               torch.arange(B + 1, dtype=torch.int32, device=dev) * window, window)
    # every query of every head gives its weights away exactly once
    total = scores.sum(-1).cpu()
    assert torch.allclose(total, torch.full_like(total, window * HQ / HKV), rtol=2e-3)

    before = cache.clone()
    old = scores.cpu().numpy()
    kept, kept_lens = cache_ops.evict_tokens(kv, scores, bt, lens_d, fresh, budget, sink, recent)
    want, _ = T.select_tokens(old, lens, budget, sink, recent)
    assert np.array_equal(kept.cpu().numpy(), want) and kept_lens.tolist() == [96, 96, 96]
    raw = cache.view(torch.uint8).cpu()
    for b in range(B):  # the old pages are as they were, the new ones hold the kept rows
        pages = bt[b].long().cpu()
        assert torch.equal(raw[:, pages], before.view(torch.uint8).cpu()[:, pages])

    # a drafted tree per sequence, appended behind the kept tokens
    parents = [[-1, 0, 0, 1, 1, 2, -1], [-1], [-1, 0, 1, 2, 0, 4, 5, -1, 7, 7, 9, 10]]
    now = [int(x) + n for x, n in zip(kept_lens, drafts)]
    now_d = torch.tensor(now, dtype=torch.int32, device=dev)
    cut = torch.tensor(np.concatenate([[0], np.cumsum(drafts)]), dtype=torch.int32, device=dev)
    mask = attention.tree_mask(torch.tensor(sum(parents, []), dtype=torch.int32, device=dev), cut, max(drafts))
    where = slots(fresh, kept_lens.tolist(), drafts)
    for layer in range(LAYERS):
        reshape_and_cache.reshape_and_cache_flash(randn(sum(drafts), HKV), randn(sum(drafts), HKV), kv[0][layer],
                                                  kv[1][layer], where)
        q = randn(sum(drafts), HQ)
        got, lse = attention.paged_tree_attention(q, kv[0][layer], kv[1][layer], fresh, now_d, mask, cut, max(drafts),
                                                  softmax_scale=scale, return_softmax_lse=True,
                                                  out=torch.empty(sum(drafts), HQ, 128, device=dev))
        host = cache[layer].view(torch.uint8).cpu().numpy()
        exp, exp_lse, _ = T.tree_attention(q.cpu().view(torch.int16).numpy().view(np.uint16), "bf16", host[:, 0],
                                           host[:, 1], fresh.cpu().numpy(), now, mask.cpu().numpy(), cut.tolist(), scale)
        # the bound of tests/test_gpu_attention_prefill.py, with vmax <= 10
        assert np.abs(got.double().cpu().numpy() - exp).max() <= 10 * (3e-4 + 2.0 ** -11 + 128 * 2.0 ** -25) + 1e-3
        assert np.abs(lse.double().cpu().numpy().T - exp_lse).max() <= 1e-3

    # accepted: 0 -> 2 -> 5, nothing of sequence 1, 7 -> 9 -> 10 -> 11
    path = torch.tensor([[0, 2, 5, 0], [0, 0, 0, 0], [7, 9, 10, 11]], dtype=torch.int32, device=dev)
    taken = torch.tensor([3, 0, 4], dtype=torch.int32, device=dev)
    host = cache.view(torch.uint8).cpu().numpy().copy()
    for k in range(2):
        T.commit_draft_tokens(host[:, :, k], fresh.cpu().numpy(), kept_lens.tolist(), path.cpu().numpy(), taken.tolist())
    cache_ops.commit_draft_tokens(kv, fresh, kept_lens, path, taken)
    assert np.array_equal(cache.view(torch.uint8).cpu().numpy(), host)

    # the next token of each sequence
    lens2 = (kept_lens + taken + 1).to(torch.int32)
    for layer in range(LAYERS):
        reshape_and_cache.reshape_and_cache_flash(randn(B, HKV), randn(B, HKV), kv[0][layer], kv[1][layer],
                                                  slots(fresh, (kept_lens + taken).tolist(), [1] * B))
        q = randn(B, HQ)
        got, lse = attention.paged_decode_attention(q, kv[0][layer], kv[1][layer], fresh, lens2, scale,
                                                    return_softmax_lse=True,
                                                    out=torch.empty(B, HQ, 128, device=dev))
        host = cache[layer].view(torch.uint8).cpu().numpy()
        exp, exp_lse = O.paged_decode_attention(q.cpu().view(torch.int16).numpy().view(np.uint16), "bf16", host[:, 0],
                                                host[:, 1], fresh.cpu().numpy(), lens2.cpu().numpy(), scale)
        assert np.abs(got.double().cpu().numpy() - exp).max() <= 10 * 3e-4 + 1e-3
        was = scores[layer].clone()
        attention.accumulate_attention_weights(scores[layer], q, kv[0][layer], lse, fresh, lens2)
        gain = (scores[layer] - was).sum(-1).cpu()
        assert torch.allclose(gain, torch.full_like(gain, HQ / HKV), rtol=2e-3)
