"""Pins of oracle/token_oracle.py: torch's masked softmax, the causal oracle, and
literal tiny cases."""

import numpy as np
import torch

from oracle import kv_oracle as O
from oracle import token_oracle as T
from pipeswift_amd.attention import tree_mask


def _case(seed, n=5, L=37, Hq=4, Hkv=2, ps=8):
    g = torch.Generator().manual_seed(seed)
    P = 9
    k = (torch.randn(P, ps, Hkv, 128, generator=g)).to(torch.float8_e4m3fn)
    v = (torch.randn(P, ps, Hkv, 128, generator=g)).to(torch.float8_e4m3fn)
    q = (torch.randn(n, Hq, 128, generator=g)).to(torch.float8_e4m3fn)
    bt = torch.randperm(P, generator=g)[:5].to(torch.int32)[None]
    return q, k, v, bt, g


def _bits(t):
    return t.view(torch.uint8).numpy()


def test_tree_attention_is_a_masked_softmax():
    n, L = 5, 37
    q, k, v, bt, g = _case(1)
    parents = torch.tensor([-1, 0, 0, 1, -1])
    mask = tree_mask(parents, torch.tensor([0, n]), n)
    assert mask[:, 0].tolist() == [0b1, 0b11, 0b101, 0b1011, 0b10000]
    out, lse, bound = T.tree_attention(_bits(q), "fp8", _bits(k), _bits(v), bt.numpy(), [L], mask.numpy(), [0, n], 0.1)
    slot = bt[0].long().repeat_interleave(8)[:L] * 8 + torch.arange(L) % 8
    K = k.double().view(-1, 2, 128)[slot].repeat_interleave(2, 1)
    V = v.double().view(-1, 2, 128)[slot].repeat_interleave(2, 1)
    x = torch.einsum("ihd,jhd->hij", q.double(), K) * float(np.float32(0.1))
    see = torch.ones(n, L, dtype=torch.bool)
    see[:, L - n:] = (mask >> torch.arange(n)) & 1 == 1
    x = x.masked_fill(~see, float("-inf"))
    want = torch.einsum("hij,jhd->ihd", x.softmax(-1), V)
    assert np.allclose(out, want.numpy(), rtol=1e-12, atol=1e-12)
    assert np.allclose(lse, x.logsumexp(-1).t().numpy(), rtol=1e-12)
    assert bound >= x[torch.isfinite(x)].abs().max()


def test_a_chain_is_the_causal_oracle():
    n, L = 5, 37
    q, k, v, bt, _ = _case(2)
    mask = tree_mask(torch.arange(n) - 1, torch.tensor([0, n]), n)
    out, lse, _ = T.tree_attention(_bits(q), "fp8", _bits(k), _bits(v), bt.numpy(), [L], mask.numpy(), [0, n], 0.1)
    want, lse_want = O.paged_decode_attention(_bits(q), "fp8", _bits(k), _bits(v), bt.numpy(), np.array([L]), 0.1,
                                              cu_seqlens_q=np.array([0, n]), causal=True)
    assert np.allclose(out, want, rtol=1e-12, atol=1e-12) and np.allclose(lse, lse_want, rtol=1e-12)


def test_masks_of_parents_with_several_sequences_and_words():
    rng = np.random.default_rng(3)
    counts = [1, 0, 70, 3, 129]
    cu = np.concatenate([[0], np.cumsum(counts)])
    parents, want = [], []
    for n in counts:
        own = [int(rng.integers(-1, i)) if i else -1 for i in range(n)]
        seen = []
        for i, p in enumerate(own):
            seen.append((seen[p] if p >= 0 else 0) | 1 << i)
        parents += own
        want += seen
    got = tree_mask(torch.tensor(parents, dtype=torch.int32), torch.tensor(cu, dtype=torch.int32), 129)
    assert got.shape == (sum(counts), 3) and got.is_contiguous()
    for i, w in enumerate(want):
        assert [int(x) & (2 ** 64 - 1) for x in got[i]] == [(w >> 64 * k) & (2 ** 64 - 1) for k in range(3)]
    assert tree_mask(torch.empty(0, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 4).shape == (0, 1)


def test_weights_of_one_query_sum_to_one_and_add_up():
    n, L = 3, 30
    q, k, v, bt, _ = _case(4, n=n)
    _, lse = O.paged_decode_attention(_bits(q), "fp8", _bits(k), _bits(v), bt.numpy(), np.array([L]), 0.1,
                                      cu_seqlens_q=np.array([0, n]), causal=True)
    old = np.zeros((1, 2, 40))
    got, _, _ = T.attention_weights(old, _bits(q), "fp8", _bits(k), lse.T, bt.numpy(), [L], [0, n], 0.1)
    assert np.allclose(got.sum(-1), n * 2)  # three tokens of two heads each
    assert (got[..., L:] == 0).all()
    again, _, _ = T.attention_weights(got, _bits(q), "fp8", _bits(k), lse.T, bt.numpy(), [L], [0, n], 0.1, decay=0.5)
    assert np.allclose(again, 1.5 * got)


def test_selection_by_hand():
    s = np.array([[[[5., 1., np.nan, 3., 3., -0.0, 0.0, 9., 2., 3.]]]], dtype=np.float32)
    kept, lens = T.select_tokens(s, [10], 5, 1, 1)
    assert kept.tolist() == [[[[0, 3, 4, 7, 9]]]] and lens.tolist() == [5]
    kept, _ = T.select_tokens(s, [9], 7, 0, 0)  # -0 and 0 tie: the lower position
    assert kept.tolist() == [[[[0, 1, 3, 4, 5, 7, 8]]]]
    kept, lens = T.select_tokens(s, [4], 5, 1, 1)
    assert kept.tolist() == [[[[0, 1, 2, 3, -1]]]] and lens.tolist() == [4]
    kept, _ = T.select_tokens(np.full((1, 1, 1, 4), -np.inf, np.float32), [4], 2, 0, 0)
    assert kept.tolist() == [[[[0, 1]]]]
    kept, _ = T.select_tokens(np.array([[[[np.nan, -np.inf, np.nan, 1.]]]], np.float32), [4], 3, 0, 0)
    assert kept.tolist() == [[[[0, 1, 3]]]]


def test_moves_by_hand():
    cache = np.arange(1 * 4 * 2 * 1 * 1).reshape(1, 4, 2, 1, 1)
    bt = np.array([[2, 0]])
    scores = np.array([[[[1., 4., 2., 3.]]]], dtype=np.float32)
    kept, lens, out = T.evict_tokens([cache], scores, bt, [4], np.array([[1, 9]]), 2, 0, 0)
    assert kept.tolist() == [[[[1, 3]]]] and out.tolist() == [[[[4., 3., 0., 0.]]]]
    assert cache[0, :, :, 0, 0].tolist() == [[0, 1], [5, 1], [4, 5], [6, 7]]
    rows = np.arange(8).reshape(1, 4, 2)
    T.commit_draft_tokens(rows, np.array([[3, 1, 0]]), [1], np.array([[2, 0, 3]]), [3])
    # positions 1..4 hold rows 7, 2, 3, 0: position 1 <- 3, 2 <- 1, 3 <- 4
    assert rows[0].tolist() == [[0, 1], [7, 0], [4, 5], [6, 3]]


def test_a_parent_outside_its_sequence_is_none():
    """An index at or past a sequence's tokens names no token of the next one."""
    cu = torch.tensor([0, 3, 3, 5, 7], dtype=torch.int32)
    parents = [-1, 0, 3, 2, 0, 9, -7]
    want = [0b001, 0b011, 0b100, 0b01, 0b11, 0b01, 0b10]
    for dtype in (torch.int32, torch.int64):
        made = tree_mask(torch.tensor(parents + [0, 2], dtype=dtype), cu, 3)  # (two rows that no sequence owns)
        assert made[:7, 0].tolist() == want
