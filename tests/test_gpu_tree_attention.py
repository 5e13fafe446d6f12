"""GPU parity of ``attention.paged_tree_attention`` with the float64 oracle.

Tolerances, from cached_case's ds (with s - m at most twice the largest score):
each normalised weight is off by a factor of at most 1 +- 2 d, d = ds + 4 eps (1
+ 2 max|s|) + K eps (its own error and the sum's), and rounds once to fp16
(2^-11 of itself, 2^-25 of the row's largest below the normal range, which a
row's K weights add up to K 2^-25, since its sum is at least 1).  P V and the
merge of partial results add sums of K terms in float32, at most (K + 64) eps.
So |out - exact| <= vmax (2 d + 2^-11 + K 2^-25 + (K + 64) eps), vmax = max |V
vd|, plus 2^-8 |exact| where it is stored as bf16 (float32: 4 eps |exact|), and
|lse - exact| <= ds + (K + 64) eps + 4 eps (|lse| + max|s|).
"""

import numpy as np
import pytest
import torch

from oracle import token_oracle as T
from oracle import kv_oracle as O
from pipeswift_amd import attention
from tests.cached_case import EPS, Case, score_error

pytestmark = pytest.mark.gpu


def _trees(case, seed, words=None, arbitrary=False):
    """int64 mask [TQ, words] of random trees, or of random bits (every bit, those past n too)."""
    rng = np.random.default_rng(seed)
    words = words or -(-case.max_q // 64)
    if arbitrary:
        return torch.from_numpy(rng.integers(-2 ** 63, 2 ** 63 - 1, (case.TQ, words), dtype=np.int64))
    parents = [int(rng.integers(-1, i)) if i and rng.random() < 0.5 else i - 1 for n in case.counts for i in range(n)]
    mask = torch.zeros(case.TQ, words, dtype=torch.int64)
    made = attention.tree_mask(torch.tensor(parents, dtype=torch.int32), torch.from_numpy(case.cu), case.max_q)
    mask[:case.rows, :made.shape[1]] = made
    return mask


def _run(case, mask, dev, out_dtype=torch.float32, scale=None, **kw):
    out = torch.full((case.TQ, case.Hq, 128), 7.0, dtype=out_dtype, device=dev)
    got, lse = attention.paged_tree_attention(
        case.qd, case.k, case.v, case.btd, case.lensd, mask.to(dev), case.cud, case.max_q,
        softmax_scale=case.scale if scale is None else scale, q_descale=case.dd[0], k_descale=case.dd[1],
        v_descale=case.dd[2], out=out, return_softmax_lse=True, **kw)
    assert got is out
    return got, lse


def _check(case, mask, got, lse, scale=None, nan=False):
    q, k, v = case.host()
    scale = case.scale if scale is None else scale
    want, lse_want, bound = T.tree_attention(q, case.name, k, v, case.bt.numpy(), case.lens, mask.numpy(), case.cu, scale,
                                             *case.ds)
    K = max([1, *case.lens])
    vals = O.e4m3fn_to_f32(v)
    vmax = float(np.nanmax(np.abs(vals))) * (1.0 if case.ds[2] is None else float(case.ds[2].max(initial=0.0)))
    s_max = bound  # |s| <= sum |q~ K|
    ds = score_error(bound, s_max)
    d = ds + 4 * EPS * (1 + 2 * s_max) + K * EPS
    n = case.rows
    o = got[:n].double().cpu().numpy()
    l = lse.double().cpu().numpy().T[:n]
    if nan:
        assert np.array_equal(np.isnan(o), np.isnan(want[:n])), "NaN in other places"
    o, w = np.nan_to_num(o), np.nan_to_num(want[:n])
    tol = vmax * (2 * d + 2.0 ** -11 + K * 2.0 ** -25 + (K + 64) * EPS)
    tol = tol + np.abs(w) * (2.0 ** -8 if got.dtype == torch.bfloat16 else 4 * EPS)
    err = np.abs(o - w)
    assert (err <= tol).all(), f"max err {err.max():.3e} (tol {np.min(tol):.3e}) at {np.unravel_index(err.argmax(), err.shape)}"
    lw = lse_want[:n]
    fin = np.isfinite(lw)
    assert np.isneginf(l[np.isneginf(lw)]).all()
    if nan:
        assert np.array_equal(np.isnan(l), np.isnan(lw))
    le = np.abs(l[fin] - lw[fin])
    assert (le <= ds + (K + 64) * EPS + 4 * EPS * (np.abs(lw[fin]) + s_max)).all(), f"lse err {le.max(initial=0):.3e}"
    if case.TQ > n:
        assert bool((got[n:] == 7.0).all()), "rows that no sequence owns"


@pytest.mark.parametrize("ps", [16, 24, 64, 7])
@pytest.mark.parametrize("Hq,Hkv", [(32, 8), (8, 1), (4, 4), (6, 2), (40, 1)])
def test_ragged_trees(dev, Hq, Hkv, ps):
    """1 to 33 drafted tokens, none in one sequence, over contexts of 0 to 900
    tokens, one sequence shorter than its draft and one empty."""
    rng = np.random.default_rng(Hq + Hkv + ps)
    counts = [int(x) for x in rng.integers(1, 34, 8)]
    counts[3] = 0
    lens = [n + int(x) for n, x in zip(counts, rng.integers(0, 900, 8))]
    lens[1] = counts[1]             # no context: the first token sees itself alone
    lens[5] = max(counts[5] - 2, 0)  # its first drafted tokens are not cached
    lens[6] = 0
    case = Case(dev, 11, lens, counts, Hq, Hkv, ps, spare_rows=3, spare_table=2)
    mask = _trees(case, 5)
    _check(case, mask, *_run(case, mask, dev))


@pytest.mark.parametrize("q_dtype", [torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_types_and_strides(dev, q_dtype, out_dtype):
    case = Case(dev, 3, [300, 61, 1025], [9, 16, 5], 16, 4, 16, q_dtype=q_dtype, strided_q=True, head_major=True)
    mask = _trees(case, 6)
    _check(case, mask, *_run(case, mask, dev, out_dtype))


@pytest.mark.parametrize("n", [1, 2, 31, 63, 64, 65, 130, 200])
@pytest.mark.parametrize("Hq,Hkv", [(8, 1), (4, 2)])
def test_tree_sizes_and_words(dev, n, Hq, Hkv):
    """Across MFMA tiles, row blocks and mask words; arbitrary masks with bits past the tree."""
    case = Case(dev, n, [n + 100, n, n + 31], [n, n, max(1, n - 1)], Hq, Hkv, 16)
    mask = _trees(case, 7, words=-(-n // 64) + 1, arbitrary=True)
    _check(case, mask, *_run(case, mask, dev))


@pytest.mark.parametrize("L", [1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 255, 256, 257, 4095, 4097])
def test_lengths_at_tile_edges(dev, L):
    case = Case(dev, L, [L, max(L - 1, 1), L + 1], [1, 1, 1], 4, 2, 16)
    mask = torch.ones(3, 1, dtype=torch.int64)
    _check(case, mask, *_run(case, mask, dev))


def test_rows_that_see_nothing_and_no_sequences(dev):
    case = Case(dev, 21, [6, 40], [6, 4], 8, 2, 16)
    mask = _trees(case, 1, arbitrary=True)
    mask[1] = 0    # no context and an empty mask
    mask[4] = 0
    mask[7] = 0    # its context alone
    _check(case, mask, *_run(case, mask, dev))
    out, lse = _run(case, mask, dev)
    assert bool((out[1] == 0).all()) and bool(torch.isneginf(lse[:, 1]).all())
    none = attention.paged_tree_attention(case.qd[:0], case.k, case.v, case.btd[:0], case.lensd[:0],
                                          mask[:0].to(dev), case.cud[:1], 4)
    assert none.shape == (0, 8, 128)


def test_missing_pages_read_as_zero_rows(dev):
    case = Case(dev, 31, [200, 90, 33], [8, 3, 20], 8, 2, 16, holes=[(0, 1), (0, 12), (1, 0), (2, 2)])
    mask = _trees(case, 2)
    _check(case, mask, *_run(case, mask, dev))


def test_scores_far_apart_and_negative_scales(dev):
    """Later keys far above the first ones (the running maximum is raised), and a negative descale."""
    case = Case(dev, 41, [700, 260], [7, 12], 8, 2, 16, k_sign=-1.0)
    case.fused[:, 0, :, :, :] = (case.fused[:, 0].float() * torch.linspace(0.05, 3.0, case.fused.shape[0]).view(-1, 1, 1, 1)
                                 ).to(torch.float8_e4m3fn)
    case.k.copy_(case.fused[:, 0].to(dev))
    mask = _trees(case, 3)
    _check(case, mask, *_run(case, mask, dev, scale=0.4), scale=0.4)


def test_nan_in_places_that_a_row_does_not_see(dev):
    """A NaN key or value of a drafted token reaches the rows that see it and no other."""
    case = Case(dev, 51, [50, 70], [6, 6], 8, 2, 16, descales=False)
    mask = _trees(case, 4)
    pos = 50 - 6 + 2  # drafted token 2 of sequence 0
    page, row = int(case.bt[0, pos // 16]), pos % 16
    pos1 = 70 - 6 + 4
    page1, row1 = int(case.bt[1, pos1 // 16]), pos1 % 16
    for t, where in ((case.fused, None), (None, (case.k, case.v))):
        k = t[:, 0] if where is None else where[0]
        v = t[:, 1] if where is None else where[1]
        k.view(torch.uint8)[page, row, 0, 5] = 0x7F
        v.view(torch.uint8)[page1, row1, 1, 9] = 0xFF
    # rows past the lengths hold NaN as well
    for b, L in enumerate(case.lens):
        if L % 16:
            p = int(case.bt[b, L // 16])
            for t in (case.k, case.v):
                t.view(torch.uint8)[p, L % 16:] = 0x7F
            case.fused.view(torch.uint8)[p, :, L % 16:] = 0x7F
    got, lse = _run(case, mask, dev)
    assert bool(torch.isnan(got).any()) and not bool(torch.isnan(got).all())
    _check(case, mask, got, lse, nan=True)


def test_the_same_inputs_give_the_same_bits(dev):
    case = Case(dev, 61, [3000, 17, 900], [16, 16, 16], 32, 4, 16)
    mask = _trees(case, 5)
    a, la = _run(case, mask, dev)
    b, lb = _run(case, mask, dev)
    assert torch.equal(a, b) and torch.equal(la, lb)


def test_bounds_are_hints_and_a_kept_workspace(dev):
    """max_seq_len below the real lengths changes nothing but the launch."""
    case = Case(dev, 71, [3000, 17, 900], [16, 3, 9], 16, 4, 16, spare_table=300)
    mask = _trees(case, 5)
    for bound in (1, 900, 3000, None):
        ws = torch.empty(attention.tree_workspace_floats(3, case.TQ, 16, 16, 4, bound or 1 << 20), device=dev)
        got, lse = _run(case, mask, dev, max_seq_len=bound, workspace=ws)
        _check(case, mask, got, lse)


def test_other_stream_and_graph_replay(dev):
    case = Case(dev, 81, [500, 33], [8, 5], 8, 2, 16)
    mask = _trees(case, 9).to(dev)  # (a capture takes no copy from the host)
    want, lse_want = _run(case, mask, dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, lse = _run(case, mask, dev)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(lse, lse_want)
    graphs, outs = [], []
    for _ in range(2):  # two graphs of the same inputs, replayed in turn
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(_run(case, mask, dev))
        graphs.append(gr)
    for r in range(4):
        case.qd.copy_((case.q.float() * (1 + r)).to(case.q.dtype))
        want, lse_want = _run(case, mask, dev)
        torch.cuda.synchronize()
        for gr, (o, l) in zip(graphs, outs):
            gr.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, want) and torch.equal(l, lse_want), r


def test_offsets_past_32_bits(dev):
    """Pages beyond 4 GiB of the cache."""
    ps, Hkv = 16, 8
    page = 2 * ps * Hkv * 128
    P = (1 << 32) // page + 64
    big = torch.zeros(P, 2, ps, Hkv, 128, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
    case = Case(dev, 91, [200, 77], [8, 3], 32, Hkv, ps)
    small = case.fused.shape[0]
    big[P - small:] = case.fused.to(dev)
    case.k, case.v = big[:, 0], big[:, 1]
    case.btd = case.btd + (P - small)
    mask = _trees(case, 8)
    _check(case, mask, *_run(case, mask, dev))


def test_refusals(dev):
    case = Case(dev, 1, [20, 30], [3, 4], 8, 2, 16)
    mask = _trees(case, 1).to(dev)
    good = dict(q=case.qd, k_cache=case.k, v_cache=case.v, block_table=case.btd, seq_lens=case.lensd, tree_mask=mask,
                cu_seqlens_q=case.cud, max_seqlen_q=4)
    attention.paged_tree_attention(**good)
    attention.paged_tree_attention(**{**good, "tree_mask": mask[:, 0]})  # one word: [total_q] too
    bad = [
        ("drafted tokens", dict(max_seqlen_q=65)),
        ("max_seqlen_q", dict(max_seqlen_q=0)),
        (None, dict(tree_mask=mask.to(torch.int32))),
        (None, dict(tree_mask=mask[:3])),
        (None, dict(tree_mask=mask.cpu())),
        ("fp8", dict(k_cache=case.k.to(torch.bfloat16))),
        ("query heads", dict(q=case.qd[:, :7])),
        (None, dict(q=case.qd[:, :, :64])),
        (None, dict(cu_seqlens_q=case.cud.long())),
        ("per sequence", dict(cu_seqlens_q=None, max_seqlen_q=3)),
        (None, dict(seq_lens=case.lensd.cpu())),
        (None, dict(block_table=case.btd.long())),
        (None, dict(out=torch.empty(7, 8, 128, dtype=torch.float16, device=dev))),
        (None, dict(out=torch.empty(6, 8, 128, device=dev))),
        ("finite", dict(softmax_scale=float("inf"))),
        ("descale", dict(k_descale=torch.ones(2, 3, device=dev))),
        ("unsupported dtype", dict(q=case.qd.to(torch.float64))),
    ]
    for match, change in bad:
        with pytest.raises(AssertionError, match=match):
            attention.paged_tree_attention(**{**good, **change})
    with pytest.raises(AssertionError, match="query rows"):
        attention.paged_tree_attention(**{**good, "max_seqlen_q": 3}, validate=True)


# --------------------------------------------------------------------------- #
# steps cut into runs: tables that could name more than 1536 keys
# --------------------------------------------------------------------------- #


def _room(ps, counts=(), Hq=0):
    """Pages past a table's own that make it one of more than 1536 keys, and the step (drafted
    tokens `counts`, Hq heads) at most 2^27 query rows x keys."""
    return -(-max(1600, 2 ** 27 // max(sum(counts) * Hq, 1) if Hq else 0) // ps)


@pytest.mark.parametrize("ps", [16, 24, 7])
@pytest.mark.parametrize("Hq,Hkv", [(32, 8), (8, 1), (4, 4), (6, 2), (40, 1)])
def test_ragged_trees_cut(dev, Hq, Hkv, ps):
    """As test_ragged_trees; 40 and 8 heads over one make blocks of 256 rows and more."""
    rng = np.random.default_rng(Hq + Hkv + ps)
    counts = [int(x) for x in rng.integers(1, 34, 8)]
    counts[3], counts[7] = 0, 33
    lens = [n + int(x) for n, x in zip(counts, rng.integers(0, 900, 8))]
    lens[1] = counts[1]
    lens[5] = max(counts[5] - 2, 0)
    lens[6] = 0
    lens[2] += 2500
    case = Case(dev, 11, lens, counts, Hq, Hkv, ps, spare_rows=3, spare_table=_room(ps, counts, Hq))
    mask = _trees(case, 5)
    _check(case, mask, *_run(case, mask, dev))


@pytest.mark.parametrize("n", [7, 8, 31, 32, 33, 64, 65, 130, 200])
@pytest.mark.parametrize("Hq,Hkv", [(8, 1), (64, 2), (5, 1)])
def test_wide_trees(dev, n, Hq, Hkv):
    """Around blocks of 256 rows and mask words; arbitrary masks with bits past the tree."""
    case = Case(dev, n, [n + 100, n, n + 31, n + 4000], [n, n, max(1, n - 1), n], Hq, Hkv, 16,
                spare_table=_room(16, [n] * 4, Hq))
    mask = _trees(case, 7, words=-(-n // 64) + 1, arbitrary=True)
    _check(case, mask, *_run(case, mask, dev))


@pytest.mark.parametrize("q_dtype", [torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_wide_types_and_strides(dev, q_dtype, out_dtype):
    case = Case(dev, 3, [300, 61, 1025], [33, 40, 37], 16, 2, 16, q_dtype=q_dtype, strided_q=True, head_major=True,
                spare_table=_room(16, [33, 40, 37], 16), spare_rows=2)
    mask = _trees(case, 6)
    _check(case, mask, *_run(case, mask, dev, out_dtype))


@pytest.mark.parametrize("n", [4, 40])
def test_cut_rows_that_see_nothing(dev, n):
    case = Case(dev, 21, [n, 40 + n, n // 2, 0], [n, n, n, n], 8, 1, 16, spare_table=_room(16, [n] * 4, 8))
    mask = _trees(case, 1, arbitrary=True)
    mask[1] = 0          # no context and an empty mask
    mask[n + 1] = 0      # its context alone
    out, lse = _run(case, mask, dev)
    _check(case, mask, out, lse)
    assert bool((out[1] == 0).all()) and bool(torch.isneginf(lse[:, 1]).all())
    assert bool((out[3 * n:] == 0).all()) and bool(torch.isneginf(lse[:, 3 * n:]).all())


@pytest.mark.parametrize("n", [6, 40])
def test_cut_missing_pages(dev, n):
    case = Case(dev, 31, [200 + n, 90 + n, 33 + n], [n, n, n], 8, 1, 16, holes=[(0, 1), (0, 12), (1, 0), (2, 2)],
                spare_table=_room(16, [n] * 3, 8))
    mask = _trees(case, 2)
    _check(case, mask, *_run(case, mask, dev))


@pytest.mark.parametrize("n", [6, 40, 70])
def test_cut_nan_in_places_that_a_row_does_not_see(dev, n):
    case = Case(dev, 51, [50 + n, 70 + n, 2000 + n], [n, n, n], 16, 2, 16, descales=False,
                spare_table=_room(16, [n] * 3, 16))
    mask = _trees(case, 4)
    for b, i, kind, h, d in ((0, 2, 0, 0, 5), (1, 4, 1, 1, 9), (1, n - 1, 1, 0, 127), (2, 0, 1, 1, 64), (2, 3, 0, 1, 0)):
        pos = case.lens[b] - n + i
        page, row = int(case.bt[b, pos // 16]), pos % 16
        (case.k, case.v)[kind].view(torch.uint8)[page, row, h, d] = 0x7F if d % 2 else 0xFF
        case.fused.view(torch.uint8)[page, kind, row, h, d] = 0x7F if d % 2 else 0xFF
    for b, L in enumerate(case.lens):  # rows past the lengths hold NaN as well
        if L % 16:
            p = int(case.bt[b, L // 16])
            for t in (case.k, case.v):
                t.view(torch.uint8)[p, L % 16:] = 0x7F
            case.fused.view(torch.uint8)[p, :, L % 16:] = 0x7F
    got, lse = _run(case, mask, dev)
    assert bool(torch.isnan(got).any()) and not bool(torch.isnan(got).all())
    _check(case, mask, got, lse, nan=True)


@pytest.mark.parametrize("n", [3, 40])
def test_cut_scores_far_apart_and_negative_scales(dev, n):
    case = Case(dev, 41, [1900 + n, 260 + n], [n, n], 8, 1, 16, k_sign=-1.0, spare_table=_room(16, [n] * 2, 8))
    case.fused[:, 0] = (case.fused[:, 0].float() * torch.linspace(0.05, 3.0, case.fused.shape[0]).view(-1, 1, 1, 1)
                        ).to(torch.float8_e4m3fn)
    case.k.copy_(case.fused[:, 0].to(dev))
    mask = _trees(case, 3)
    _check(case, mask, *_run(case, mask, dev, scale=0.4), scale=0.4)


@pytest.mark.parametrize("n,spare", [(2, 0), (2, 200), (70, 800)])
def test_many_sequences(dev, n, spare):
    """More than one window of 64 sequences, some without drafted tokens."""
    rng = np.random.default_rng(3)
    counts = [int(x) for x in rng.integers(0, n + 1, 150)]
    lens = [c + int(x) for c, x in zip(counts, rng.integers(0, 120, 150))]
    case = Case(dev, 91, lens, counts, 8, 1, 8, spare_table=spare)
    mask = _trees(case, 3)
    _check(case, mask, *_run(case, mask, dev))


@pytest.mark.parametrize("n", [2, 40])
def test_pages_of_one_token(dev, n):
    """More page ids than are staged at a time, eight tables' worth of keys in one row."""
    case = Case(dev, 95, [5000, 1030], [n, n], 8, 1, 1)
    mask = _trees(case, 3)
    _check(case, mask, *_run(case, mask, dev))


def test_wide_other_stream_and_graph_replay(dev):
    case = Case(dev, 81, [2500, 133], [40, 37], 8, 1, 16, spare_table=_room(16, [40, 37], 8))
    mask = _trees(case, 9).to(dev)
    want, lse_want = _run(case, mask, dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, lse = _run(case, mask, dev)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(lse, lse_want)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out, lse = _run(case, mask, dev)
    for r in range(3):
        case.qd.copy_((case.q.float() * (1 + r)).to(case.q.dtype))
        want, lse_want = _run(case, mask, dev)
        torch.cuda.synchronize()
        out.fill_(7.0)
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, lse_want)


def test_wide_trees_over_short_contexts(dev):
    """A table of at most 1536 keys, and enough query rows for the wide form."""
    rng = np.random.default_rng(8)
    counts = [int(x) for x in rng.integers(50, 70, 16)]
    counts[4] = 0
    lens = [c + int(x) for c, x in zip(counts, rng.integers(0, 60, 16))]
    lens[7] = counts[7] - 5
    case = Case(dev, 97, lens, counts, 64, 2, 16, spare_table=96 - -(-max(lens) // 16))
    assert sum(counts) * 64 * 1536 >= 8e7
    assert attention.tree_workspace_floats(16, case.TQ, case.max_q, 64, 2, 1536) > 0
    mask = _trees(case, 3)
    _check(case, mask, *_run(case, mask, dev))


# --------------------------------------------------------------------------- #
# what P V loses of the weights
# --------------------------------------------------------------------------- #
#
# A weight is rounded once to fp16 (r = 2^-11 of itself), whose least step is 2^-24; a
# row's largest weight is at least 2^8 where its maximum was last raised, so a weight is
# also off by 2^-25 of 2^-8 times the largest: 2^-33 of the row's sum.  With S = sum
# p |V| vd and vmax the largest |V vd|,
#   |out - exact| <= S (2 d + r + (K + 64) eps) + K 2^-33 vmax,
# beside the output's own rounding.  Where every q~ . K is an exact float32 (small
# integers), d = eps (8 max(|s|, 1) + 4 (1 + 2 max|s|) + K).


def _check_weights(case, mask, got, scale, most, r=2.0 ** -11):
    q, k, v = case.host()
    args = (case.bt.numpy(), case.lens, mask.numpy(), case.cu, scale, *case.ds)
    want, _, _ = T.tree_attention(q, case.name, k, v, *args)
    size, _, _ = T.tree_attention(q, case.name, k, v & 0x7F, *args)
    K = max([1, *case.lens])
    d = EPS * (8 * max(most, 1.0) + 4 * (1 + 2 * most) + K)
    vmax = float(np.abs(O.e4m3fn_to_f32(v)).max())
    tol = size * (2 * d + r + (K + 64) * EPS) + K * 2.0 ** -33 * vmax
    tol = tol + np.abs(want) * (2.0 ** -8 if got.dtype == torch.bfloat16 else 4 * EPS)
    o = got.double().cpu().numpy()
    assert np.isfinite(o[:case.rows]).all()
    err = np.abs(o - want)[:case.rows]
    assert (err <= tol[:case.rows]).all(), f"{(err / tol[:case.rows]).max():.3g} of the bound"


# (drafted tokens, Hq, Hkv, page, wide): uncut, cut (pages shared by a load or not), the prefill kernel's form
_FORMS = [(3, 8, 2, 16, False), (3, 8, 1, 16, True), (3, 8, 1, 24, True), (40, 8, 1, 16, True)]


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,Hq,Hkv,ps,wide", _FORMS)
def test_weights_far_below_the_largest_add_up(dev, n, Hq, Hkv, ps, wide, out_dtype):
    """A first key 2^26 above all others, whose values alone are not zero."""
    L = 1400 if not wide else 3000
    spare = _room(ps, [n] * 2, Hq) if wide else 0
    case = Case(dev, 6, [L + n, L + n + 45], [n, n], Hq, Hkv, ps, descales=False, spare_table=spare)
    case.q = torch.zeros_like(case.q)
    case.q[:, :, 0] = 1
    case.fused = torch.zeros_like(case.fused, dtype=torch.float32)
    case.fused[:, 1] = 1.0
    for b in range(2):
        case.fused[int(case.bt[b, 0]), 0, 0, :, 0] = 1.0
        case.fused[int(case.bt[b, 0]), 1, 0] = 0.0
    case.fused = case.fused.to(torch.float8_e4m3fn)
    case.qd.copy_(case.q)
    case.k.copy_(case.fused[:, 0].to(dev))
    case.v.copy_(case.fused[:, 1].to(dev))
    mask = _trees(case, 2)
    scale = 26 * np.log(2.0)
    got, _ = _run(case, mask, dev, out_dtype=out_dtype, scale=scale)
    _check_weights(case, mask, got, scale, scale)


def _integers(case, dev, seed):
    """Integer queries and keys: every q~ . K is an exact float32."""
    g = torch.Generator().manual_seed(seed)
    case.q = torch.randint(-1, 2, case.q.shape, generator=g).to(case.q.dtype)
    case.fused[:, 0] = torch.randint(-2, 3, case.fused[:, 0].shape, generator=g).float().to(torch.float8_e4m3fn)
    case.qd.copy_(case.q)
    case.k.copy_(case.fused[:, 0].to(dev))
    case.v.copy_(case.fused[:, 1].to(dev))


@pytest.mark.parametrize("n,Hq,Hkv,ps,wide", _FORMS)
def test_a_float32_out_has_both_halves_of_the_weights(dev, n, Hq, Hkv, ps, wide):
    """P as the sum of two fp16, r = 2^-22; few keys a row, so that no rounding averages out."""
    spare = _room(ps, [n] * 3, Hq) if wide else 0
    case = Case(dev, 5, [n + 5, n + 2, n + 9], [n, n, n], Hq, Hkv, ps, descales=False, spare_table=spare)
    _integers(case, dev, 1)
    mask = torch.zeros(case.TQ, -(-n // 64), dtype=torch.int64)  # their contexts alone
    scale = 0.02
    most = float(np.abs(case.q.double().numpy()).sum(-1).max()) * 2 * scale
    for dtype in (torch.float32, torch.bfloat16):
        got, _ = _run(case, mask, dev, out_dtype=dtype, scale=scale)
        _check_weights(case, mask, got, scale, most, r=2.0 ** -22 if dtype == torch.float32 else 2.0 ** -11)
