"""GPU parity of ``attention.accumulate_attention_weights`` with the float64 oracle.

A weight exp(s - lse) is off by a factor within 1 +- 2 d, d = ds + 8 eps (1 +
max|s| + max|lse|) (cached_case's ds; the rounding of lse log2(e) and of the
argument, the exponential), a sum of N = n G weights by N eps more, and the
addition of the old sum by 2 eps of its own and 1 eps of the result.
"""

import numpy as np
import pytest
import torch

from oracle import token_oracle as T
from pipeswift_amd import attention
from tests.cached_case import EPS, Case, score_error

pytestmark = pytest.mark.gpu


def _lse(case, causal=True):
    """float32 [Hq, TQ] of the attention over the case, from the oracle's scores (-inf: a row that sees nothing)."""
    q, k, _ = case.host()
    qd, kd = (np.ones((case.B, case.Hkv), np.float32) if d is None else d for d in case.ds[:2])
    G = case.Hq // case.Hkv
    lse = np.full((case.Hq, case.TQ), -np.inf)
    for b, h, c0, n, s, _ in T._sequences(q, case.name, k, case.bt.numpy(), case.lens, case.cu, case.scale, qd, kd):
        see = T.causal_visible(n, s.shape[2], causal)
        for i in range(n):
            if see[i].any():
                x = s[i][:, see[i]]
                lse[h * G:(h + 1) * G, c0 + i] = np.logaddexp.reduce(x, axis=1)
    return lse.astype(np.float32)


def _run(case, dev, lse, scores, causal=True, decay=1.0, **kw):
    d = scores.to(dev)
    got = attention.accumulate_attention_weights(
        d, case.qd, case.k, torch.from_numpy(lse).to(dev), case.btd, case.lensd, case.cud, case.max_q,
        softmax_scale=case.scale, q_descale=case.dd[0], k_descale=case.dd[1], causal=causal, decay=decay, **kw)
    assert got is d
    return got


def _check(case, lse, scores, got, causal=True, decay=1.0):
    q, k, _ = case.host()
    want, bound, most = T.attention_weights(scores.numpy(), q, case.name, k, lse, case.bt.numpy(), case.lens, case.cu,
                                            case.scale, *case.ds[:2], causal=causal, decay=decay)
    fin = np.isfinite(lse)
    d = score_error(bound, most) + 8 * EPS * (1 + most + (np.abs(lse[fin]).max() if fin.any() else 0.0))
    N = case.max_q * case.Hq // case.Hkv
    g = got.double().cpu().numpy()
    old = scores.double().numpy()
    tol = np.abs(want) * (2 * d + (N + 1) * EPS) + 4 * EPS * np.abs(np.nan_to_num(old))
    same = np.isnan(g) & np.isnan(want)
    err = np.where(same, 0.0, np.abs(g - want))
    assert (err <= tol).all() or (same | (err <= tol)).all(), f"max err {np.nanmax(err):.3e}"
    for b, L in enumerate(case.lens):  # places past the length keep their bits
        assert np.array_equal(g[b, :, L:], old[b, :, L:], equal_nan=True)
    assert np.array_equal(g[case.B:], old[case.B:], equal_nan=True)


def _scores(case, seed=1, width=None, rows=0):
    g = torch.Generator().manual_seed(seed)
    return torch.rand(case.B + rows, case.Hkv, width or max([1, *case.lens]) + 5, generator=g) * 0.01


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("ps", [16, 24, 7])
@pytest.mark.parametrize("Hq,Hkv", [(32, 8), (8, 1), (4, 4), (6, 2), (40, 1)])
def test_ragged_steps(dev, Hq, Hkv, ps, causal):
    """0 to 70 query tokens over contexts of 0 to 900 tokens, one sequence empty, one shorter than its queries."""
    rng = np.random.default_rng(Hq + ps)
    counts = [int(x) for x in rng.integers(1, 70, 7)]
    counts[2], counts[4] = 0, 1
    lens = [n + int(x) for n, x in zip(counts, rng.integers(0, 900, 7))]
    lens[1], lens[5], lens[6] = counts[1], max(counts[5] - 3, 0), 0
    case = Case(dev, 13, lens, counts, Hq, Hkv, ps, spare_rows=2, spare_table=1)
    lse, scores = _lse(case, causal), _scores(case, rows=1)
    _check(case, lse, scores, _run(case, dev, lse, scores, causal), causal)


@pytest.mark.parametrize("q_dtype", [torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn])
@pytest.mark.parametrize("decay", [1.0, 0.0, 0.5])
def test_types_strides_and_decay(dev, q_dtype, decay):
    case = Case(dev, 5, [300, 61, 1025], [1, 16, 5], 16, 4, 16, q_dtype=q_dtype, strided_q=True, head_major=True)
    lse, scores = _lse(case), _scores(case)
    if decay == 0.0:
        scores[:, :, ::7] = float("nan")  # not read
    got = _run(case, dev, lse, scores, decay=decay)
    if decay == 0.0:
        assert not bool(torch.isnan(got[2, :, :1025]).any())
    _check(case, lse, scores, got, decay=decay)


@pytest.mark.parametrize("L", [1, 2, 31, 32, 33, 127, 128, 129, 511, 512, 513, 4097])
def test_decode_lengths_at_tile_edges(dev, L):
    case = Case(dev, L, [L, max(1, L - 1), L + 1], [1, 1, 1], 8, 2, 16)
    lse, scores = _lse(case), _scores(case)
    _check(case, lse, scores, _run(case, dev, lse, scores))


@pytest.mark.parametrize("n", [15, 16, 17, 32, 33, 64, 257])
def test_windows(dev, n):
    case = Case(dev, n, [n + 700, n, n + 1], [n, n, n], 8, 2, 16)
    lse, scores = _lse(case), _scores(case)
    _check(case, lse, scores, _run(case, dev, lse, scores, decay=0.0), decay=0.0)


def test_the_last_queries_of_a_prompt_by_slices(dev):
    """q and lse sliced along the tokens of a longer call."""
    n, w = 90, 20
    case = Case(dev, 3, [400], [n], 16, 4, 16)
    lse = _lse(case)
    scores = _scores(case)
    lse_d = torch.from_numpy(lse).to(dev)
    cu = torch.tensor([0, w], dtype=torch.int32, device=dev)
    got = attention.accumulate_attention_weights(
        scores.to(dev), case.qd[n - w:], case.k, lse_d[:, n - w:], case.btd, case.lensd, cu, w, case.scale, case.dd[0],
        case.dd[1])
    case.q, case.rows, case.TQ, case.cu, case.counts, case.max_q = case.q[n - w:], w, w, np.array([0, w]), [w], w
    _check(case, lse[:, n - w:], scores, got)


def test_no_query_rows_decay_alone_and_a_narrow_width(dev):
    case = Case(dev, 7, [50, 20], [0, 0], 8, 2, 16)
    scores = _scores(case, width=33)
    got = attention.accumulate_attention_weights(
        scores.to(dev), case.qd, case.k, torch.empty(8, 0, device=dev), case.btd, case.lensd, case.cud, 1, decay=0.5)
    want = scores.clone()
    want[0] *= 0.5
    want[1, :, :20] *= 0.5
    assert torch.equal(got.cpu(), want)
    case = Case(dev, 8, [50, 20], [2, 1], 8, 2, 16)
    lse, scores = _lse(case), _scores(case, width=33)
    _check(case, lse, scores, _run(case, dev, lse, scores))


def test_missing_pages_and_rows_without_keys(dev):
    case = Case(dev, 9, [90, 3, 64], [4, 6, 64], 8, 2, 16, holes=[(0, 2), (2, 0)])
    lse, scores = _lse(case), _scores(case)
    assert np.isneginf(lse).any()  # the drafted positions before a sequence's start
    _check(case, lse, scores, _run(case, dev, lse, scores))


def test_the_same_inputs_give_the_same_bits_and_bounds_are_hints(dev):
    case = Case(dev, 10, [3000, 17, 900], [64, 1, 9], 32, 8, 16, spare_table=100)
    lse, scores = _lse(case), _scores(case)
    a = _run(case, dev, lse, scores)
    for bound in (1, 900, 3000, 1 << 20):
        assert torch.equal(a, _run(case, dev, lse, scores, max_seq_len=bound))


def test_streams_and_graph_replay(dev):
    case = Case(dev, 12, [500, 33], [1, 1], 8, 2, 16)
    lse = torch.from_numpy(_lse(case)).to(dev)
    kw = dict(softmax_scale=case.scale, q_descale=case.dd[0], k_descale=case.dd[1])
    args = (case.qd, case.k, lse, case.btd, case.lensd, case.cud, 1)
    total = torch.zeros(2, 2, 512, device=dev)
    want = torch.zeros(2, 2, 512, device=dev)
    attention.accumulate_attention_weights(total.clone(), *args, **kw)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        attention.accumulate_attention_weights(total, *args, **kw)
    for _ in range(4):
        gr.replay()
        torch.cuda.synchronize()
        attention.accumulate_attention_weights(want, *args, **kw)
        torch.cuda.synchronize()
        assert torch.equal(total, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attention.accumulate_attention_weights(total, *args, **kw)
    side.synchronize()
    attention.accumulate_attention_weights(want, *args, **kw)
    assert torch.equal(total, want)


def test_refusals(dev):
    case = Case(dev, 1, [20, 30], [3, 4], 8, 2, 16)
    lse = torch.from_numpy(_lse(case)).to(dev)
    good = dict(scores=torch.zeros(2, 2, 32, device=dev), q=case.qd, k_cache=case.k, lse=lse, block_table=case.btd,
                seq_lens=case.lensd, cu_seqlens_q=case.cud, max_seqlen_q=4)
    attention.accumulate_attention_weights(**good)
    bad = [
        ("scores", dict(scores=torch.zeros(1, 2, 32, device=dev))),
        ("scores", dict(scores=torch.zeros(2, 8, 32, device=dev))),
        ("scores", dict(scores=torch.zeros(2, 2, 64, device=dev)[:, :, ::2])),
        (None, dict(scores=torch.zeros(2, 2, 32, device=dev, dtype=torch.float64))),
        (None, dict(scores=torch.zeros(2, 2, 32))),
        (None, dict(lse=lse[:, :5])),
        ("lse", dict(lse=lse.t().contiguous().t())),
        (None, dict(lse=lse.double())),
        ("finite", dict(decay=float("nan"))),
        ("finite", dict(softmax_scale=float("inf"))),
        ("max_seqlen_q", dict(max_seqlen_q=0)),
        ("per sequence", dict(cu_seqlens_q=None, max_seqlen_q=2)),
        ("query heads", dict(q=case.qd[:, :7])),
        ("fp8", dict(k_cache=case.k.to(torch.bfloat16))),
    ]
    for match, change in bad:
        with pytest.raises(AssertionError, match=match):
            attention.accumulate_attention_weights(**{**good, **change})


# --------------------------------------------------------------------------- #
# many query rows a key
# --------------------------------------------------------------------------- #


@pytest.mark.parametrize("n", [1, 7, 8, 9, 20, 33, 64, 100])
@pytest.mark.parametrize("Hq,Hkv", [(40, 1), (5, 1), (12, 4), (9, 3), (64, 1), (2, 2)])
def test_shapes_of_row_tiles(dev, n, Hq, Hkv):
    """Tiles of 32 rows as heads by tokens, neither a multiple of the tile."""
    case = Case(dev, n + Hq, [n + 200, n, max(n - 2, 0), n + 1], [n, n, n, max(n // 2, 1)], Hq, Hkv, 16, spare_rows=1)
    lse, scores = _lse(case), _scores(case)
    _check(case, lse, scores, _run(case, dev, lse, scores, decay=0.5), decay=0.5)


@pytest.mark.parametrize("strided", [True, False])
@pytest.mark.parametrize("causal", [True, False])
def test_many_rows_of_fp8_queries(dev, strided, causal):
    """Read where they lie, without a workspace."""
    case = Case(dev, 6, [300, 61, 1025], [30, 16, 50], 15, 3, 24, q_dtype=torch.float8_e4m3fn, strided_q=strided)
    assert attention.weights_workspace_bytes(case.TQ, case.max_q, 15, 3, case.qd.dtype) == 0
    lse, scores = _lse(case, causal), _scores(case)
    _check(case, lse, scores, _run(case, dev, lse, scores, causal), causal)


@pytest.mark.parametrize("n", [3, 40])
def test_many_sequences(dev, n):
    """More than one window of 64 sequences, some without query tokens, whose sums decay all the same."""
    rng = np.random.default_rng(2)
    counts = [int(x) for x in rng.integers(0, n + 1, 150)]
    lens = [c + int(x) for c, x in zip(counts, rng.integers(0, 90, 150))]
    case = Case(dev, 14, lens, counts, 8, 2, 8)
    lse, scores = _lse(case), _scores(case)
    _check(case, lse, scores, _run(case, dev, lse, scores, decay=0.25), decay=0.25)


@pytest.mark.parametrize("n", [1, 40])
def test_pages_of_one_token_and_long_rows(dev, n):
    case = Case(dev, 15, [4100, 1030], [n, n], 4, 2, 1)
    lse, scores = _lse(case), _scores(case)
    _check(case, lse, scores, _run(case, dev, lse, scores))


@pytest.mark.parametrize("n", [2, 40])
def test_nan_keys_that_a_row_does_not_see(dev, n):
    """A NaN key gives its own column NaN and no other; one that no query sees, none."""
    case = Case(dev, 16, [60 + n, 30 + n], [n, n], 8, 2, 16)
    lse, scores = _lse(case), _scores(case)
    want = _run(case, dev, lse, scores)
    page, row = int(case.bt[0, 1]), 3
    case.k.view(torch.uint8)[page, row, 1, 7] = 0x7F
    for b, L in enumerate(case.lens):
        if L % 16:
            case.k.view(torch.uint8)[int(case.bt[b, L // 16]), L % 16:] = 0x7F
    got = _run(case, dev, lse, scores)
    assert bool(torch.isnan(got[0, 1, 19]))
    got[0, 1, 19] = want[0, 1, 19]
    assert torch.equal(got, want)


def test_a_query_row_of_nan_reaches_the_keys_it_sees(dev):
    n = 20
    case = Case(dev, 17, [70], [n], 4, 1, 16, descales=False)
    lse, scores = _lse(case), _scores(case)
    want = _run(case, dev, lse, scores)
    case.qd[5, 2, 9] = float("nan")
    got = _run(case, dev, lse, scores)
    assert bool(torch.isnan(got[0, 0, :56]).all())
    assert torch.equal(got[0, 0, 56:], want[0, 0, 56:])


def test_scores_that_are_a_broadcast_are_refused(dev):
    case = Case(dev, 1, [20, 30], [3, 4], 8, 2, 16)
    lse = torch.from_numpy(_lse(case)).to(dev)
    with pytest.raises(AssertionError, match="broadcast"):
        attention.accumulate_attention_weights(torch.zeros(1, 2, 32, device=dev).expand(2, 2, 32), case.qd, case.k, lse,
                                               case.btd, case.lensd, case.cud, 4)


def test_many_rows_replayed_in_a_graph(dev):
    case = Case(dev, 18, [500, 133], [40, 30], 8, 2, 16)
    lse = torch.from_numpy(_lse(case)).to(dev)
    kw = dict(softmax_scale=case.scale, q_descale=case.dd[0], k_descale=case.dd[1], decay=0.5)
    args = (case.qd, case.k, lse, case.btd, case.lensd, case.cud, 40)
    total, want = torch.zeros(2, 2, 512, device=dev), torch.zeros(2, 2, 512, device=dev)
    attention.accumulate_attention_weights(total.clone(), *args, **kw)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        attention.accumulate_attention_weights(total, *args, **kw)
    for r in range(4):
        case.qd.copy_((case.q.float() * (1 + r)).to(case.q.dtype))
        gr.replay()
        torch.cuda.synchronize()
        attention.accumulate_attention_weights(want, *args, **kw)
        torch.cuda.synchronize()
        assert torch.equal(total, want)
