"""Tree attention, attention weights, eviction and commits where addresses, layouts and
bounds go further than in their own tests: caches past 4 GiB in every form of the
kernels, K and V apart, NaN in every byte that is not to be read, loose bounds, more
sequences than are ordered, and query layouts that run past the rows."""

import numpy as np
import pytest
import torch

from oracle import token_oracle as T
from pipeswift_amd import attention, cache_ops
from tests import test_gpu_attention_weights as W
from tests.cached_case import Case
from tests.test_gpu_tree_attention import _check, _room, _run, _trees

pytestmark = pytest.mark.gpu

NAN = 0x7F


def _bytes(t):
    return t.view(torch.uint8)


# (drafted tokens, query heads, kv heads, page, cut or wide): uncut; cut, its loads of one
# page each or a look-up a lane; the prefill kernel's form
FORMS = [(5, 8, 2, 16, False), (5, 8, 2, 24, False), (9, 8, 1, 16, True), (9, 8, 1, 24, True), (40, 8, 1, 16, True)]


def _form(dev, seed, form, lens=(300, 61, 1025), **kw):
    n, Hq, Hkv, ps, cut = form
    counts = [n, max(n - 2, 1), n]
    return Case(dev, seed, [L + c for L, c in zip(lens, counts)], counts, Hq, Hkv, ps,
                spare_table=_room(ps, counts, Hq) if cut else 0, **kw)


@pytest.mark.parametrize("holes", [(), ((0, 1), (1, 0), (2, 3))])
@pytest.mark.parametrize("form", FORMS)
def test_no_nan_comes_from_bytes_that_are_not_cached(dev, form, holes):
    """Every byte of the cache that no token of a sequence lies in is NaN."""
    case = _form(dev, 1, form, spare_rows=2, holes=holes)
    owned = torch.zeros(case.fused.shape[0], case.ps, dtype=torch.bool)
    for b, L in enumerate(case.lens):
        pos = torch.arange(L)
        page = case.bt[b, pos // case.ps].long()
        ok = (page >= 0) & (page < owned.shape[0])
        owned[page[ok], (pos % case.ps)[ok]] = True
    where = owned.to(dev)
    for t in (case.k, case.v):
        b = _bytes(t)
        b[~where] = NAN
    _bytes(case.fused)[:, 0][~owned] = NAN
    _bytes(case.fused)[:, 1][~owned] = NAN
    mask = _trees(case, 2)
    out, lse = _run(case, mask, dev)
    assert not bool(torch.isnan(out).any()) and not bool(torch.isnan(lse[:, :case.rows]).any())
    _check(case, mask, out, lse, nan=True)
    scores = W._scores(case)
    for causal in (True, False):
        weights = W._lse(case, causal)
        got = W._run(case, dev, weights, scores, causal)
        assert not bool(torch.isnan(got).any())
        W._check(case, weights, scores, got, causal)


def _apart(case, dev, kind):
    """The case's K and V moved to tensors of their own."""
    k, v = case.k.contiguous(), case.v.contiguous()
    P, ps, H, D = k.shape
    if kind == "same strides":
        case.k, case.v = k, v
    elif kind == "V rows apart":  # a head more than K has, and pages further apart
        wide = torch.full((P, ps + 3, H + 1, D), NAN, dtype=torch.uint8, device=dev).view(v.dtype)
        _bytes(wide)[:, :ps, 1:] = _bytes(v)
        case.k, case.v = k, wide[:, :ps, 1:]
    elif kind == "K rows apart":
        wide = torch.full((P, ps + 1, H + 2, D), NAN, dtype=torch.uint8, device=dev).view(v.dtype)
        _bytes(wide)[:, 1:, :H] = _bytes(k)
        case.k, case.v = wide[:, 1:, :H], v
    else:  # V heads first
        case.k, case.v = k, _bytes(v).transpose(1, 2).contiguous().transpose(1, 2).view(v.dtype)


@pytest.mark.parametrize("kind", ["same strides", "V rows apart", "K rows apart", "V heads first"])
@pytest.mark.parametrize("form", FORMS)
def test_keys_and_values_in_tensors_of_their_own(dev, form, kind):
    case = _form(dev, 2, form)
    _apart(case, dev, kind)
    mask = _trees(case, 3)
    _check(case, mask, *_run(case, mask, dev))
    lse, scores = W._lse(case), W._scores(case)
    W._check(case, lse, scores, W._run(case, dev, lse, scores))


@pytest.mark.parametrize("loose", [1, 4, 200])
@pytest.mark.parametrize("form", FORMS)
def test_a_loose_bound_of_query_tokens(dev, form, loose):
    """max_seqlen_q above every count: other row blocks and runs, other forms, the same results."""
    case = _form(dev, 3, form, spare_rows=3)
    case.max_q += loose
    mask = _trees(case, 4)
    _check(case, mask, *_run(case, mask, dev))
    for decay in (1.0, 0.0):
        lse, scores = W._lse(case), W._scores(case)
        W._check(case, lse, scores, W._run(case, dev, lse, scores, decay=decay), decay=decay)


@pytest.mark.parametrize("B", [1024, 1025])
def test_as_many_sequences_as_are_ordered_and_one_more(dev, B):
    """192 query rows a sequence and a wide table: the prefill kernel's form up to 1024 sequences."""
    rng = np.random.default_rng(B)
    counts = [3] * B
    lens = [3 + int(x) for x in rng.integers(0, 18, B)]
    lens[7], lens[700] = 2, 0
    case = Case(dev, B, lens, counts, 64, 1, 16, spare_table=110)
    assert 3 * 64 >= 192 and sum(counts) * 64 * 110 * 16 >= 8e7
    mask = _trees(case, 5, arbitrary=True)
    _check(case, mask, *_run(case, mask, dev))


@pytest.mark.parametrize("ends", [[0, 4, 9, 30], [0, 4, 9, 2 ** 31 - 1], [-5, 4, 9, 30]])
@pytest.mark.parametrize("wide", [False, True])
def test_query_layouts_that_run_past_the_rows(dev, wide, ends):
    """A sequence has the rows that there are; the others, and rows around them, are left."""
    Hq, Hkv = (64, 1) if wide else (8, 2)
    counts, total = [4, 5, 3], 12
    case = Case(dev, 4, [40, 60, 33], counts, Hq, Hkv, 16, spare_table=_room(16, counts, Hq) if wide else 0)
    case.max_q = 5
    case.cu[0] = max(ends[0], 0)
    mask = _trees(case, 6)
    kw = dict(softmax_scale=case.scale, q_descale=case.dd[0], k_descale=case.dd[1])
    none = ends[0] < 0  # the first sequence begins before the rows: it has none

    def tree(cu):
        room = torch.full((total + 8, Hq, 128), 7.0, device=dev)
        attention.paged_tree_attention(case.qd, case.k, case.v, case.btd, case.lensd, mask.to(dev),
                                       torch.tensor(cu, dtype=torch.int32, device=dev), 5, v_descale=case.dd[2],
                                       out=room[4:4 + total], **kw)
        return room

    want, got = tree([0, 4, 9, 12]), tree(ends)
    assert bool((got[:4] == 7.0).all()) and bool((got[4 + total:] == 7.0).all())
    if none:
        assert bool((got[4:8] == 7.0).all())
    first = 4 if none else 0
    assert torch.equal(got[4 + first:4 + total], want[4 + first:4 + total])
    lse, scores = torch.from_numpy(W._lse(case)).to(dev), W._scores(case)

    def weights(cu, bound):
        return attention.accumulate_attention_weights(
            scores.to(dev), case.qd, case.k, lse, case.btd, case.lensd, torch.tensor(cu, dtype=torch.int32, device=dev),
            bound, **kw)

    for bound in (5, 40):
        want, got = weights([0, 4, 9, 12], bound), weights(ends, 5)
        if none:
            want[0] = scores[0].to(dev)
        assert torch.allclose(got, want, rtol=1e-5, atol=1e-7)


# --------------------------------------------------------------------------- #
# past 4 GiB
# --------------------------------------------------------------------------- #


def _far(case, dev):
    """The case's pages at the end of a cache of more than 4 GiB, the rest of it NaN."""
    page = 2 * case.ps * case.Hkv * 128
    small = case.fused.shape[0]
    P = (1 << 32) // page + 8 + small
    big = torch.full((P, 2, case.ps, case.Hkv, 128), NAN, dtype=torch.uint8, device=dev)
    big[P - small:, 0], big[P - small:, 1] = _bytes(case.k), _bytes(case.v)
    big = big.view(torch.float8_e4m3fn)
    case.k, case.v = big[:, 0], big[:, 1]
    holes = (case.btd < 0) | (case.btd >= small)
    case.btd = torch.where(holes, torch.full_like(case.btd, P), case.btd + (P - small))


@pytest.mark.parametrize("form", FORMS)
def test_trees_and_weights_past_4_gib(dev, form):
    case = _form(dev, 5, form, holes=((0, 1),))
    _far(case, dev)
    mask = _trees(case, 7)
    _check(case, mask, *_run(case, mask, dev))
    lse, scores = W._lse(case), W._scores(case)
    W._check(case, lse, scores, W._run(case, dev, lse, scores))


@pytest.mark.parametrize("n,ps", [(1, 16), (1, 24), (40, 16)])
def test_decode_and_window_weights_past_4_gib(dev, n, ps):
    case = Case(dev, 8, [700 + n, 90 + n], [n, n], 8, 2, ps)
    _far(case, dev)
    lse, scores = W._lse(case), W._scores(case)
    W._check(case, lse, scores, W._run(case, dev, lse, scores, decay=0.5), decay=0.5)


@pytest.mark.parametrize("latent", [False, True])
def test_evictions_and_commits_past_4_gib(dev, latent):
    """Layers 4 GiB apart, pages at their ends: rows moved as in a small cache of the same pages."""
    g = torch.Generator().manual_seed(1)
    layers, ps, lens, budget = 2, 16, [90, 200], 48
    row = (640,) if latent else (2, 128)
    outer = 1 if latent else 2
    page = outer * ps * int(np.prod(row))
    small = 40
    P = (1 << 32) // page + small
    shape = (ps,) + row if latent else (2, ps) + row
    host = torch.randint(0, 255, (layers, small) + shape, generator=g, dtype=torch.uint8)
    big = torch.zeros((layers, P) + shape, dtype=torch.uint8, device=dev)
    big[:, P - small:] = host.to(dev)
    views = (lambda c: [c]) if latent else (lambda c: [c[:, :, 0], c[:, :, 1]])
    perm = torch.randperm(small, generator=g).to(torch.int32)
    bt, dst = perm[:26].view(2, 13), perm[26:32].view(2, 3).contiguous()
    scores = torch.rand(layers, 2, 1 if latent else 2, 210, generator=g)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    cache_ops.evict_tokens(views(big), scores.to(dev), (bt + (P - small)).to(dev), i32(lens), (dst + (P - small)).to(dev),
                           budget, 2, 5)
    want = host.numpy().copy()
    T.evict_tokens([v[..., None, :] if latent else v for v in views(want)], scores.numpy(), bt.numpy(), lens, dst.numpy(),
                   budget, 2, 5)
    assert np.array_equal(big[:, P - small:].cpu().numpy(), want)
    starts, path, count = [60, 190], [[1, 3, 4, 9], [0, 2, 7, 0]], [4, 3]
    cache_ops.commit_draft_tokens(views(big), (bt + (P - small)).to(dev), i32(starts), i32(path), i32(count))
    for v in views(want):
        T.commit_draft_tokens(v, bt.numpy(), starts, np.asarray(path), count)
    assert np.array_equal(big[:, P - small:].cpu().numpy(), want)
    assert not bool(big[:, :P - small].any())
