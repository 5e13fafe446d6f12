"""GPU parity of ``cache_ops.evict_tokens`` and ``cache_ops.commit_draft_tokens``
with the oracle, bit for bit."""

import numpy as np
import pytest
import torch

from oracle import token_oracle as T
from pipeswift_amd import cache_ops

pytestmark = pytest.mark.gpu


def _bits(t):
    """The tensor's bytes on the host, with its shape."""
    t = t.detach().cpu().contiguous()
    size = t.element_size()
    return t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[size]).numpy()


class Evict:
    def __init__(self, seed, layers, lens, budget, ps, heads=2, row=128, dtype=torch.float8_e4m3fn, shared=False,
                 fused=True, spread=None, holes=()):
        g = torch.Generator().manual_seed(seed)
        B = len(lens)
        need = [-(-n // ps) for n in lens]
        dneed = -(-budget // ps)
        P = sum(need) + B * dneed + 2
        perm = torch.randperm(P, generator=g).to(torch.int32)
        self.bt = torch.full((B, max([1, *need])), -1, dtype=torch.int32)
        at = 0
        for b, k in enumerate(need):
            self.bt[b, :k] = perm[at:at + k]
            at += k
        for b, page in holes:
            self.bt[b, page] = P + 3
        self.dst = perm[at:at + B * dneed].view(B, dneed).contiguous()
        shape = (layers, P, 2, ps, heads, row) if fused else (layers, P, ps, row)
        self.cache = torch.randint(-2 ** 31, 2 ** 31 - 1, shape[:-1] + (-(-shape[-1] * dtype.itemsize // 4),), generator=g,
                                   dtype=torch.int32).view(dtype)[..., :row].contiguous()
        self.views = (lambda c: [c[:, :, 0], c[:, :, 1]]) if fused else (lambda c: [c])
        Hs = 1 if shared or not fused else heads
        self.scores = torch.rand(layers, B, Hs, max([1, *lens]) + 3, generator=g)
        if spread == "ties":
            self.scores = torch.randint(0, 4, self.scores.shape, generator=g).float() - 1.0
            self.scores[self.scores == 0] = -0.0
        elif spread == "odd":
            pick = torch.randint(0, 6, self.scores.shape, generator=g)
            for k, x in enumerate((float("nan"), float("inf"), float("-inf"), 1e-42, -3.0)):
                self.scores[pick == k] = x
        elif spread == "wide":
            self.scores = torch.exp(torch.randn(self.scores.shape, generator=g) * 20).float()
        self.lens, self.budget, self.heads = lens, budget, heads

    def check(self, dev, sink, recent, scores_out=None):
        cache, scores = self.cache.to(dev), self.scores.to(dev)
        lens = torch.tensor(self.lens, dtype=torch.int32, device=dev)
        out = None if scores_out is None else scores_out.to(dev)
        kept, new_lens = cache_ops.evict_tokens(self.views(cache), scores, self.bt.to(dev), lens, self.dst.to(dev),
                                                self.budget, sink=sink, recent=recent, scores_out=out)
        host = _bits(self.cache).copy()
        views = self.views(torch.from_numpy(host))
        views = [v.numpy() if v.dim() == 5 else v.numpy()[:, :, :, None] for v in views]
        ek, el, es = T.evict_tokens(views, self.scores.numpy(), self.bt.numpy(), self.lens, self.dst.numpy(), self.budget,
                                    sink, recent)
        assert np.array_equal(kept.cpu().numpy(), ek), "kept positions"
        assert np.array_equal(new_lens.cpu().numpy(), el)
        if out is None:
            assert np.array_equal(_bits(scores), es.view(np.int32)), "scores in place"
        else:
            assert np.array_equal(_bits(scores), _bits(self.scores)), "the scores are left alone"
            want = scores_out.numpy().copy()
            w = min(want.shape[3], es.shape[3])
            for b, n in enumerate(self.lens):
                want[:, b, :, :min(n, w)] = es[:, b, :, :min(n, w)]
            assert np.array_equal(_bits(out), want.view(np.int32)), "scores in another tensor"
        assert np.array_equal(_bits(cache), host), "cache rows"


@pytest.mark.parametrize("spread", [None, "ties", "odd", "wide"])
@pytest.mark.parametrize("budget,sink,recent", [(40, 4, 16), (40, 0, 0), (40, 40, 0), (40, 0, 40), (1, 0, 0), (33, 32, 0)])
def test_ragged_selection(dev, budget, sink, recent, spread):
    """Lengths around the budget, below it, zero and one, in three layers."""
    lens = [budget + 1, budget, max(budget - 1, 0), 0, 1, 300, 2 * budget + 7, 1025]
    Evict(1, 3, lens, budget, 16, spread=spread).check(dev, sink, recent)


@pytest.mark.parametrize("ps", [1, 7, 16, 64])
@pytest.mark.parametrize("heads,row,dtype,shared", [(8, 128, torch.float8_e4m3fn, False), (1, 128, torch.bfloat16, False),
                                                    (4, 128, torch.bfloat16, True), (3, 20, torch.float8_e4m3fn, False),
                                                    (2, 6, torch.float16, True), (2, 5, torch.uint8, False),
                                                    (2, 64, torch.float32, False)])
def test_layouts(dev, ps, heads, row, dtype, shared):
    Evict(2, 2, [200, 77, 130], 70, ps, heads, row, dtype, shared).check(dev, 3, 9)


def test_latent_cache_and_missing_pages(dev):
    Evict(3, 3, [150, 40, 333], 64, 16, row=576, dtype=torch.bfloat16, fused=False).check(dev, 4, 8)
    Evict(4, 2, [150, 40, 333], 64, 16, holes=[(0, 0), (0, 8), (2, 3)]).check(dev, 4, 8)


@pytest.mark.parametrize("extra", [0, -60, 50])
def test_scores_to_another_tensor(dev, extra):
    e = Evict(5, 2, [200, 60, 130], 64, 16)
    width = e.scores.shape[3] + extra
    e.check(dev, 4, 8, scores_out=torch.full((2, 3, 2, width), 9.0))


@pytest.mark.parametrize("n", [1023, 1024, 1025, 4096, 30000, 33000, 70001])
def test_long_rows(dev, n):
    """Across the workgroup's passes, with many equal scores at the cut."""
    e = Evict(n, 1, [n, n - 1], n // 3, 64, heads=1, row=16)
    e.scores = (e.scores * 50).round()
    e.check(dev, 5, n // 7)
    e.scores.fill_(0.25)
    e.check(dev, 0, 3)


def test_a_length_past_the_scores_and_empty_calls(dev):
    e = Evict(6, 1, [100, 50], 30, 16)
    e.scores = e.scores[..., :80].contiguous()  # sequence 0 is cut to 80 tokens
    e.check(dev, 2, 4)
    e = Evict(7, 1, [10], 4, 16)
    kept, lens = cache_ops.evict_tokens(e.views(e.cache.to(dev)), e.scores[:, :0].to(dev), e.bt[:0].to(dev),
                                        torch.empty(0, dtype=torch.int32, device=dev), e.dst[:0].to(dev), 4)
    assert kept.shape == (1, 0, 2, 4) and lens.shape == (0,)


def test_strided_scores_and_head_major_cache(dev):
    e = Evict(8, 2, [90, 120], 50, 16, heads=4)
    want_cache, want_scores = e.cache.clone(), e.scores.clone()
    views = [v.numpy() for v in e.views(torch.from_numpy(_bits(want_cache).copy()))]
    host = _bits(want_cache).copy()
    views = [host[:, :, 0], host[:, :, 1]]
    ek, _, es = T.evict_tokens(views, want_scores.numpy(), e.bt.numpy(), e.lens, e.dst.numpy(), 50, 2, 6)
    cache = e.cache.to(dev).transpose(3, 4).contiguous().transpose(3, 4)
    wide = torch.zeros(2, 4, 2, e.scores.shape[3] + 10, device=dev).transpose(1, 2)  # heads outside sequences
    s = wide[..., 3:3 + e.scores.shape[3]]
    s.copy_(e.scores)
    bt = torch.zeros(2, e.bt.shape[1] + 2, dtype=torch.int32, device=dev)[:, 1:-1]
    bt.copy_(e.bt)
    kept, _ = cache_ops.evict_tokens([cache[:, :, 0], cache[:, :, 1]], s, bt,
                                     torch.tensor(e.lens, dtype=torch.int32, device=dev), e.dst.to(dev), 50, 2, 6)
    assert np.array_equal(kept.cpu().numpy(), ek)
    assert np.array_equal(_bits(s), es.view(np.int32))
    assert np.array_equal(_bits(cache), host)


def test_graph_replay_and_stream(dev):
    e = Evict(9, 2, [200, 77], 60, 16)
    cache, scores = e.cache.to(dev), e.scores.to(dev)
    bt, dst, lens = e.bt.to(dev), e.dst.to(dev), torch.tensor(e.lens, dtype=torch.int32, device=dev)
    out = torch.zeros_like(scores)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        kept, new = cache_ops.evict_tokens(e.views(cache), scores, bt, lens, dst, 60, 4, 8, scores_out=out)
    for r in range(4):
        scores.copy_(torch.rand(scores.shape, generator=torch.Generator().manual_seed(r)))
        lens.copy_(torch.tensor([200 - r, 58 + r], dtype=torch.int32))
        gr.replay()
        torch.cuda.synchronize()
        ek, el = T.select_tokens(scores.cpu().numpy(), lens.tolist(), 60, 4, 8)
        assert np.array_equal(kept.cpu().numpy(), ek) and np.array_equal(new.cpu().numpy(), el), r
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        k2, _ = cache_ops.evict_tokens(e.views(cache), scores, bt, lens, dst, 60, 4, 8, scores_out=out)
    side.synchronize()
    assert np.array_equal(k2.cpu().numpy(), ek)


def test_evict_refusals(dev):
    e = Evict(10, 1, [50, 60], 20, 16)
    cache = e.cache.to(dev)
    k, v = e.views(cache)
    good = dict(caches=[k, v], scores=e.scores.to(dev), block_table=e.bt.to(dev),
                seq_lens=torch.tensor(e.lens, dtype=torch.int32, device=dev), dst_block_table=e.dst.to(dev), budget=20)
    cache_ops.evict_tokens(**good)
    s = good["scores"]
    bad = [
        ("budget", dict(budget=0)),
        ("budget", dict(sink=12, recent=9)),
        ("budget", dict(sink=-1)),
        ("cannot hold", dict(budget=33)),
        ("own", dict(dst_block_table=good["block_table"])),
        ("scores", dict(scores=s[:, :, :, ::2])),
        ("layers", dict(scores=s.repeat(2, 1, 1, 1))),
        ("layers", dict(scores=torch.zeros(1, 2, 3, 60, device=dev))),
        (None, dict(scores=s.half())),
        (None, dict(scores_out=s[:, :1])),
        ("block_table", dict(block_table=good["block_table"].long())),
        ("block_table", dict(block_table=good["block_table"][:1])),
        ("seq_lens", dict(seq_lens=good["seq_lens"].cpu())),
        ("contiguous", dict(caches=[k[..., ::2], v[..., ::2]])),
        ("layered", dict(caches=k[0, 0])),
        ("GPU", dict(caches=[k.cpu()])),
    ]
    for match, change in bad:
        with pytest.raises(AssertionError, match=match):
            cache_ops.evict_tokens(**{**good, **change})


# --------------------------------------------------------------------------- #
# commits
# --------------------------------------------------------------------------- #


def _commit(dev, seed, shape, dtype, starts, path, lens, views, holes=(), extra=2):
    g = torch.Generator().manual_seed(seed)
    L, P, ps = shape[0], shape[1], shape[-3] if len(shape) == 6 else shape[2]
    cache = torch.randint(-2 ** 31, 2 ** 31 - 1, shape[:-1] + (-(-shape[-1] * dtype.itemsize // 4),), generator=g,
                          dtype=torch.int32).view(dtype)[..., :shape[-1]].contiguous()
    B = len(starts)
    W = -(-(max(starts) + 260) // ps)
    bt = torch.randperm(P, generator=g)[:B * W].view(B, W).to(torch.int32)
    for b, page in holes:
        bt[b, page] = -1
    host = _bits(cache).copy()
    for v in views(torch.from_numpy(host)):
        T.commit_draft_tokens(v.numpy(), bt.numpy(), starts, np.asarray(path), lens)
    d = cache.to(dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    cache_ops.commit_draft_tokens(views(d), bt.to(dev), i32(starts), i32(path), i32(lens))
    assert np.array_equal(_bits(d), host)


_FUSED = lambda c: [c[:, :, 0], c[:, :, 1]]  # noqa: E731
_ONE = lambda c: [c]  # noqa: E731


@pytest.mark.parametrize("ps", [1, 7, 16])
@pytest.mark.parametrize("shape,dtype,views", [((3, 0, 2, 0, 8, 128), torch.float8_e4m3fn, _FUSED),
                                               ((2, 0, 2, 0, 4, 128), torch.bfloat16, _FUSED),
                                               ((2, 0, 0, 576), torch.bfloat16, _ONE),
                                               ((2, 0, 0, 656), torch.uint8, _ONE),
                                               ((2, 0, 0, 7), torch.uint8, _ONE)])
def test_commit_paths(dev, ps, shape, dtype, views):
    """Paths in order, with rows that stay, unsorted ones, a repeated source, none, and negative entries."""
    path = [[0, 2, 5, 9, 30], [0, 1, 2, 0, 0], [4, 4, 4, 1, 0], [7, 0, 0, 0, 0], [3, -1, 6, 2, 8]]
    shape = tuple(ps if i == len(shape) - (3 if len(shape) == 6 else 2) else x for i, x in enumerate(shape))
    shape = (shape[0], 5 * (-(-(500 + 260) // ps)) + 1) + shape[2:]
    _commit(dev, 1, shape, dtype, [0, 37, 63, 200, 500], path, [5, 3, 5, 0, 9], views)


def test_commit_long_paths_and_missing_pages(dev):
    rng = np.random.default_rng(1)
    path = [rng.permutation(256).tolist(), sorted(rng.permutation(256).tolist()), [255 - i for i in range(256)]]
    shape = (2, 100, 2, 16, 2, 128)
    _commit(dev, 2, shape, torch.float8_e4m3fn, [5, 40, 0], path, [256, 256, 255], _FUSED)
    _commit(dev, 3, shape, torch.float8_e4m3fn, [5, 40, 0], path, [256, 100, 1], _FUSED, holes=[(0, 3), (1, 2)])


def test_commit_refusals_and_nothing_to_do(dev):
    cache = torch.zeros(2, 10, 2, 16, 2, 128, dtype=torch.float8_e4m3fn, device=dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    good = dict(caches=_FUSED(cache), block_table=i32([[1, 2], [3, 4]]), starts=i32([3, 4]), path=i32([[1, 2], [0, 3]]),
                path_lens=i32([2, 2]))
    cache_ops.commit_draft_tokens(**good)
    cache_ops.commit_draft_tokens(**{**good, "path": i32([[1, 2], [0, 3]])[:0]})
    cache_ops.commit_draft_tokens(**{**good, "path": i32([[1, 2], [0, 3]])[:, :0]})
    bad = [
        ("at most 256", dict(path=torch.zeros(2, 257, dtype=torch.int32, device=dev))),
        ("path", dict(path=good["path"].long())),
        ("starts", dict(starts=good["starts"][:1])),
        ("path_lens", dict(path_lens=good["path_lens"].cpu())),
        ("block_table", dict(block_table=good["block_table"][:1])),
        ("contiguous", dict(caches=cache[:, :, 0, :, :, ::2])),
        ("layered", dict(caches=cache[0, 0, 0])),
        ("same layers", dict(caches=[cache[:, :, 0], cache[:1, :, 1]])),
    ]
    for match, change in bad:
        with pytest.raises(AssertionError, match=match):
            cache_ops.commit_draft_tokens(**{**good, **change})


def test_commit_replayed_in_a_graph(dev):
    cache = torch.randint(0, 255, (2, 40, 16, 64), dtype=torch.uint8, device=dev)
    bt = torch.randperm(40)[:20].view(2, 10).to(torch.int32)
    starts, lens = torch.tensor([20, 5], dtype=torch.int32, device=dev), torch.tensor([4, 3], dtype=torch.int32, device=dev)
    path = torch.tensor([[0, 3, 5, 11], [2, 3, 4, 0]], dtype=torch.int32, device=dev)
    btd = bt.to(dev)
    host = cache.cpu().numpy().copy()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        cache_ops.commit_draft_tokens(cache, btd, starts, path, lens)
    for r in range(4):
        lens.copy_(torch.tensor([4 - r, 3], dtype=torch.int32))
        gr.replay()
        torch.cuda.synchronize()
        T.commit_draft_tokens(host, bt.numpy(), [20, 5], path.cpu().numpy(), [4 - r, 3])
        assert np.array_equal(cache.cpu().numpy(), host), r


# --------------------------------------------------------------------------- #
# equal scores, rounds of long rows, refusals before anything is written
# --------------------------------------------------------------------------- #


@pytest.mark.parametrize("n,budget,sink,recent", [(40, 12, 0, 0), (5000, 700, 4, 64), (20000, 3000, 4, 64), (40000, 64, 32, 32),
                                                  (16384, 16383, 0, 0), (16385, 1, 0, 0), (4096, 4096, 7, 9), (4097, 4096, 1, 0)])
@pytest.mark.parametrize("value", [0.0, float("nan"), float("-inf"), -1.5])
def test_equal_scores_keep_the_first(dev, n, budget, sink, recent, value):
    e = Evict(3, 1, [n, n // 2], budget, 16, heads=1, row=16)
    e.scores.fill_(value)
    e.check(dev, sink, recent)


def test_many_long_rows(dev):
    """More chunks than one round of launches takes, lengths apart."""
    lens = [17000, 1, 0, 16385, 900, 65540]
    e = Evict(4, 2, lens, 64, 64, heads=69, row=16, dtype=torch.uint8)
    assert 2 * 6 * 69 * 5 > 4096
    e.check(dev, 4, 8)


def test_eviction_refuses_before_it_writes(dev):
    e = Evict(10, 1, [50, 60], 20, 16)
    cache = e.cache.to(dev)
    k, v = e.views(cache)
    scores = e.scores.to(dev)
    good = dict(caches=[k, v], scores=scores, block_table=e.bt.to(dev),
                seq_lens=torch.tensor(e.lens, dtype=torch.int32, device=dev), dst_block_table=e.dst.to(dev), budget=20)
    bad = [
        ("scores_out", dict(scores_out=scores.transpose(1, 2).contiguous().transpose(1, 2).transpose(0, 0)[:, :, :1]
                            .expand(1, 2, 2, scores.shape[3]))),
        ("scores_out", dict(scores_out=torch.as_strided(scores, scores.shape, (0, scores.stride(2), scores.stride(1), 1)))),
        ("block table", dict(block_table=good["block_table"][:, :0])),
        ("layers", dict(caches=[k[:0], v[:0]], scores=scores[:0])),
    ]
    for match, change in bad:
        with pytest.raises(AssertionError, match=match):
            cache_ops.evict_tokens(**{**good, **change})
    torch.cuda.synchronize()
    assert np.array_equal(_bits(scores), _bits(e.scores)) and np.array_equal(_bits(cache), _bits(e.cache))
    none = dict(scores=scores[:, :0], block_table=good["block_table"][:0], seq_lens=good["seq_lens"][:0],
                dst_block_table=good["dst_block_table"][:0])
    kept, lens = cache_ops.evict_tokens(**{**good, **none})
    assert kept.shape == (1, 0, 2, 20) and lens.shape == (0,)


def test_a_path_that_names_a_token_twice(dev):
    """Both rows get the token's; one that stays where it is, is left."""
    _commit(dev, 5, (2, 40, 2, 16, 2, 128), torch.float8_e4m3fn, [5, 33], [[3, 3, 0, 2], [0, 1, 1, 7]], [4, 3], _FUSED)


@pytest.mark.parametrize("shared", [True, False])
def test_a_budget_past_every_length_needs_pages_for_the_tokens_alone(dev, shared):
    e = Evict(12, 2, [30, 20, 0], 100, 16, shared=shared)  # scores of 33 places
    e.dst = e.dst[:, :3].contiguous()
    e.check(dev, 4, 8)
    e.dst = e.dst[:, :2].contiguous()
    with pytest.raises(AssertionError, match="cannot hold"):
        e.check(dev, 4, 8)


@pytest.mark.parametrize("n", [300, 20000])
def test_scores_out_beside_or_over_the_scores(dev, n):
    """Rows between the scores' own are another tensor; views that share elements are refused."""
    e = Evict(13, 2, [n, n // 2], 64, 16)
    w = e.scores.shape[3]
    buf = torch.full((16 * w + 8,), 9.0, device=dev)[:16 * w].view(2, 2, 2, 2 * w)
    scores, other = buf[..., :w], buf[..., w:]
    scores.copy_(e.scores)
    cache = e.cache.to(dev)
    args = dict(block_table=e.bt.to(dev), seq_lens=torch.tensor(e.lens, dtype=torch.int32, device=dev),
                dst_block_table=e.dst.to(dev), budget=64, sink=4, recent=8)
    kept, _ = cache_ops.evict_tokens(e.views(cache), scores, scores_out=other, **args)
    ek, _ = T.select_tokens(e.scores.numpy(), e.lens, 64, 4, 8)
    assert np.array_equal(kept.cpu().numpy(), ek)
    assert torch.equal(scores.cpu(), e.scores)
    for b, k in enumerate(e.lens):
        got = other[:, b, :, :k].cpu()
        want = torch.zeros_like(got)
        want[..., :min(k, 64)] = torch.gather(e.scores[:, b], 2, torch.from_numpy(ek[:, b, :, :min(k, 64)]).long())
        assert torch.equal(got, want)
    before = buf.clone()
    over = [buf[..., 1:w + 1], buf[..., w - 1:], scores.transpose(0, 1), torch.as_strided(buf, (2, 2, 2, w), (4 * w, 2 * w, w, 1), 8 * w - 1),
            torch.as_strided(buf, (2, 2, 2, 2 * w + 1), scores.stride())]  # the same first elements, rows too wide
    over += [torch.as_strided(buf, (2, 2, 2, w), (2 * w, w, w - 1, 1), 0)]
    for out in over:
        with pytest.raises(AssertionError, match="scores_out"):
            cache_ops.evict_tokens(e.views(cache), scores, scores_out=out, **args)
    with pytest.raises(AssertionError, match="scores_out"):  # rows of the scores over each other, in place
        cache_ops.evict_tokens(e.views(cache), over[-1], **args)
    torch.cuda.synchronize()
    assert torch.equal(buf, before)


@pytest.mark.parametrize("heads,row", [(2, 0), (0, 16), (0, 0)])
def test_caches_without_rows_are_refused_before_a_write(dev, heads, row):
    e = Evict(10, 1, [50, 60], 20, 16, shared=True)
    k, v = e.views(e.cache.to(dev))
    scores = e.scores.to(dev)
    none = torch.empty(k.shape[:3] + (heads, row), dtype=k.dtype, device=dev)
    args = (scores, e.bt.to(dev), torch.tensor(e.lens, dtype=torch.int32, device=dev), e.dst.to(dev), 20)
    with pytest.raises(AssertionError, match="rows|heads"):
        cache_ops.evict_tokens([none, none.clone()], *args)
    torch.cuda.synchronize()
    assert np.array_equal(_bits(scores), _bits(e.scores))


@pytest.mark.parametrize("row", [(0,), (2, 0), (0, 16)])
def test_a_cache_without_rows_beside_a_commit(dev, row):
    """Refused before the caches in front of it are written."""
    cache = torch.randint(0, 255, (2, 10, 16, 2, 64), dtype=torch.uint8, device=dev)
    before = cache.clone()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    none = torch.empty(cache.shape[:3] + row, dtype=torch.uint8, device=dev)
    with pytest.raises(AssertionError, match="rows"):
        cache_ops.commit_draft_tokens([cache, none], i32([[1, 2], [3, 4]]), i32([3, 4]), i32([[1, 2], [2, 3]]), i32([2, 2]))
    torch.cuda.synchronize()
    assert torch.equal(cache, before)


def test_a_fused_cache_goes_as_its_views(dev):
    """Its two halves are no page of two tokens."""
    e = Evict(14, 1, [50, 60], 20, 16, shared=True)
    cache = e.cache.to(dev)
    scores = e.scores.to(dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    for caches in (cache, [cache]):
        with pytest.raises(AssertionError, match="K and V views"):
            cache_ops.commit_draft_tokens(caches, i32([[1, 2], [3, 4]]), i32([0, 1]), i32([[1, 2], [2, 3]]), i32([2, 2]))
        with pytest.raises(AssertionError, match="K and V views"):
            cache_ops.evict_tokens(caches, scores, e.bt.to(dev), i32(e.lens), e.dst[:, :1].repeat(1, 20).to(dev), 20)
    torch.cuda.synchronize()
    assert np.array_equal(_bits(cache), _bits(e.cache)) and np.array_equal(_bits(scores), _bits(e.scores))


def test_a_commit_moves_every_cache_once(dev):
    cache = torch.randint(0, 255, (2, 10, 2, 16, 2, 64), dtype=torch.uint8, device=dev)
    other = torch.randint(0, 255, (2, 10, 16, 64), dtype=torch.uint8, device=dev)
    k, v = cache[:, :, 0], cache[:, :, 1]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    args = (i32([[1, 2], [3, 4]]), i32([3, 4]), i32([[1, 2], [2, 3]]), i32([2, 2]))
    before, left = cache.clone(), other.clone()
    for caches in ([k, v, k], [k, other, k], [other, k, v, other]):
        with pytest.raises(AssertionError, match="twice"):
            cache_ops.commit_draft_tokens(caches, *args)
    torch.cuda.synchronize()
    assert torch.equal(cache, before) and torch.equal(other, left)
    cache_ops.commit_draft_tokens([k, k], *args)  # one launch
    once = before.clone()
    cache_ops.commit_draft_tokens(once[:, :, 0], *args)
    assert torch.equal(cache, once)
