"""Attention over the 4-bit cache against the oracle in 64 bits.

Bounds, e = 2^-24, A the largest sum |q K| of a score, scaled, K the most keys:
  * a score is 128 products, exact for bf16 and f16 queries (an f32 one is a pair of
    bf16, 2^-17 of it off), summed in float32 (128 e A), scaled and offset (8 e max(|s|, 1)):
    off by ds;
  * a weight exp(s - m) is then off by a factor of exp(d), d = ds + 4 e (1 + 2 A);
    it meets V as a pair of bf16, 2^-17 of it off, or (steps of many rows into a 16-bit
    output) rounded to fp16, 2^-11 off, and 2^-25 of the largest weight's 2^-8 at the low end;
  * numerator and denominator are sums of K such (K e), and merged parts (64 e).
So out is off by (2 (exp(d) - 1) + p + (K + 64) 2 e) max |V| and its own rounding, lse
by d + (K + 64) e + 2 e |lse|.
"""

import numpy as np
import pytest
import torch

from oracle import mxfp4_oracle as M
from pipeswift_amd import attention

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


class Case:
    def __init__(self, dev, seed, lens, counts, Hq, Hkv, ps, dtype=torch.bfloat16, holes=(), head_major=False,
                 spare_rows=0, spare_table=0, strided_q=False, spread=1.0, v_shift=0):
        g = self.g = torch.Generator().manual_seed(seed)
        B = len(lens)
        need = [-(-n // ps) for n in lens]
        P = sum(need) + 3
        values = torch.randn(P, 2, ps, Hkv, 128, generator=g) * torch.exp(spread * 0.5 * torch.randn(Hkv, 128, generator=g))
        self.fused = M.quantize(values.double().numpy())
        self.fused[:, 1, ..., 64:] = np.clip(self.fused[:, 1, ..., 64:].astype(int) + v_shift, 1, 254).astype(np.uint8)
        W = max([1, *need]) + spare_table
        perm = torch.randperm(P, generator=g).to(torch.int32)
        self.bt = torch.randint(0, P, (B, W), generator=g, dtype=torch.int32)
        at = 0
        for b, k in enumerate(need):
            self.bt[b, :k] = perm[at:at + k]
            at += k
        for k, (b, page) in enumerate(holes):
            self.bt[b, page] = -3 if k % 2 else P + 5
        self.cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.rows = int(self.cu[-1])
        TQ = self.rows + spare_rows
        self.q = (torch.randn(TQ, Hq, 128, generator=g) * 2).to(dtype)
        self.lens, self.counts, self.Hq, self.Hkv, self.ps, self.dtype = list(lens), list(counts), Hq, Hkv, ps, dtype
        self.dev, self.max_q, self.head_major = dev, max([1, *counts]), head_major
        if strided_q:
            wide = torch.zeros(TQ, Hq * 128 + 256, dtype=dtype, device=dev)
            wide[:, 128:128 + Hq * 128] = self.q.view(TQ, -1).to(dev)
            self.qd = wide[:, 128:128 + Hq * 128].view(TQ, Hq, 128)
        else:
            self.qd = self.q.to(dev)
        self.btd, self.cud = self.bt.to(dev), torch.from_numpy(self.cu).to(dev)
        self.lensd = torch.tensor(self.lens, dtype=torch.int32, device=dev)

    def caches(self):
        f = torch.from_numpy(self.fused).to(self.dev)
        if self.head_major:
            f = f.transpose(2, 3).contiguous().transpose(2, 3)
        return f[:, 0], f[:, 1]

    def run(self, scale=128 ** -0.5, causal=True, **kw):
        k, v = self.caches()
        return attention.paged_mxfp4_attention(self.qd, k, v, self.btd, self.lensd, self.cud, self.max_q, softmax_scale=scale,
                                               causal=causal, return_softmax_lse=True, **kw)

    def want(self, scale=128 ** -0.5, causal=True):
        return M.attention(self.q[:self.rows].double().numpy(), self.fused[:, 0], self.fused[:, 1], self.bt.numpy(), self.lens,
                           self.cu, scale, causal)

    def bounds(self, most, want, lse, out_dtype):
        K = max([1, *self.lens])
        ds = EPS * (128 * most + 8 * max(most, 1.0)) + (2.0 ** -17 * most if self.dtype == torch.float32 else 0.0)
        d = ds + 4 * EPS * (1 + 2 * most)
        vmax = np.nanmax(np.abs(M.dequantize(self.fused[:, 1], 128)))
        p = 2.0 ** -17 if out_dtype == torch.float32 else 2.0 ** -11 + K * 2.0 ** -33
        tol = vmax * (2 * np.expm1(d) + p + 2 * (K + 64) * EPS)
        fine = np.where(np.isfinite(lse), np.abs(lse), 0.0)
        return tol + STEP[out_dtype] * (np.abs(want) + tol), d + (K + 64) * EPS + 2 * EPS * fine

    def check(self, got, want):
        out, lse = got
        w, wl, most = want
        tol, tol_lse = self.bounds(most, w, wl, out.dtype)
        err = np.abs(out[:self.rows].double().cpu().numpy() - w)
        assert (err <= tol).all(), f"out off by {np.nanmax(err / tol):.3f} of the bound"
        gl = lse[:, :self.rows].double().cpu().numpy().T
        assert np.array_equal(np.isneginf(gl), np.isneginf(wl))
        with np.errstate(invalid="ignore"):
            el = np.where(np.isneginf(wl), 0.0, np.abs(gl - wl))
        assert (el <= tol_lse).all(), f"lse off by {np.max(el / tol_lse):.3f} of the bound"


def _both(c, **kw):
    c.check(c.run(**kw), c.want(**{k: v for k, v in kw.items() if k in ("scale", "causal")}))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("Hq,Hkv,ps,lens", [
    (32, 8, 16, [1000]), (8, 8, 16, [1, 31, 32, 33, 200]), (4, 1, 24, [700, 0, 64, 5]), (12, 3, 64, [129, 1100]),
    (6, 6, 1, [40, 77]), (14, 7, 16, [300, 18]), (32, 2, 16, [65, 515]), (20, 10, 48, [222]), (18, 9, 16, [100]),
    (32, 16, 7, [90, 3])])
def test_decode(dev, dtype, Hq, Hkv, ps, lens):
    _both(Case(dev, sum(lens) + Hq, lens, [1] * len(lens), Hq, Hkv, ps, dtype))


@pytest.mark.parametrize("Hq,Hkv,ps,lens", [
    (32, 8, 16, [5000, 1, 2049]), (8, 1, 24, [9000]), (8, 2, 64, [3000, 4100, 0, 1500]), (6, 3, 16, [2000, 2500]),
    (10, 5, 16, [1025])])
def test_cut_contexts(dev, Hq, Hkv, ps, lens):
    """Contexts past what a workgroup takes alone, in runs and records."""
    _both(Case(dev, sum(lens) + Hq, lens, [1] * len(lens), Hq, Hkv, ps, spare_table=2))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("Hq,Hkv,ps,lens,counts", [
    (8, 2, 16, [50, 40, 9], [4, 1, 3]),
    (8, 1, 24, [6, 600, 33, 1], [4, 2, 0, 1]),
    (32, 8, 16, [100, 300], [8, 5]),
    (4, 4, 16, [3, 1300], [7, 33]),          # more query tokens than keys: rows that see nothing
    (8, 2, 16, [65, 130, 64], [65, 100, 1]),
    (16, 1, 16, [300, 20], [20, 20]),
    (2, 1, 32, [700], [300]),
    (40, 1, 16, [70], [9]),
])
def test_several_query_tokens(dev, causal, dtype, Hq, Hkv, ps, lens, counts):
    c = Case(dev, sum(lens) + Hq, lens, counts, Hq, Hkv, ps, dtype, spare_rows=3)
    out = torch.full(c.q.shape, 7.0, dtype=dtype, device=dev)
    _both(c, causal=causal, out=out)
    assert (out[c.rows:] == 7.0).all()


@pytest.mark.parametrize("counts", [[1, 1, 1], [5, 1, 9], [90, 1, 40]])
def test_missing_pages_read_as_zeros(dev, counts):
    _both(Case(dev, 3, [200, 1300, 100], counts, 8, 2, 16, holes=[(0, 3), (1, 0), (1, 70), (2, 6)]))


def test_lengths_past_the_table_and_below_zero(dev):
    c = Case(dev, 4, [100, 64], [2, 2], 8, 2, 16)
    c.lensd = torch.tensor([112 + 20, -5], dtype=torch.int32, device=dev)  # the table has 7 pages
    c.lens = [132, 0]
    _both(c)


@pytest.mark.parametrize("counts", [[1, 1], [6, 2], [70, 30]])
def test_any_strides(dev, counts):
    _both(Case(dev, 5, [150, 1200], counts, 8, 4, 16, head_major=True, strided_q=True))


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("counts", [[1, 1], [40, 30]])
def test_output_types_and_strides(dev, out_dtype, dtype, counts):
    c = Case(dev, 6, [150, 1200], counts, 8, 4, 16, dtype)
    wide = torch.zeros(c.rows, 8, 160, dtype=out_dtype, device=dev)
    _both(c, out=wide[..., 16:144])
    assert (wide[..., :16] == 0).all() and (wide[..., 144:] == 0).all()


@pytest.mark.parametrize("scale", [-0.05, 0.0, 3.0])
@pytest.mark.parametrize("counts", [[1, 1], [50, 3]])
def test_scales(dev, scale, counts):
    """Negative, zero (all weights equal) and so large that single keys take all."""
    _both(Case(dev, 7, [60, 1100], counts, 8, 2, 16), scale=scale)


@pytest.mark.parametrize("counts", [[1, 1], [3, 40]])
@pytest.mark.parametrize("shift", [-60, 60])
def test_values_far_from_one(dev, counts, shift):
    """V beyond fp16's range, and far below it."""
    _both(Case(dev, 8, [60, 1100], counts, 8, 2, 16, v_shift=shift))


@pytest.mark.parametrize("counts", [[1, 1, 1], [5, 8, 3], [60, 100, 65]])
def test_nan_reaches_only_what_sees_it(dev, counts):
    """NaN groups in K and V at the last tokens, and NaN in every byte that no token owns."""
    lens = [70, 1200, 100]
    c = Case(dev, 9, lens, counts, 8, 2, 16)
    used = np.zeros(c.fused.shape[0] * 16, dtype=bool)
    for b, L in enumerate(lens):
        for p in range(L):
            used[c.bt[b, p // 16] * 16 + p % 16] = True
    c.fused.reshape(-1, 2, 16, 2, 68).transpose(0, 2, 1, 3, 4)[~used.reshape(-1, 16)] = 255
    at = lambda b, p: (int(c.bt[b, p // 16]), p % 16)  # noqa: E731
    page, row = at(0, lens[0] - 1)
    c.fused[page, 1, row, 0, 64 + 2] = 255          # V of the last token, one group of one head
    page, row = at(1, lens[1] - 2)
    c.fused[page, 1, row, :, 64:] = 255             # V of the one before the last, all of it
    page, row = at(2, lens[2] - 1)
    c.fused[page, 0, row, 1, 64 + 3] = 255          # K of the last token, one head
    out, lse = c.run()
    with np.errstate(invalid="ignore"):
        w, wl, most = c.want()
    got, gl = out.double().cpu().numpy(), lse.double().cpu().numpy().T
    assert np.array_equal(np.isnan(got), np.isnan(w)) and np.array_equal(np.isnan(gl), np.isnan(wl))
    assert np.isnan(w).any() and not np.isnan(w).all()
    tol, tol_lse = c.bounds(most, np.nan_to_num(w), np.nan_to_num(wl), out.dtype)
    assert (np.nan_to_num(np.abs(got - w)) <= tol).all() and (np.nan_to_num(np.abs(gl - wl)) <= tol_lse).all()


def test_many_sequences(dev):
    lens = [(37 * i) % 90 for i in range(1030)]
    _both(Case(dev, 10, lens, [i % 3 for i in range(1030)], 4, 2, 16), max_seq_len=90)


@pytest.mark.parametrize("bound", [1024, 1025, 2000, 100000])
def test_loose_and_close_bounds(dev, bound):
    c = Case(dev, 11, [700, 20, 1000], [2, 1, 5], 8, 2, 16, spare_table=7000)
    c.max_q = 9
    _both(c, max_seq_len=bound)


def test_a_workspace_of_the_callers_own_and_the_same_bits(dev):
    c = Case(dev, 12, [5000, 3000], [1, 1], 32, 8, 16)
    need = attention.mxfp4_workspace_floats(2, 2, 1, 32, 8, c.bt.shape[1] * 16)
    ws = torch.full((need,), float("nan"), device=dev)
    a, la = c.run(workspace=ws)
    c.check((a, la), c.want())
    for _ in range(3):
        b, lb = c.run()
        assert torch.equal(a, b) and torch.equal(la, lb)


def test_without_cu_seqlens_and_through_the_flash_entry(dev):
    c = Case(dev, 13, [100, 1300], [3, 3], 8, 2, 16)
    k, v = c.caches()
    a = attention.paged_mxfp4_attention(c.qd, k, v, c.btd, c.lensd, None, 3)
    b, lse = attention.flash_attn_varlen_func(c.qd, k, v, 3, c.cud, None, c.lensd, c.btd, causal=True, return_softmax_lse=True)
    assert torch.equal(a, b)
    c.check((b, lse), c.want())
    with pytest.raises(AssertionError):
        attention.flash_attn_varlen_func(c.qd, k, v, 3, c.cud, None, c.lensd, c.btd, k_descale=torch.ones(1, device=dev))


@pytest.mark.parametrize("counts", [[1, 1], [30, 60]])
def test_replayed_from_a_graph_as_lengths_grow(dev, counts):
    c = Case(dev, 14, [1500, 2200], counts, 8, 2, 16)
    k, v = c.caches()
    call = lambda: attention.paged_mxfp4_attention(  # noqa: E731
        c.qd, k, v, c.btd, c.lensd, c.cud, c.max_q, return_softmax_lse=True)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for lens in ([1500, 2200], [100, 64], [1499, 17], [700, 2100]):
        c.lensd.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        c.lens = lens
        c.check(got, c.want())
        eager = call()
        assert torch.equal(got[0], eager[0]) and torch.equal(got[1], eager[1])


def test_on_another_stream(dev):
    c = Case(dev, 15, [100, 3000], [1, 1], 8, 2, 16)
    want = c.want()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = c.run()
    side.synchronize()
    c.check(got, want)


def test_cycle_of_a_layer(dev):
    """Prompt and decode steps as they are used: norm, rotation, append and attention, over one cache."""
    from pipeswift_amd import rotary
    g = torch.Generator().manual_seed(16)
    Hq, Hkv, ps, P, B = 8, 2, 16, 40, 2
    cache = torch.zeros(P, 2, ps, Hkv, 68, dtype=torch.uint8, device=dev)
    host = cache.cpu().numpy()
    bt = torch.randperm(P, generator=g)[:P].to(torch.int32).view(B, -1)
    angle = torch.rand(400, 64, generator=g, dtype=torch.float64) * 6
    table = torch.cat([angle.cos(), angle.sin()], 1).float()
    w = (1 + 0.1 * torch.randn(128, generator=g)).to(torch.bfloat16)
    lens = [0, 0]
    for counts in ([90, 37], [1, 1], [4, 1], [1, 1]):
        n = sum(counts)
        pos = np.concatenate([np.arange(lens[b], lens[b] + counts[b]) for b in range(B)])
        seq = np.repeat(np.arange(B), counts)
        slots = bt.numpy()[seq, pos // ps].astype(np.int64) * ps + pos % ps
        qkv = (torch.randn(n, Hq + 2 * Hkv, 128, generator=g) * 2).to(torch.bfloat16)
        d = qkv.to(dev)
        q = rotary.norm_rope_and_cache(d[:, :Hq], d[:, Hq:Hq + Hkv], d[:, Hq + Hkv:], cache[:, 0], cache[:, 1],
                                       torch.from_numpy(slots).to(dev), torch.from_numpy(pos).to(dev), table.to(dev),
                                       w.to(dev), w.to(dev))
        lens = [a + k for a, k in zip(lens, counts)]
        cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        out, lse = attention.paged_mxfp4_attention(
            q, cache[:, 0], cache[:, 1], bt.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev),
            torch.from_numpy(cu).to(dev), max(counts), return_softmax_lse=True)
        host = cache.cpu().numpy()
        # V as it was given; K within a step of the rotated keys' own rows
        v = M.quantize(qkv[:, Hq + Hkv:].double().numpy())
        assert np.array_equal(host[slots // ps, 1, slots % ps], v)
        k, _ = M.norm_rope(qkv[:, Hq:Hq + Hkv].double().numpy(), pos, table.numpy(), w.double().numpy())
        got = M.dequantize(host[slots // ps, 0, slots % ps], 128)
        s = np.repeat(np.ldexp(1.0, host[slots // ps, 0, slots % ps][..., 64:].astype(int) - 127), 32, -1)
        assert (np.abs(got - k) <= np.maximum(np.abs(k) / 4, s / 4) * (1 + 2.0 ** -6) + 2.0 ** -7 * np.abs(k)).all()
        c = Case.__new__(Case)
        c.lens, c.rows, c.dtype, c.fused = lens, n, torch.bfloat16, host
        c.check((out, lse), M.attention(q.double().cpu().numpy(), host[:, 0], host[:, 1], bt.numpy(), lens, cu, 128 ** -0.5))


def test_offsets_past_4_gib(dev):
    P, ps, Hq, Hkv, L = 80000, 16, 32, 8, 40
    big = torch.empty(P, 4, 2, ps, Hkv, 68, dtype=torch.uint8, device=dev)  # a layer of four: 5.5 GB apart
    cache = big[:, 3]
    c = Case(dev, 17, [L], [1], Hq, Hkv, ps)
    far = torch.tensor([P - 1, 5, P // 2])
    cache[far.to(dev)] = torch.from_numpy(c.fused[c.bt[0, :3].numpy()]).to(dev)
    out, lse = attention.paged_mxfp4_attention(c.qd, cache[:, 0], cache[:, 1], far.to(torch.int32).view(1, 3).to(dev), c.lensd,
                                               None, 1, return_softmax_lse=True)
    c.check((out, lse), c.want())


def test_empty_steps_and_refusals(dev):
    c = Case(dev, 18, [100, 50], [2, 1], 8, 2, 16)
    k, v = c.caches()
    good = dict(q=c.qd, k_cache=k, v_cache=v, block_table=c.btd, seq_lens=c.lensd, cu_seqlens_q=c.cud, max_seqlen_q=2)
    attention.paged_mxfp4_attention(**good)
    none = attention.paged_mxfp4_attention(**{**good, "q": c.qd[:0], "cu_seqlens_q": torch.zeros(3, dtype=torch.int32, device=dev)})
    assert none.shape == (0, 8, 128)
    for change in (dict(q=c.qd[..., :64]), dict(q=c.qd.to(torch.float8_e4m3fn)), dict(q=c.qd[:, :7]), dict(k_cache=k[..., :64]),
                   dict(k_cache=k.view(torch.float8_e4m3fn)), dict(v_cache=v[:, :8]), dict(block_table=c.btd.long()),
                   dict(seq_lens=c.lensd.long()), dict(seq_lens=c.lensd[:1]), dict(max_seqlen_q=0), dict(cu_seqlens_q=None),
                   dict(softmax_scale=float("nan")), dict(out=torch.empty(3, 8, 128, dtype=torch.float64, device=dev)),
                   dict(out=torch.empty(1, 8, 128, device=dev).expand(3, 8, 128)), dict(workspace=torch.empty(1 << 22, device=dev).int()),
                   dict(cu_seqlens_q=torch.tensor([0, 3, 3], dtype=torch.int32, device=dev), validate=True)):
        with pytest.raises(AssertionError):
            attention.paged_mxfp4_attention(**{**good, **change})


@pytest.mark.parametrize("n", [1, 3])
@pytest.mark.parametrize("Hq,Hkv,ps,pad,lens", [
    (16, 16, 16, 0, [600, 40, 1100]),   # two groups of eight heads
    (32, 32, 8, 0, [2100, 9]),
    (8, 8, 8, 0, [777, 3000]),          # a page a unit of loads
    (16, 4, 24, 16, [500, 1300, 2]),    # rows longer than their heads
    (16, 8, 16, 16, [90, 2500]),
    (24, 12, 40, 0, [333, 1100]),       # two groups of six heads, that begin off 16-byte boundaries
    (4, 1, 8, 0, [9000, 17]),           # more pages than are looked up at a time
    (4, 2, 1, 0, [1700, 3]),
])
def test_head_groups_pages_and_padded_rows(dev, n, Hq, Hkv, ps, pad, lens):
    c = Case(dev, sum(lens) + Hq + n, lens, [n] * len(lens), Hq, Hkv, ps)
    f = torch.from_numpy(c.fused).to(dev)
    P, _, _, _, entry = f.shape
    wide = torch.full((P, 2, ps, Hkv * entry + pad), 255, dtype=torch.uint8, device=dev)
    wide[..., :Hkv * entry] = f.flatten(3)
    rows = wide.as_strided(f.shape, (*wide.stride()[:3], entry, 1))
    c.caches = lambda: (rows[:, 0], rows[:, 1])
    _both(c)


@pytest.mark.parametrize("B,Hq,Hkv,n,longest,bound", [
    (16, 32, 8, 1, 2048, 2048),    # uncut past 1024 keys
    (16, 32, 8, 8, 2000, 2048),    # 32 rows a head, uncut and cut
    (16, 32, 8, 8, 2500, 2500),
    (20, 8, 2, 5, 1500, 4000),     # 20 rows: by blocks
    (70, 8, 2, 6, 300, 3000),      # by rows, many of them to join
    (140, 4, 1, 7, 200, 1500),
])
def test_many_rows(dev, B, Hq, Hkv, n, longest, bound):
    lens = [longest if b == 3 else (b * 131) % 400 for b in range(B)]
    _both(Case(dev, B + n, lens, [n] * B, Hq, Hkv, 16), max_seq_len=bound)


@pytest.mark.parametrize("lens,counts", [([1500, 300, 2200, 64], [1, 90, 4, 33]), ([900, 40, 1000, 7], [2, 40, 1, 0])])
def test_few_and_many_rows_in_one_step_replayed_from_a_graph(dev, lens, counts):
    c = Case(dev, 19, lens, counts, 8, 2, 16)
    k, v = c.caches()
    call = lambda: attention.paged_mxfp4_attention(  # noqa: E731
        c.qd, k, v, c.btd, c.lensd, c.cud, c.max_q, return_softmax_lse=True)
    call()
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    got = []
    for g in graphs:
        with torch.cuda.graph(g):
            got.append(call())
    for lens in (lens, [100, 250, 64, 1], lens[::-1]):
        c.lensd.copy_(torch.tensor(lens, dtype=torch.int32))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        c.lens = lens
        want = c.want()
        for x in got:
            c.check(x, want)
        eager = call()
        assert torch.equal(got[0][0], eager[0]) and torch.equal(got[1][1], eager[1])


@pytest.mark.parametrize("byte", [253, 254, 255])
@pytest.mark.parametrize("counts", [[1, 1, 1], [5, 8, 3], [60, 100, 65]])
def test_infinite_values_reach_only_what_sees_them(dev, counts, byte):
    """Codes of 6 under the largest scales, past the largest float, in V of a sequence's last token."""
    lens = [70, 1200, 100]
    c = Case(dev, 20, lens, counts, 8, 2, 16)
    last = lens[1] - 1
    at = (int(c.bt[1, last // 16]), 1, last % 16, 1)
    c.fused[at][64 + 2] = 127
    c.fused[at][32:48] = 0
    w, wl, most = c.want()
    tol, tol_lse = c.bounds(most, w, wl, torch.bfloat16)
    c.fused[at][64 + 2] = byte
    c.fused[at][32:48] = 0x77
    out, lse = c.run()
    got, gl = out.double().cpu().numpy(), lse.double().cpu().numpy().T
    struck = np.zeros(got.shape, bool)
    struck[c.cu[2] - 1, 4:, 64:96] = True  # the heads of kv head 1
    assert not np.isfinite(got[struck]).any()
    assert (np.abs(got - w) <= tol)[~struck].all() and (np.abs(gl - wl) <= tol_lse).all()


def test_sequences_that_share_their_first_pages(dev):
    c = Case(dev, 21, [1500, 1400, 1500], [1, 1, 1], 8, 2, 16)
    c.bt[1, :60] = c.bt[0, :60]
    c.bt[2] = c.bt[0]
    c.btd = c.bt.to(dev)
    _both(c)


class ExactScores(Case):
    """Queries of small whole numbers, so that every q K and every sum of them is exact, and
    V of 6 at the first token, 0 at all others: out is 6 times the first token's weight."""

    def __init__(self, dev, seed, lens, counts, Hq, Hkv, ps, dtype, k_byte=127):
        super().__init__(dev, seed, lens, counts, Hq, Hkv, ps, dtype)
        self.q = torch.randint(-2, 3, self.q.shape, generator=self.g).to(dtype)
        self.qd = self.q.to(dev)
        self.fused[:, 0, ..., 64:] = k_byte
        self.fused[:, 1, ..., :64], self.fused[:, 1, ..., 64:] = 0, 127
        for b in range(len(lens)):
            self.fused[self.bt[b, 0], 1, 0, :, :64] = 0x77


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("counts", [[300, 40], [1, 1]])
def test_weights_under_an_fp16_output_are_finer_than_it(dev, dtype, counts):
    """The scores are exact but for their scaling, an error d of 4 e of the largest; a weight is off by
    2 (exp(d) - 1) of itself, 2^-17 of it as a sum of two 16-bit parts, (K + 64) 2 e by the sums; what
    is left is the output's own rounding, 2^-11 (2^-25 below its normal range), and what the parts
    lose of weights 2^-33 of the largest."""
    c = ExactScores(dev, 31, [300, 700], counts, 8, 2, 16, dtype)
    out = torch.empty(c.q.shape, dtype=torch.float16, device=dev)
    c.run(out=out)
    w, _, most = c.want()
    d = 4 * EPS * max(most, 1.0) * 2
    fine = np.abs(w) * (2 * np.expm1(d) + 2.0 ** -17 + (700 + 64) * 2 * EPS) + 6 * 2.0 ** -33
    err = np.abs(out.double().cpu().numpy() - w)
    tol = fine + 2.0 ** -11 * (np.abs(w) + fine) + 2.0 ** -25
    assert (err <= tol).all(), f"off by {(err / tol).max():.3f} of the bound"


@pytest.mark.parametrize("k_byte", [150, 170, 238])
@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("counts", [[1, 1, 1], [50, 3, 9], [100, 200, 40]])
def test_scores_far_from_zero(dev, counts, dtype, sign, k_byte):
    """Finite scores of one sign, up to 5 10^35, exact but for their scaling: the largest takes all,
    equal ones share.  Values of 1 to 6 under one scale 2^(byte - 127) and queries of 1 and 2 make
    scores of 2^(byte - 123) to 2^(byte - 119) in the exponent of 2, half a scale apart, which is
    2^(byte - 131) there; their rounding is 2^(byte - 144) at most.  So from byte 150 on all but the
    largest have weight 0, and equal scores equal weights: out is off by a sum's division, 4 e of the
    largest |V|, and its own rounding; lse by 6 e of itself (scale, products, log 2, sum)."""
    c = ExactScores(dev, 32, [1500, 70, 200], counts, 8, 2, 16, dtype, k_byte)
    c.q = (torch.randint(1, 3, c.q.shape, generator=c.g) * sign).to(dtype)
    c.qd = c.q.to(dev)
    c.fused[:, 0, ..., :64] = (c.fused[:, 0, ..., :64] & 0x77) | 0x22  # codes 2, 3, 6 and 7
    c.fused[:, 1] = M.quantize(np.random.default_rng(1).standard_normal((*c.fused[:, 1].shape[:-1], 128)))
    (out, lse), (w, wl, _) = c.run(), c.want()
    got, gl = out.double().cpu().numpy(), lse.double().cpu().numpy().T
    see = np.isfinite(wl)
    assert (np.sign(wl[see]) == sign).all() and (np.abs(wl[see]) > 2.0 ** (k_byte - 124)).all()
    tol = STEP[out.dtype] * np.abs(w) + 4 * EPS * np.abs(M.dequantize(c.fused[:, 1], 128)).max()
    assert np.array_equal(np.isneginf(gl), ~see)
    assert (np.abs(got - w) <= tol).all(), f"off by {np.nanmax(np.abs(got - w) / tol):.3f} of the bound"
    assert (np.abs(gl[see] - wl[see]) <= 6 * EPS * np.abs(wl[see])).all()


@pytest.mark.parametrize("counts", [[1, 1], [40, 3], [1, 90]])
def test_scores_past_the_largest_float_are_not_taken_for_no_keys(dev, counts):
    """All of a row's scores minus infinity: NaN, where a row that sees no key is zeros."""
    c = ExactScores(dev, 33, [1300, 50], counts, 8, 2, 16, torch.bfloat16, 254)
    c.qd = torch.full_like(c.qd, -2.0)
    c.fused[:, 0, ..., :64] = 0x77
    out, lse = c.run()
    see = np.concatenate([[L - n + 1 + i > 0 for i in range(n)] for L, n in zip(c.lens, counts)])
    assert torch.isnan(out[torch.from_numpy(see)]).all() and (out[torch.from_numpy(~see)] == 0).all()
    assert torch.isneginf(lse).all()


@pytest.mark.parametrize("causal", [True, False])
def test_blocks_of_more_sequences_than_are_ordered(dev, causal):
    """1100 sequences, among them some without query tokens, of up to 46 rows a kv head: blocks in batch order."""
    lens = [(37 * i) % 90 for i in range(1100)]
    _both(Case(dev, 34, lens, [(5 * i) % 24 for i in range(1100)], 4, 2, 16, spare_rows=2), causal=causal, max_seq_len=90)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("Hq,Hkv,lens,counts", [
    (300, 1, [700, 40], [1, 3]), (520, 2, [1500, 0, 90], [2, 1, 2]), (257, 1, [5], [1]), (1000, 1, [2100], [20])])
def test_more_query_heads_than_a_block_has_rows(dev, dtype, Hq, Hkv, lens, counts):
    _both(Case(dev, Hq, lens, counts, Hq, Hkv, 16, dtype))


@pytest.mark.parametrize("L,n", [(3000, 200), (2600, 20)])
def test_a_chunk_is_cut_the_same_beside_decode_sequences(dev, L, n):
    """The bits of a chunk alone, whose blocks' keys are split over the CUs, and of the same chunk beside
    sequences that go by rows; replayed from one graph as the step turns into other ones of its bounds."""
    lens, counts = [L, *[40 + 13 * i for i in range(31)]], [n] + [1] * 31
    c = Case(dev, 35, lens, counts, 8, 2, 16)
    k, v = c.caches()
    call = lambda: attention.paged_mxfp4_attention(c.qd, k, v, c.btd, c.lensd, c.cud, n, return_softmax_lse=True)  # noqa: E731
    out, lse = call()
    one, one_lse = attention.paged_mxfp4_attention(c.qd[:n], k, v, c.btd[:1], c.lensd[:1], c.cud[:2], n,
                                                   return_softmax_lse=True)
    assert torch.equal(out[:n], one) and torch.equal(lse[:, :n], one_lse)
    c.check((out, lse), c.want())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for counts in ([n] + [1] * 31, [1] * 32, [n // 2 + 1] + [1] * 31, [9] * (n // 9) + [1] * (32 - n // 9)):
        c.cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        c.rows = int(c.cu[-1])
        c.cud.copy_(torch.from_numpy(c.cu))
        graph.replay()
        torch.cuda.synchronize()
        c.check(got, c.want())
        eager = call()
        assert torch.equal(got[0][:c.rows], eager[0][:c.rows]) and torch.equal(got[1][:, :c.rows], eager[1][:, :c.rows])
