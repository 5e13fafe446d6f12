"""The 4-bit cache written and read back: every byte against the oracle."""

import numpy as np
import pytest
import torch

from oracle import mxfp4_oracle as M
from pipeswift_amd import cache_ops, impl_utils, metadata, mxfp4_kv

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _values(g, shape, dtype, spread=2.0):
    x = torch.randn(shape, generator=g) * torch.exp(torch.randn(shape[-2:], generator=g) * spread)
    return x.to(dtype)


def _cache(g, P, ps, H, D, dev, head_major=False):
    """(host bytes [P, 2, ps, H, entry], device tensor)"""
    fused = torch.randint(0, 256, (P, 2, ps, H, M.entry_bytes(D)), generator=g, dtype=torch.uint8)
    d = fused.to(dev)
    if head_major:
        d = d.transpose(2, 3).contiguous().transpose(2, 3)
    return fused.numpy().copy(), d


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,H,D,ps", [(1, 1, 32, 1), (3, 5, 64, 24), (130, 8, 128, 16), (77, 1, 96, 7), (9, 2, 256, 64)])
def test_append(dev, dtype, N, H, D, ps):
    g = torch.Generator().manual_seed(N * 7 + D)
    P = -(-N // ps) + 3
    host, cache = _cache(g, P, ps, H, D, dev)
    k, v = _values(g, (N, H, D), dtype), _values(g, (N, H, D), dtype)
    slots = torch.randperm(P * ps, generator=g)[:N].to(torch.int64)
    slots[2::5] = -1
    slots[4::11] = P * ps + 3
    mxfp4_kv.reshape_and_cache_mxfp4(k.to(dev), v.to(dev), cache[:, 0], cache[:, 1], slots.to(dev))
    M.append(k.double().numpy(), v.double().numpy(), host[:, 0], host[:, 1], slots.numpy())
    assert np.array_equal(cache.cpu().numpy(), host)


@pytest.mark.parametrize("dtype,offset", [(torch.bfloat16, 0), (torch.bfloat16, 1), (torch.float32, 1), (torch.float16, 8)])
def test_append_of_a_projections_columns(dev, dtype, offset):
    """Strided heads, on 16-byte boundaries and off them; a cache whose heads lie pages apart."""
    g = torch.Generator().manual_seed(3)
    N, H, D, ps, P = 33, 4, 64, 16, 5
    host, cache = _cache(g, P, ps, H, D, dev, head_major=True)
    wide = _values(g, (N, 3, H * (D + 8)), dtype).to(dev).view(N, -1)
    k = wide[:, offset:offset + H * (D + 8)].unflatten(1, (H, D + 8))[..., :D]
    v = wide[:, 512 + offset:512 + offset + H * D].unflatten(1, (H, D))
    slots = torch.randperm(P * ps, generator=g)[:N].to(torch.int64)
    mxfp4_kv.reshape_and_cache_mxfp4(k, v, cache[:, 0], cache[:, 1], slots.to(dev))
    M.append(k.double().cpu().numpy(), v.double().cpu().numpy(), host[:, 0], host[:, 1], slots.numpy())
    assert np.array_equal(cache.cpu().numpy(), host)


def test_every_bf16_value_at_every_place_of_a_group(dev):
    """All finite bf16 as a group's largest (with smaller ones about it), zeros, NaN and infinities."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    x = bits.view(torch.bfloat16)[:, None].repeat(1, 32)
    g = torch.Generator().manual_seed(1)
    factor = torch.rand(65536, 32, generator=g) * 2 - 1
    place = torch.arange(65536) % 32
    factor[torch.arange(65536), place] = 1.0
    x = torch.where(torch.isfinite(x), x.float() * factor, x.float()).to(torch.bfloat16)
    x[torch.arange(65536), place] = bits.view(torch.bfloat16)
    keys = x.view(512, 32, 128)
    cache = torch.zeros(32, 2, 16, 32, 68, dtype=torch.uint8, device=dev)
    mxfp4_kv.reshape_and_cache_mxfp4(keys.to(dev), keys.flip(0).contiguous().to(dev), cache[:, 0], cache[:, 1],
                                     torch.arange(512, device=dev))
    want = M.quantize(keys.double().numpy())
    got = cache.cpu().numpy()
    assert np.array_equal(got[:, 0].reshape(want.shape), want)
    assert np.array_equal(got[:, 1].reshape(want.shape), want[::-1])


def _gathered(host, bt, cu, starts, D, total):
    rows = np.full((total, host.shape[2], D), np.inf)  # inf: untouched
    for b in range(len(cu) - 1):
        n = cu[b + 1] - cu[b]
        at = range(starts[b], starts[b] + n)
        rows[cu[b]:cu[b + 1]] = M.dequantize(M.rows_of(host, bt[b], at), D)
    return rows


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,D,ps,lens,use_starts", [
    (8, 128, 16, [50, 0, 128, 1], False), (5, 64, 24, [7, 31, 24], True), (1, 96, 1, [5, 9], False),
    (2, 256, 64, [100], True), (3, 32, 16, [0, 0, 3] + [1] * 70, False)])
def test_gather(dev, dtype, H, D, ps, lens, use_starts):
    g = torch.Generator().manual_seed(sum(lens) + D)
    B = len(lens)
    starts = [(7 * b) % 11 if use_starts else 0 for b in range(B)]
    W = max(-(-(n + s) // ps) for n, s in zip(lens, starts)) + 1
    P = B * W + 2
    host, cache = _cache(g, P, ps, H, D, dev, head_major=D == 64)
    # scales around one (fp16 can hold them); any codes
    s0, s1 = D // 2, D // 2 + D // 32
    host[..., s0:s1] = 120 + host[..., s0:s1] % 12
    if dtype != torch.float16:
        host[0, 0, 0, 0, s0], host[1, :, 0, -1, s1 - 1] = 255, 1
    cache.copy_(torch.from_numpy(host))
    bt = torch.randperm(P, generator=g)[:B * W].to(torch.int32).view(B, W)
    bt[0, 0] = 0
    if B > 1:
        bt[-1, 0] = P + 4
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    T = int(cu[-1]) + 3
    k = torch.full((T, H, D), float("inf"), dtype=dtype, device=dev)
    v = torch.full((T, H, D + 8), float("inf"), dtype=dtype, device=dev)[..., :D].contiguous()
    mxfp4_kv.gather_mxfp4(cache[:, 0], k, bt.to(dev), torch.from_numpy(cu).to(dev),
                          seq_starts=torch.tensor(starts, dtype=torch.int32, device=dev) if use_starts else None,
                          src_cache_v=cache[:, 1], dst_v=v)
    for got, c in ((k, host[:, 0]), (v, host[:, 1])):
        want = _gathered(c, bt.numpy(), cu, starts, D, T)
        assert np.array_equal(got.double().cpu().numpy(), want, equal_nan=True)


def test_gather_into_rows_off_the_boundaries(dev):
    g = torch.Generator().manual_seed(9)
    host, cache = _cache(g, 4, 16, 2, 64, dev)
    host[..., 32:34] = 127
    cache.copy_(torch.from_numpy(host))
    wide = torch.zeros(40, 2 * 64 + 3, dtype=torch.bfloat16, device=dev)
    dst = wide[:, 1:129].unflatten(1, (2, 64))
    bt, cu = torch.tensor([[2, 0, 1]], dtype=torch.int32), np.array([0, 40], np.int32)
    mxfp4_kv.gather_mxfp4(cache[:, 1], dst, bt.to(dev), torch.from_numpy(cu).to(dev))
    assert np.array_equal(dst.double().cpu().numpy(), _gathered(host[:, 1], bt.numpy(), cu, [0], 64, 40))
    assert (wide[:, 0] == 0).all() and (wide[:, 129:] == 0).all()


def test_append_kv_cache_takes_a_4_bit_cache(dev):
    g = torch.Generator().manual_seed(4)
    L, P, ps, H, D, N = 2, 6, 16, 8, 128, 20
    fused = torch.zeros(L, P, 2, ps, H, mxfp4_kv.entry_bytes(D), dtype=torch.uint8, device=dev)
    k, v = _values(g, (N, H, D), torch.bfloat16), _values(g, (N, H, D), torch.bfloat16)
    slots = torch.randperm(P * ps, generator=g)[:N].to(torch.int64)
    info = metadata.KVCacheInfo.__new__(metadata.KVCacheInfo)
    info.kv_cache, info.slot_mapping, info.k_scale, info.v_scale = (fused[:, :, 0], fused[:, :, 1]), slots.to(dev), None, None
    impl_utils.append_kv_cache(k.to(dev), v.to(dev), info, 1)
    want = np.zeros(fused.shape, np.uint8)
    M.append(k.double().numpy(), v.double().numpy(), want[1, :, 0], want[1, :, 1], slots.numpy())
    assert np.array_equal(fused.cpu().numpy(), want)


def test_pages_and_tokens_of_the_cache_move_as_others_do(dev):
    """copy_blocks, evict_tokens and commit_draft_tokens on its rows."""
    from oracle import kv_oracle as O
    from oracle import token_oracle as TO
    g = torch.Generator().manual_seed(11)
    L, P, ps, H = 2, 20, 16, 4
    fused = torch.randint(0, 256, (L, P, 2, ps, H, 68), generator=g, dtype=torch.uint8)
    d, want = fused.to(dev), fused.numpy().copy()
    pairs = torch.tensor([[1, 17], [4, 18]], dtype=torch.int64)
    cache_ops.copy_blocks(d, pairs)
    O.copy_blocks(want, pairs.numpy())
    assert np.array_equal(d.cpu().numpy(), want)
    lens, bt = [100, 30], torch.tensor([[0, 3, 5, 7, 9, 11, 13], [2, 4, 0, 0, 0, 0, 0]], dtype=torch.int32)
    dst = torch.tensor([[1, 6, 8], [10, 12, 14]], dtype=torch.int32)
    scores = torch.rand(L, 2, H, 112, generator=g)
    caches = [d[:, :, 0], d[:, :, 1]]
    kept, _ = cache_ops.evict_tokens(caches, scores.to(dev), bt.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev),
                                     dst.to(dev), 40, 2, 8)
    host = [want[:, :, 0], want[:, :, 1]]
    want_kept, _, _ = TO.evict_tokens(host, scores.numpy(), bt.numpy(), lens, dst.numpy(), 40, 2, 8)
    assert np.array_equal(kept.cpu().numpy(), want_kept) and np.array_equal(d.cpu().numpy(), want)
    starts, path, count = [34, 25], [[1, 2, 4], [0, 1, 3]], [3, 2]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    cache_ops.commit_draft_tokens(caches, dst.to(dev), i32(starts), i32(path), i32(count))
    for c in host:
        TO.commit_draft_tokens(c, dst.numpy(), starts, np.asarray(path), count)
    assert np.array_equal(d.cpu().numpy(), want)


def test_write_and_read_replayed_from_a_graph(dev):
    g = torch.Generator().manual_seed(12)
    P, ps, H, D, N = 8, 16, 2, 128, 30
    cache = torch.zeros(P, 2, ps, H, 68, dtype=torch.uint8, device=dev)
    k, v = torch.zeros(N, H, D, dtype=torch.bfloat16, device=dev), torch.zeros(N, H, D, dtype=torch.bfloat16, device=dev)
    slots = torch.arange(N, device=dev) + 3
    bt, cu = torch.arange(P, dtype=torch.int32, device=dev).view(1, P), torch.tensor([0, N], dtype=torch.int32, device=dev)
    starts = torch.tensor([3], dtype=torch.int32, device=dev)
    out = torch.zeros(N, H, D, device=dev)

    def step():
        mxfp4_kv.reshape_and_cache_mxfp4(k, v, cache[:, 0], cache[:, 1], slots)
        mxfp4_kv.gather_mxfp4(cache[:, 1], out, bt, cu, seq_starts=starts)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        x = _values(g, (N, H, D), torch.bfloat16)
        v.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        want = M.dequantize(M.quantize(x.double().numpy()), D)
        assert np.array_equal(out.double().cpu().numpy(), want)


def test_offsets_past_4_gib(dev):
    """Pages 5 GiB apart."""
    P, ps, H, D = 80000, 16, 32, 128
    page = 2 * ps * H * 68  # 69632 bytes
    store = torch.empty(P * page, dtype=torch.uint8, device=dev)
    cache = store.view(P, 2, ps, H, 68)
    far = torch.tensor([P - 1, 3, P // 2], device=dev)
    cache[far] = 0
    g = torch.Generator().manual_seed(2)
    k = _values(g, (48, H, D), torch.bfloat16)
    slots = (far[:, None] * ps + torch.arange(ps, device=dev)).flatten()
    mxfp4_kv.reshape_and_cache_mxfp4(k.to(dev), k.to(dev), cache[:, 0], cache[:, 1], slots)
    out = torch.empty(48, H, D, device=dev)
    mxfp4_kv.gather_mxfp4(cache[:, 1], out, far.to(torch.int32).view(1, 3), torch.tensor([0, 48], dtype=torch.int32, device=dev))
    assert np.array_equal(out.double().cpu().numpy(), M.dequantize(M.quantize(k.double().numpy()), D))


def test_python_refusals(dev):
    k = torch.zeros(4, 2, 128, dtype=torch.bfloat16, device=dev)
    cache = torch.zeros(3, 2, 16, 2, 68, dtype=torch.uint8, device=dev)
    kc, vc = cache[:, 0], cache[:, 1]
    slots = torch.arange(4, device=dev)
    ok = (k, k, kc, vc, slots)
    mxfp4_kv.reshape_and_cache_mxfp4(*ok)
    for i, bad in ((0, k.double()), (0, k[:, :1]), (1, k.half()), (2, kc.view(torch.int8)), (2, kc[..., :64]),
                   (3, vc[:, :, :1]), (4, slots.int()), (4, torch.arange(5, device=dev)), (4, slots.cpu())):
        args = list(ok)
        args[i] = bad
        with pytest.raises(AssertionError):
            mxfp4_kv.reshape_and_cache_mxfp4(*args)
    dst, bt = torch.zeros(8, 2, 128, device=dev), torch.zeros(1, 1, dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 8], dtype=torch.int32, device=dev)
    mxfp4_kv.gather_mxfp4(kc, dst, bt, cu)
    for args in ((kc, dst[..., :64], bt, cu), (kc, dst.double(), bt, cu), (kc, dst, bt.long(), cu), (kc, dst, bt, cu.long()),
                 (kc, dst, bt, cu, 2), (kc, dst, bt, cu, 1, None, vc, None), (kc, dst.transpose(0, 1), bt, cu)):
        with pytest.raises(AssertionError):
            mxfp4_kv.gather_mxfp4(*args)


@pytest.mark.parametrize("dtype", TYPES)
def test_every_code_under_every_scale_byte(dev, dtype):
    """Scales from 2^-127 to past the largest finite value, which is infinity, and NaN: exact in bf16 and
    f32, subnormal results included; rounded to nearest even in fp16."""
    cache = np.zeros((1, 256, 1, 20), np.uint8)  # row s: every code, twice, under scale byte s
    cache[0, :, 0, :16] = np.tile(np.arange(8) * 2 | (np.arange(8) * 2 + 1) << 4, 2)
    cache[0, :, 0, 16] = np.arange(256)
    out = torch.zeros(256, 1, 32, dtype=dtype, device=dev)
    mxfp4_kv.gather_mxfp4(torch.from_numpy(cache).to(dev), out, torch.zeros(1, 1, dtype=torch.int32, device=dev),
                          torch.tensor([0, 256], dtype=torch.int32, device=dev))
    want = M.dequantize(cache[0], 32)
    with np.errstate(over="ignore", invalid="ignore"):
        if dtype == torch.float16:
            want = want.astype(np.float16).astype(np.float64)
        else:  # (bf16 holds all of these values that float32 does)
            want = np.where(np.abs(want) > np.finfo(np.float32).max, np.sign(want) * np.inf, want)
    got = out.double().cpu().numpy()
    assert np.array_equal(got, want, equal_nan=True)
    known = ~np.isnan(want)
    assert np.array_equal(np.signbit(got)[known], np.signbit(want)[known])
