"""Norms with rotation against the oracle in 64 bits, and its appends against the
append's own bytes.

Bound of a result y of type t, made of the two products a c and b s with a = x rstd w:
the sum of squares of D values in float32 is off by a factor of 1 + (8 + 6) e at most
(eight fused adds in a lane, six across lanes), e = 2^-24; its mean, the added eps and
the reciprocal root add 4 e to half of it; x rstd, w c and their product add 3 e; the
final sum e.  18 e of |a c| + |b s| covers all; then the rounding to t, half a step.
"""

import numpy as np
import pytest
import torch

from oracle import mxfp4_oracle as M
from pipeswift_amd import fp8_kv, impl_utils, metadata, mxfp4_kv, reshape_and_cache, rotary

pytestmark = pytest.mark.gpu

STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}


def _table(g, P, rot):
    angle = torch.rand(P, rot // 2, generator=g, dtype=torch.float64) * 6.283
    return torch.cat([torch.cos(angle), torch.sin(angle)], 1).float()


def _check(got, want, size, dtype):
    fine = 18 * 2.0 ** -24 * size
    bound = fine + STEP[dtype] * (np.abs(want) + fine) + TINY[dtype]
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= bound).all(), f"off by {np.max(err / bound):.3f} of the bound"


class Inputs:
    def __init__(self, dev, seed, N, Hq, Hkv, D, rot, dtype, axes=1, norm=True, weight_dtype=None, pos=torch.int64, P=500):
        g = self.g = torch.Generator().manual_seed(seed)
        self.qkv = (torch.randn(N, (Hq + 2 * Hkv) * D, generator=g) * 3).to(dtype)
        self.on_dev = self.qkv.to(dev)
        cut = [Hq * D, Hkv * D, Hkv * D]
        self.host = [x.unflatten(1, (-1, D)) for x in self.qkv.split(cut, 1)]
        self.q, self.k, self.v = [x.unflatten(1, (-1, D)) for x in self.on_dev.split(cut, 1)]
        self.pos = torch.randint(0, P, (axes, N), generator=g).to(pos)
        if axes == 1:
            self.pos = self.pos[0].contiguous()
        half = rot // 2
        self.sections = None if axes == 1 else [half // 4, half * 3 // 8, half - half // 4 - half * 3 // 8]
        self.table = _table(g, P, rot)
        wd = weight_dtype or dtype
        self.w = [(1 + 0.3 * torch.randn(D, generator=g)).to(wd) if norm else None for _ in range(2)]
        self.dtype = dtype
        self.dev = dev
        self.args = dict(positions=self.pos.to(dev), cos_sin=self.table.to(dev), q_weight=None if not norm else self.w[0].to(dev),
                         k_weight=None if not norm else self.w[1].to(dev), sections=self.sections)

    def want(self, i, **kw):
        w = None if self.w[i] is None else self.w[i].double().numpy()
        return M.norm_rope(self.host[i].double().numpy(), self.pos.numpy(), self.table.numpy(), w, sections=self.sections, **kw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("N,Hq,Hkv,D,rot,axes,interleaved,norm", [
    (1, 1, 1, 128, 128, 1, False, True),
    (5, 32, 8, 128, 128, 1, False, True),
    (7, 12, 4, 64, 32, 3, True, True),
    (3, 3, 1, 96, 64, 1, False, False),
    (9, 8, 2, 256, 128, 3, False, True),
    (2, 2, 2, 512, 512, 1, True, True),
    (4, 70, 1, 32, 16, 1, False, True),
    (6, 5, 5, 80, 48, 3, False, False),
    (130, 4, 1, 8, 8, 1, True, True),
])
def test_norm_rope(dev, dtype, N, Hq, Hkv, D, rot, axes, interleaved, norm):
    x = Inputs(dev, N + D, N, Hq, Hkv, D, rot, dtype, axes, norm, pos=torch.int32 if N % 2 else torch.int64)
    q, k = rotary.norm_rope(x.q, x.k, **x.args, interleaved=interleaved)
    for i, got in enumerate((q, k)):
        _check(got, *x.want(i, interleaved=interleaved), dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_float32_weights_one_norm_another_eps_and_places(dev, dtype):
    x = Inputs(dev, 5, 11, 6, 2, 128, 128, dtype, weight_dtype=torch.float32)
    x.w[0], x.args["q_weight"] = None, None
    want = [x.want(i, eps=0.5) for i in range(2)]
    q, k = rotary.norm_rope(x.q, x.k, **x.args, eps=0.5, q_out=x.q, k_out=x.k)  # in place
    assert q is x.q and k is x.k
    for i, got in enumerate((q, k)):
        _check(got, *want[i], dtype)
    assert torch.equal(x.v.cpu(), x.host[2])


def test_rows_of_zeros_and_large_values(dev):
    x = Inputs(dev, 6, 6, 2, 1, 64, 64, torch.bfloat16)
    for t in (x.q, x.host[0]):
        t[0] = 0.0
        t[1] *= 1e15
        t[2] *= 1e-15
        t[3, 0, 5] = float("nan")
    q, _ = rotary.norm_rope(x.q, x.k, **x.args)
    want, size = x.want(0)
    assert torch.isnan(q[3, 0]).all() and (q[0] == 0).all()
    keep = [0, 1, 2, 4, 5]
    _check(q[keep], want[keep], size[keep], torch.bfloat16)
    _check(q[3, 1:], want[3, 1:], size[3, 1:], torch.bfloat16)


@pytest.mark.parametrize("axes", [1, 3])
def test_positions_outside_the_table_turn_to_nan(dev, axes):
    x = Inputs(dev, 7, 5, 3, 1, 128, 64, torch.bfloat16, axes)
    x.pos.view(axes, 5)[-1, 1], x.pos.view(axes, 5)[-1, 3] = -1, 500
    x.args["positions"] = x.pos.to(dev)
    q, _ = rotary.norm_rope(x.q, x.k, **x.args)
    got = torch.isnan(q).cpu().numpy()
    want, size = x.want(0)
    assert np.array_equal(got, np.isnan(want)) and got.any() and not got[0].any() and not got[1, :, 64:].any()
    _check(q[[0, 2, 4]], want[[0, 2, 4]], size[[0, 2, 4]], torch.bfloat16)


def test_infinite_elements_beyond_the_rotation_stay_their_own(dev):
    x = Inputs(dev, 8, 2, 1, 1, 64, 32, torch.bfloat16, norm=False)
    x.q[0, 0, 40] = float("inf")
    q, _ = rotary.norm_rope(x.q, x.k, **x.args)
    assert q[0, 0, 40] == float("inf") and torch.isfinite(q[0, 0, :40]).all() and torch.isfinite(q[0, 0, 41:]).all()


def _caches(g, kind, dtype, P, ps, H, D, dev):
    if kind == "mxfp4":
        return torch.randint(0, 256, (P, 2, ps, H, M.entry_bytes(D)), generator=g, dtype=torch.uint8).to(dev)
    raw = torch.randn(P, 2, ps, H, D, generator=g)
    return raw.to(torch.float8_e4m3fn if kind == "fp8" else dtype).to(dev)


def _bytes(t):
    return t.contiguous().view(torch.uint8)


@pytest.mark.parametrize("kind", ["same", "fp8", "mxfp4"])
@pytest.mark.parametrize("dtype,N,Hq,Hkv,D,rot,ps", [
    (torch.bfloat16, 40, 32, 8, 128, 128, 16), (torch.float16, 17, 6, 2, 64, 32, 24), (torch.float32, 9, 4, 1, 256, 256, 7),
    (torch.bfloat16, 3, 12, 12, 96, 64, 16)])
def test_the_cache_holds_what_norm_rope_and_the_append_would_leave(dev, kind, dtype, N, Hq, Hkv, D, rot, ps):
    x = Inputs(dev, N * 3 + D, N, Hq, Hkv, D, rot, dtype)
    P = -(-N // ps) + 2
    cache = _caches(x.g, kind, dtype, P, ps, Hkv, D, dev)
    other = cache.clone()
    slots = torch.randperm(P * ps, generator=x.g)[:N].to(torch.int64)
    slots[1::6] = -1
    slots[2::9] = P * ps
    slots = slots.to(dev)
    scales = {}
    if kind == "fp8":
        scales = dict(k_scale=torch.tensor([0.037], device=dev), v_scale=torch.tensor([0.21], device=dev))
    q, k = rotary.norm_rope(x.q, x.k, **x.args)
    v = x.v.contiguous()
    if kind == "mxfp4":
        mxfp4_kv.reshape_and_cache_mxfp4(k, v, other[:, 0], other[:, 1], slots)
    else:
        reshape_and_cache.reshape_and_cache_flash(k, v, other[:, 0], other[:, 1], slots, **scales)
    k2 = torch.empty_like(k)
    q2 = rotary.norm_rope_and_cache(x.q, x.k, x.v, cache[:, 0], cache[:, 1], slots, **x.args, **scales, k_out=k2)
    assert torch.equal(_bytes(q), _bytes(q2)) and torch.equal(_bytes(k), _bytes(k2))
    assert torch.equal(_bytes(cache), _bytes(other))
    q3 = rotary.norm_rope_and_cache(x.q, x.k, x.v, cache[:, 0], cache[:, 1], slots, **x.args, **scales)
    assert torch.equal(_bytes(q), _bytes(q3)) and torch.equal(_bytes(cache), _bytes(other))


def test_layer_call_and_graph(dev):
    """impl_utils.norm_rope_append_kv_cache, captured and replayed with other inputs."""
    x = Inputs(dev, 3, 12, 8, 2, 128, 128, torch.bfloat16)
    fused = torch.zeros(2, 4, 2, 16, 2, 128, dtype=torch.bfloat16, device=dev).to(torch.float8_e4m3fn)
    info = metadata.KVCacheInfo.__new__(metadata.KVCacheInfo)
    info.kv_cache, info.slot_mapping = (fused[:, :, 0], fused[:, :, 1]), torch.arange(12, device=dev) + 5
    info.k_scale, info.v_scale = torch.tensor([0.5, 0.25], device=dev), fp8_kv.unit_scale(dev)
    call = lambda: impl_utils.norm_rope_append_kv_cache(x.q, x.k, x.v, **x.args, kv_cache_info=info, layer_idx=1)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = call()
    for seed in (1, 2, 3):
        new = (torch.randn(x.qkv.shape, generator=torch.Generator().manual_seed(seed)) * 2).to(torch.bfloat16)
        x.on_dev.copy_(new)
        fused.view(torch.uint8).zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = _bytes(fused).clone()
        want_q, k = rotary.norm_rope(x.q, x.k, **x.args)
        fused.view(torch.uint8).zero_()
        reshape_and_cache.reshape_and_cache_flash(k, x.v, fused[1, :, 0], fused[1, :, 1], info.slot_mapping,
                                                  info.k_scale[1:2], info.v_scale)
        assert torch.equal(q, want_q) and torch.equal(got, _bytes(fused))
    assert call().shape == (12, 8, 128)


def test_python_refusals(dev):
    x = Inputs(dev, 1, 4, 4, 2, 64, 64, torch.bfloat16)
    wide = torch.zeros(4, 4, 64, dtype=torch.bfloat16, device=dev)
    good = dict(q=x.q, k=x.k, **x.args)
    rotary.norm_rope(**good)
    rotary.norm_rope(**good, q_out=wide)
    for change in (dict(q=x.q.double()), dict(k=x.k.half()), dict(k=x.k[:3]), dict(q=x.q[..., :32]),
                   dict(cos_sin=x.args["cos_sin"].double()), dict(cos_sin=x.args["cos_sin"][:, :24]),
                   dict(positions=x.args["positions"][:3]), dict(positions=x.args["positions"].float()),
                   dict(positions=x.args["positions"].view(1, 4).expand(2, 4)), dict(sections=[16, 16]),
                   dict(q_weight=x.args["q_weight"][:32]), dict(k_weight=x.args["k_weight"].double()),
                   dict(q_out=wide[:3]), dict(q_out=wide.half()), dict(q_out=wide[:, :1].expand(4, 4, 64)), dict(k_out=x.q[:, :2]),
                   dict(q_out=wide.transpose(1, 2)), dict(positions=x.args["positions"].cpu()), dict(eps=-1.0),
                   dict(q_out=x.on_dev[:, 64:64 + 256].unflatten(1, (4, 64)))):
        with pytest.raises(AssertionError):
            rotary.norm_rope(**{**good, **change})
    cache = torch.zeros(2, 2, 16, 2, 64, dtype=torch.bfloat16, device=dev)
    slots = torch.arange(4, device=dev)
    good = dict(good, v=x.v, key_cache=cache[:, 0], value_cache=cache[:, 1], slot_mapping=slots)
    rotary.norm_rope_and_cache(**good)
    for change in (dict(v=x.v[:, :1]), dict(key_cache=cache[:, 0].half()), dict(slot_mapping=slots.int()),
                   dict(slot_mapping=slots[:3]), dict(k_scale=torch.ones(1, device=dev)), dict(value_cache=cache[:, 1, :8]),
                   dict(key_cache=cache[:, 0].to(torch.uint8), value_cache=cache[:, 1].to(torch.uint8))):
        with pytest.raises(AssertionError):
            rotary.norm_rope_and_cache(**{**good, **change})


@pytest.mark.parametrize("kind", ["same", "fp8", "mxfp4"])
@pytest.mark.parametrize("dtype,N,Hq,Hkv,D,rot,axes,interleaved", [
    (torch.bfloat16, 2049, 8, 2, 128, 128, 1, False), (torch.float16, 2111, 5, 3, 96, 64, 3, True),
    (torch.float32, 2050, 2, 2, 32, 32, 1, True), (torch.bfloat16, 2048, 3, 1, 512, 256, 1, False)])
def test_many_tokens(dev, kind, dtype, N, Hq, Hkv, D, rot, axes, interleaved):
    """A prompt's worth, with slots that are skipped: results, and the cache as the append would leave it."""
    x = Inputs(dev, N + D, N, Hq, Hkv, D, rot, dtype, axes)
    ps = 16
    P = -(-N // ps) + 2
    cache, other = (_caches(torch.Generator().manual_seed(1), kind, dtype, P, ps, Hkv, D, dev) for _ in range(2))
    slots = torch.randperm(P * ps, generator=x.g)[:N]
    slots[::7] = -1
    slots[5] = P * ps
    slots = slots.to(dev)
    q, k = rotary.norm_rope(x.q, x.k, **x.args, interleaved=interleaved)
    for i, got in enumerate((q, k)):
        _check(got, *x.want(i, interleaved=interleaved), dtype)
    scales = {}
    if kind == "fp8":
        scales = dict(k_scale=torch.tensor([0.037], device=dev), v_scale=torch.tensor([0.21], device=dev))
    got = rotary.norm_rope_and_cache(x.q, x.k, x.v, cache[:, 0], cache[:, 1], slots, **x.args, **scales,
                                     interleaved=interleaved)
    v = x.v.contiguous()
    if kind == "mxfp4":
        mxfp4_kv.reshape_and_cache_mxfp4(k, v, other[:, 0], other[:, 1], slots)
    else:
        reshape_and_cache.reshape_and_cache_flash(k, v, other[:, 0], other[:, 1], slots, **scales)
    assert torch.equal(_bytes(got), _bytes(q)) and torch.equal(_bytes(cache), _bytes(other))


@pytest.mark.parametrize("kind", ["same", "fp8", "mxfp4"])
def test_layer_calls_over_a_list_of_layers(dev, kind):
    """The layer's calls with each layer's cache a tensor of its own, and scales where 4-bit rows have no use for them."""
    x = Inputs(dev, 4, 9, 8, 2, 128, 128, torch.bfloat16)
    layers, other = ([_caches(torch.Generator().manual_seed(i), kind, torch.bfloat16, 3, 16, 2, 128, dev) for i in range(2)]
                     for _ in range(2))
    info = metadata.KVCacheInfo.__new__(metadata.KVCacheInfo)
    info.slot_mapping = torch.arange(9, device=dev) * 5
    info.k_scale = info.v_scale = None if kind == "same" else torch.tensor([0.5, 0.25], device=dev)
    info.kv_cache = [[c[:, 0] for c in layers], [c[:, 1] for c in layers]]
    q = impl_utils.norm_rope_append_kv_cache(x.q, x.k, x.v, **x.args, kv_cache_info=info, layer_idx=1)
    want, k = rotary.norm_rope(x.q, x.k, **x.args)
    info.kv_cache = [[c[:, 0] for c in other], [c[:, 1] for c in other]]
    impl_utils.append_kv_cache(k, x.v, info, 1)
    assert torch.equal(_bytes(q), _bytes(want))
    assert all(torch.equal(_bytes(a), _bytes(b)) for a, b in zip(layers, other))
    assert not torch.equal(_bytes(layers[1]), _bytes(_caches(torch.Generator().manual_seed(1), kind, torch.bfloat16, 3, 16, 2, 128, dev)))


def test_tables_that_are_broadcasts_or_single_rows(dev):
    """A broadcast table is refused; a table of one row has whatever stride it likes."""
    x = Inputs(dev, 9, 4, 3, 1, 64, 64, torch.bfloat16, P=1)
    with pytest.raises(AssertionError):
        rotary.norm_rope(x.q, x.k, **{**x.args, "cos_sin": x.args["cos_sin"].expand(500, 64)})
    for stride in (0, 3, 64, 1000):
        one = x.args["cos_sin"].as_strided((1, 64), (stride, 1))
        q, k = rotary.norm_rope(x.q, x.k, **{**x.args, "cos_sin": one})
        for i, got in enumerate((q, k)):
            _check(got, *x.want(i), torch.bfloat16)


@pytest.mark.parametrize("N", [6, 2050])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_whose_squares_are_subnormal_without_an_eps(dev, dtype, N):
    """Squares of about 2^-130: each is off by 2^-150 and so is each of their sums, the mean by 2^-149
    with its division, and the reciprocal root by no more than the mean's share of that."""
    x = Inputs(dev, 10, N, 4, 2, 128, 64, dtype)
    for t in (x.on_dev, x.qkv):
        t *= 2.0 ** -66
    for i, got in enumerate(rotary.norm_rope(x.q, x.k, **x.args, eps=0.0)):
        want, size = x.want(i, eps=0.0)
        mean = (x.host[i].double().numpy() ** 2).mean(-1, keepdims=True)
        assert (mean < 2.0 ** -126).any() and (mean > 2.0 ** -131).all()
        _check(got, want, size * (1 + 2.0 ** -149 / mean / (18 * 2.0 ** -24)), dtype)
