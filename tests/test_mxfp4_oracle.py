"""The 4-bit oracle against closed forms, and the host-side checks of the C entries
of the 4-bit cache and of the norms with rotation (no pointer given here could be
read)."""

import numpy as np
import pytest

from oracle import mxfp4_oracle as M
from pipeswift_amd import _lib

FAKE = 1 << 20  # aligned, never dereferenced
ARG, DTYPE, WORKSPACE = -1, -2, -4


def test_row_of_known_values():
    x = np.zeros((1, 64))
    x[0, :9] = [6.0, -0.25, 0.75, 1.25, 2.5, -5.0, 0.5, 0.26, 1.75]
    x[0, 32] = 7.0  # not below 7: the next scale, where it is 3.5 and rounds to 4
    row = M.quantize(x)[0]
    assert row.shape == (36,) and list(row[32:]) == [127, 128, 0, 0]
    assert list(M.dequantize(row, 64)[:9]) == [6.0, -0.0, 1.0, 1.0, 2.0, -4.0, 0.5, 0.5, 2.0]
    assert M.dequantize(row, 64)[32] == 8.0
    assert row[0] == 7 | 8 << 4  # the even element low; minus zero keeps its sign


def test_scales_at_the_ends():
    x = np.zeros((5, 32))
    x[1, 3], x[2, 0], x[3, 0], x[4, 5] = 2.0 ** -149, float.fromhex("0x1.fep127"), np.nan, np.inf
    rows = M.quantize(x)
    assert list(rows[:, 16]) == [127, 1, 253, 255, 255]
    v = M.dequantize(rows, 32)
    assert (v[0] == 0).all() and (v[1] == 0).all() and v[2, 0] == 2.0 ** 128
    assert np.isnan(v[3:]).all() and (rows[3:, :16] == 0).all()


def test_every_value_is_within_half_a_step():
    rng = np.random.default_rng(5)
    x = rng.standard_normal((400, 96)) * np.exp(rng.standard_normal((400, 96)) * 3)
    rows = M.quantize(x)
    v = M.dequantize(rows, 96)
    s = np.repeat(np.ldexp(1.0, rows[:, 48:51].astype(int) - 127), 32, -1)
    assert (np.abs(v - x) <= np.maximum(np.abs(x) / 4, s / 4)).all()
    assert (np.abs(x) < 7 * s).all() and (np.abs(x).reshape(400, 3, 32).max(-1) >= 3.5 * s[:, ::32]).all()


def test_entry_bytes():
    for d in (32, 64, 96, 128, 256, 512, 4096):
        assert _lib.lib().psk_mxfp4_entry_bytes(d) == M.entry_bytes(d)
    assert M.entry_bytes(128) == 68 and M.entry_bytes(64) == 36
    for d in (0, -32, 48, 4128):
        assert _lib.lib().psk_mxfp4_entry_bytes(d) == ARG


def _call(entry, good, change):
    assert set(change) <= set(good)
    return getattr(_lib.lib(), entry)(*{**good, **change}.values())


def _refused(entry, good, status, message, change):
    st = _call(entry, good, change)
    assert st == status and message in _lib.lib().psk_last_error(), (st, _lib.lib().psk_last_error())


def _strides(head, **change):
    """Those of rows [token, 4 heads, 128] for each name of ``head``, and of two caches of 4-bit rows."""
    s = dict.fromkeys(head, (4 * 128, 128)) | dict(kc=(2 * 16 * 4 * 68, 4 * 68, 68), vc=(2 * 16 * 4 * 68, 4 * 68, 68))
    assert set(change) <= set(s)
    return _lib.i64_array([x for t in (s | change).values() for x in t])


ENTRIES = _lib.i64_array([2 * 16 * 4 * 68, 4 * 68, 68])
APPEND = dict(k=FAKE, v=FAKE, kc=FAKE, vc=FAKE, slots=FAKE, n=8, H=4, D=128, ps=16, P=10, strides=_strides("kv"), dt=2,
              stream=None)


@pytest.mark.parametrize("status,message,change", [
    (ARG, b"bad sizes", dict(n=-1)),
    (ARG, b"bad sizes", dict(H=0)),
    (ARG, b"bad sizes", dict(D=48)),
    (ARG, b"bad sizes", dict(ps=0)),
    (DTYPE, b"bf16, f16 or f32", dict(dt=3)),
    (ARG, b"NULL", dict(k=None)),
    (ARG, b"NULL", dict(vc=None)),
    (ARG, b"NULL", dict(slots=None)),
    (ARG, b"4-byte", dict(kc=FAKE + 2)),
    (ARG, b"NULL", dict(strides=None)),
    (ARG, b"4-byte", dict(strides=_strides("kv", vc=(2 * 16 * 4 * 68, 4 * 68 + 2, 68)))),
    (ARG, b"shorter", dict(strides=_strides("kv", kc=(16 * 4 * 64, 4 * 64, 64)))),
    (ARG, b"num_tokens", dict(n=1 << 31)),
])
def test_append_refuses(status, message, change):
    _refused("psk_reshape_and_cache_mxfp4", APPEND, status, message, change)


GATHER = dict(c=FAKE, cv=FAKE, d=FAKE, dv=FAKE, bt=FAKE, cu=FAKE, starts=None, B=2, bts=10, btw=10, T=8, H=4, D=128, ps=16,
              P=10, cs=ENTRIES, ds=512, dt=2, stream=None)


@pytest.mark.parametrize("status,message,change", [
    (ARG, b"bad sizes", dict(B=-1)),
    (ARG, b"bad sizes", dict(D=100)),
    (ARG, b"bad sizes", dict(T=1 << 31)),
    (DTYPE, b"read as", dict(dt=3)),
    (ARG, b"NULL", dict(c=None)),
    (ARG, b"NULL", dict(cv=None)),
    (ARG, b"NULL", dict(cu=None)),
    (ARG, b"4-byte", dict(c=FAKE + 1)),
    (ARG, b"row stride", dict(ds=511)),
])
def test_gather_refuses(status, message, change):
    _refused("psk_gather_mxfp4", GATHER, status, message, change)


SECTIONS = _lib.i64_array([16, 24, 24])
NORM_ROPE = dict(q=FAKE, k=FAKE, v=FAKE, qo=FAKE, ko=None, kc=FAKE, vc=FAKE, strides=_strides("qkvop"), dt=2, n=8, Hq=4,
                 Hkv=4, D=128, qw=FAKE, kw=FAKE, wdt=2, eps=1e-6, pos=FAKE, pb=8, pa=8, axes=3, sections=SECTIONS, cs=FAKE,
                 css=128, P=100, rot=128, inter=0, cdt=4, slots=FAKE, ps=16, blocks=10, ksc=None, vsc=None, stream=None)


@pytest.mark.parametrize("status,message,change", [
    (ARG, b"bad sizes", dict(n=-1)),
    (ARG, b"bad sizes", dict(n=1 << 31)),
    (ARG, b"bad sizes", dict(Hq=0, Hkv=0)),
    (ARG, b"head_size", dict(D=132)),
    (ARG, b"head_size", dict(D=520)),
    (ARG, b"rot_dim", dict(rot=0)),
    (ARG, b"rot_dim", dict(rot=144)),
    (ARG, b"rot_dim", dict(rot=24)),
    (ARG, b"rot_dim", dict(rot=12, inter=1)),
    (DTYPE, b"queries and keys", dict(dt=3)),
    (DTYPE, b"weights", dict(wdt=1)),
    (ARG, b"axes", dict(axes=5)),
    (DTYPE, b"positions", dict(pb=2)),
    (ARG, b"eps", dict(eps=-1.0)),
    (ARG, b"eps", dict(eps=float("nan"))),
    (ARG, b"table", dict(P=0)),
    (ARG, b"table", dict(css=64)),
    (DTYPE, b"cache dtype", dict(cdt=1)),
    (ARG, b"multiple of 32", dict(D=80, rot=64)),
    (ARG, b"geometry", dict(ps=0)),
    (ARG, b"NULL", dict(q=None)),
    (ARG, b"NULL", dict(v=None)),
    (ARG, b"NULL", dict(vc=None)),
    (ARG, b"NULL", dict(slots=None)),
    (ARG, b"NULL", dict(sections=None)),
    (ARG, b"NULL", dict(qo=None)),
    (ARG, b"NULL", dict(kc=None, vc=None)),
    (ARG, b"16-byte", dict(q=FAKE + 8)),
    (ARG, b"16-byte", dict(strides=_strides("qkvop", v=(4 * 128 + 4, 128)))),
    (ARG, b"NULL", dict(strides=None)),
    (ARG, b"shorter", dict(strides=_strides("qkvop", kc=(2 * 16 * 4 * 68, 0, 68)))),
    (ARG, b"shorter", dict(strides=_strides("qkvop", vc=(2 * 16 * 4 * 68, 4 * 68, 64)))),
    (ARG, b"4-byte", dict(kc=FAKE + 2)),
    (ARG, b"8-byte", dict(cdt=3, kc=FAKE + 4)),
    (ARG, b"16-byte", dict(cdt=2, kc=FAKE + 8)),
    (ARG, b"scales", dict(ksc=FAKE)),
    (ARG, b"section", dict(sections=_lib.i64_array([16, -1, 49]))),
    (ARG, b"sections", dict(sections=_lib.i64_array([16, 24, 23]))),
])
def test_norm_rope_refuses(status, message, change):
    _refused("psk_norm_rope", NORM_ROPE, status, message, change)


def test_empty_calls_touch_nothing():
    assert _call("psk_reshape_and_cache_mxfp4", APPEND, dict(n=0, k=None, v=None, slots=None)) == 0
    assert _call("psk_gather_mxfp4", GATHER, dict(T=0, d=None, dv=None)) == 0
    assert _call("psk_gather_mxfp4", GATHER, dict(B=0, bt=None)) == 0
    assert _call("psk_norm_rope", NORM_ROPE, dict(n=0, q=None, k=None, v=None, qo=None, pos=None, slots=None)) == 0


STRIDES = _lib.i64_array([2 * 16 * 4 * 68, 4 * 68, 68])
ATTENTION = dict(q=FAKE, qt=8 * 128, qh=128, qdt=2, kc=FAKE, vc=FAKE, ks=STRIDES, vs=STRIDES, bt=FAKE, bts=10, btw=10, lens=FAKE,
                 B=2, Hq=8, Hkv=4, D=128, ps=16, P=10, most=5000, TQ=4, n=2, cu=FAKE, causal=1, scale=0.1, out=FAKE, ot=8 * 128,
                 oh=128, odt=2, lse=None, ls=0, ws=FAKE, wl=1 << 40, stream=None)


@pytest.mark.parametrize("status,message,change", [
    (ARG, b"", dict(B=-1)),
    (ARG, b"", dict(TQ=-1)),
    (ARG, b"", dict(Hq=6)),
    (ARG, b"", dict(Hkv=0)),
    (ARG, b"128", dict(D=64)),
    (ARG, b"max_seqlen_q", dict(n=0)),
    (ARG, b"max_seqlen_q", dict(n=1 << 31)),
    (ARG, b"max_seq_len", dict(most=-1)),
    (ARG, b"without cu_seqlens_q", dict(cu=None, TQ=3)),
    (DTYPE, b"", dict(qdt=3)),
    (DTYPE, b"output dtype", dict(odt=3)),
    (ARG, b"", dict(scale=float("nan"))),
    (ARG, b"", dict(ps=0)),
    (ARG, b"NULL", dict(q=None)),
    (ARG, b"NULL", dict(kc=None)),
    (ARG, b"NULL", dict(vc=None)),
    (ARG, b"NULL", dict(vs=None)),
    (ARG, b"NULL", dict(bt=None)),
    (ARG, b"NULL", dict(lens=None)),
    (ARG, b"NULL", dict(out=None)),
    (ARG, b"align", dict(q=FAKE + 8)),
    (ARG, b"align", dict(kc=FAKE + 2)),
    (ARG, b"4-byte", dict(vc=FAKE + 2)),
    (ARG, b"4-byte", dict(vs=_lib.i64_array([2 * 16 * 4 * 68, 4 * 68, 66]))),
    (ARG, b"8-byte", dict(out=FAKE + 4)),
    (ARG, b"16-byte", dict(odt=0, oh=130)),
    (WORKSPACE, b"need", dict(wl=100)),
    (WORKSPACE, b"need", dict(ws=None)),
])
def test_attention_refuses(status, message, change):
    _refused("psk_paged_mxfp4_attention", ATTENTION, status, message, change)


@pytest.mark.parametrize("change", [dict(B=-1), dict(TQ=-1), dict(n=0), dict(Hq=6), dict(Hkv=0), dict(most=-1), dict(n=1 << 31)])
def test_workspace_of_a_bad_step(change):
    good = dict(B=2, TQ=4, n=2, Hq=8, Hkv=4, most=5000)
    assert _call("psk_paged_mxfp4_workspace_len", good, {}) > 0
    assert _call("psk_paged_mxfp4_workspace_len", good, change) == ARG


def test_empty_attention_touches_nothing():
    assert _call("psk_paged_mxfp4_attention", ATTENTION, dict(TQ=0, q=None, out=None)) == 0
    assert _call("psk_paged_mxfp4_attention", ATTENTION, dict(B=0, TQ=0, lens=None, bt=None)) == 0


def test_a_short_step_needs_no_workspace():
    assert _call("psk_paged_mxfp4_workspace_len", dict(B=2, TQ=2, n=1, Hq=8, Hkv=4, most=1024), {}) == 0


@pytest.mark.parametrize("change", [
    dict(B=65537, TQ=65537, n=1, Hq=256, Hkv=8),               # 2^24 rows and more to join
    dict(B=1024, TQ=1024 * 32, n=33, Hq=1024, Hkv=1024),       # the same, behind the launch for the longer sequences
    dict(B=9 << 20, TQ=9 << 20, n=1, Hq=1, Hkv=1, most=100),   # uncut, 2^32 threads
])
def test_attention_refuses_too_many_rows_before_any_launch(change):
    _refused("psk_paged_mxfp4_attention", ATTENTION, ARG, b"too many rows", change)
