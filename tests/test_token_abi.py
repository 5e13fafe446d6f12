"""The C entries of tree attention, attention weights, selection, moves and
commits refuse bad arguments on the host, before any device call (no pointer
given here could be read)."""

import pytest
import torch

from pipeswift_amd import _lib, attention, cache_ops

FAKE = 1 << 20  # aligned, never dereferenced
ARG, DTYPE, WORKSPACE = -1, -2, -4


def _call(entry, names, good, **change):
    args = {**good, **change}
    assert list(args) == names
    return getattr(_lib.lib(), entry)(*args.values())


STRIDES = _lib.i64_array([2 * 16 * 4 * 128, 4 * 128, 128])

TREE = dict(q=FAKE, q_tok=8 * 128, q_head=128, q_dtype=2, k=FAKE, v=FAKE, ks=STRIDES, vs=STRIDES, bt=FAKE, bts=100, btw=100,
            lens=FAKE, B=2, Hq=8, Hkv=4, D=128, ps=16, P=64, max_len=1600, TQ=8, n=4, cu=None, mask=FAKE, mask_stride=1,
            mask_words=1, scale=0.1, qd=None, kd=None, vd=None, ds=None, out=FAKE, out_tok=8 * 128, out_head=128,
            out_dtype=2, lse=None, lse_stride=0, ws=FAKE, ws_len=1 << 40, stream=None)


@pytest.mark.parametrize("status,message,change", [
    (ARG, b"head counts", dict(Hq=7)),
    (ARG, b"head counts", dict(Hkv=0)),
    (ARG, b"head_size", dict(D=64)),
    (ARG, b"max_seqlen_q", dict(n=0)),
    (ARG, b"rows", dict(n=3)),
    (ARG, b"geometry", dict(ps=0)),
    (ARG, b"geometry", dict(P=0)),
    (ARG, b"geometry", dict(btw=0)),
    (ARG, b"finite", dict(scale=float("nan"))),
    (ARG, b"mask words", dict(mask_words=0)),
    (ARG, b"mask words", dict(TQ=130, n=65)),
    (ARG, b"max_seq_len", dict(max_len=-1)),
    (ARG, b"NULL", dict(k=None)),
    (ARG, b"NULL", dict(v=None)),
    (ARG, b"NULL", dict(mask=None)),
    (ARG, b"NULL", dict(out=None)),
    (ARG, b"16-byte", dict(k=FAKE + 8)),
    (ARG, b"16-byte", dict(v=FAKE + 8)),
    (ARG, b"16-byte", dict(vs=_lib.i64_array([2 * 16 * 4 * 128, 4 * 128 + 8, 128]))),
    (ARG, b"query rows", dict(q_tok=8 * 128 + 1)),
    (ARG, b"output rows", dict(out_tok=8 * 128 + 1)),
    (DTYPE, b"output dtype", dict(out_dtype=1)),
    (DTYPE, b"query dtype", dict(q_dtype=9)),
    (WORKSPACE, b"workspace", dict(ws_len=16)),
    (WORKSPACE, b"workspace", dict(ws=None)),
    (ARG, b"sequences", dict(B=1 << 30, TQ=0, cu=FAKE)),
    (ARG, b"total_q", dict(TQ=1 << 30, cu=FAKE)),
])
def test_tree_attention_refuses(status, message, change):
    st = _call("psk_paged_tree_attention", list(TREE), TREE, **change)
    assert st == status and message in _lib.lib().psk_last_error(), _lib.lib().psk_last_error()


def test_tree_workspace_and_empty_steps():
    lib = _lib.lib()
    assert lib.psk_paged_tree_workspace_len(2, 8, 4, 8, 4, 1536) == 0  # nothing is merged
    cut = lib.psk_paged_tree_workspace_len(2, 8, 4, 8, 4, 1537)
    assert cut > 0
    assert lib.psk_paged_tree_workspace_len(4, 256, 64, 32, 4, 60000) > cut  # wide
    for bad in ((2, 8, 0, 8, 4, 1), (2, 8, 4, 7, 4, 1), (-1, 8, 4, 8, 4, 1), (2, 8, 4, 8, 0, 1), (2, 8, 4, 8, 4, -1)):
        assert lib.psk_paged_tree_workspace_len(*bad) == ARG
    assert _call("psk_paged_tree_attention", list(TREE), TREE, B=0, TQ=0, q=None, out=None, ws=None, ws_len=0) == 0
    assert _call("psk_paged_tree_attention", list(TREE), TREE, TQ=0, cu=FAKE, q=None, out=None, ws=None, ws_len=0) == 0


WEIGHTS = dict(scores=FAKE, seq=4 * 200, head=200, width=200, q=FAKE, q_tok=8 * 128, q_head=128, q_dtype=2, k=FAKE, ks=STRIDES,
               lse=FAKE, lse_stride=64, bt=FAKE, bts=100, btw=100, lens=FAKE, B=2, Hq=8, Hkv=4, D=128, ps=16, P=64,
               max_len=1600, TQ=64, n=32, cu=None, causal=1, scale=0.1, decay=1.0, qd=None, kd=None, ds=None, ws=FAKE,
               ws_len=1 << 40, stream=None)


@pytest.mark.parametrize("status,message,change", [
    (ARG, b"head counts", dict(Hq=7)),
    (ARG, b"head_size", dict(D=64)),
    (ARG, b"max_seqlen_q", dict(n=0)),
    (ARG, b"rows", dict(n=3)),
    (ARG, b"geometry", dict(ps=0)),
    (ARG, b"scores_width", dict(width=-1)),
    (ARG, b"max_seq_len", dict(max_len=-1)),
    (ARG, b"decay", dict(decay=float("inf"))),
    (ARG, b"finite", dict(scale=float("inf"))),
    (ARG, b"NULL", dict(scores=None)),
    (ARG, b"NULL", dict(lse=None)),
    (ARG, b"NULL", dict(lens=None)),
    (ARG, b"16-byte", dict(k=FAKE + 8)),
    (ARG, b"query rows", dict(q=FAKE + 8)),
    (DTYPE, b"query dtype", dict(q_dtype=4)),
    (WORKSPACE, b"workspace", dict(ws_len=64)),
    (WORKSPACE, b"workspace", dict(ws=None)),
])
def test_attention_weights_refuse(status, message, change):
    st = _call("psk_accumulate_attention_weights", list(WEIGHTS), WEIGHTS, **change)
    assert st == status and message in _lib.lib().psk_last_error(), _lib.lib().psk_last_error()


def test_weights_workspace_and_empty_steps():
    lib = _lib.lib()
    assert lib.psk_attention_weights_workspace_bytes(64, 16, 8, 4, 2) == 0  # at most 32 rows share a key
    assert lib.psk_attention_weights_workspace_bytes(64, 17, 8, 4, 2) >= 64 * 8 * 128
    assert lib.psk_attention_weights_workspace_bytes(64, 17, 8, 4, 3) == 0  # already e4m3
    assert lib.psk_attention_weights_workspace_bytes(64, 0, 8, 4, 2) == ARG
    assert lib.psk_attention_weights_workspace_bytes(64, 4, 8, 3, 2) == ARG
    for empty in (dict(width=0), dict(B=0, TQ=0)):
        assert _call("psk_accumulate_attention_weights", list(WEIGHTS), WEIGHTS, **empty) == 0


SELECT = dict(scores=FAKE, ss=STRIDES, width=20000, out=FAKE, os=STRIDES, out_width=20000, lens=FAKE, layers=2, B=2, H=4,
              budget=100, sink=4, recent=8, kept=FAKE, new_lens=FAKE, ws=FAKE, ws_bytes=1 << 40, stream=None)


@pytest.mark.parametrize("status,message,change", [
    (ARG, b"budget", dict(budget=0)),
    (ARG, b"budget", dict(budget=2 ** 31)),
    (ARG, b"do not fit", dict(sink=93)),
    (ARG, b"do not fit", dict(recent=-1)),
    (ARG, b"bad sizes", dict(H=0)),
    (ARG, b"bad sizes", dict(width=2 ** 31)),
    (ARG, b"too many rows", dict(layers=1 << 20, B=1 << 20)),
    (ARG, b"NULL", dict(scores=None)),
    (ARG, b"NULL", dict(kept=None)),
    (WORKSPACE, b"workspace", dict(ws_bytes=100)),
    (WORKSPACE, b"workspace", dict(ws=None)),
])
def test_selection_refuses(status, message, change):
    st = _call("psk_select_tokens", list(SELECT), SELECT, **change)
    assert st == status and message in _lib.lib().psk_last_error(), _lib.lib().psk_last_error()


def test_selection_workspace_and_nothing_to_do():
    lib = _lib.lib()
    assert lib.psk_select_tokens_workspace_bytes(2, 2, 4, 16384, 100) == 0
    assert lib.psk_select_tokens_workspace_bytes(2, 2, 4, 16385, 100) > 0
    assert lib.psk_select_tokens_workspace_bytes(2, 2, 4, 100, 0) == ARG
    assert _call("psk_select_tokens", list(SELECT), SELECT, B=0) == 0


MOVE = dict(c0=FAKE, c1=FAKE, layer=1 << 20, blk=8192, row=512, head=128, head_bytes=128, layers=2, H=4, ps=16, P=64, bt=FAKE,
            bts=10, btw=10, dst=FAKE, dsts=7, dstw=7, kept=FAKE, kept_heads=4, budget=100, B=2, stream=None)


@pytest.mark.parametrize("message,change", [
    (b"65535", dict(layers=65536)),
    (b"65535", dict(B=65536)),
    (b"kept lists", dict(kept_heads=2)),
    (b"bad sizes", dict(btw=0)),
    (b"bad sizes", dict(head_bytes=0)),
    (b"bad sizes", dict(P=0)),
    (b"budget", dict(budget=2 ** 30)),
    (b"NULL", dict(kept=None)),
    (b"NULL", dict(c0=None)),
])
def test_moves_refuse(message, change):
    assert _call("psk_move_kept_tokens", list(MOVE), MOVE, **change) == ARG
    assert message in _lib.lib().psk_last_error(), _lib.lib().psk_last_error()


COMMIT = dict(c0=FAKE, c1=None, layer=1 << 20, blk=8192, row=512, row_bytes=512, layers=2, ps=16, P=64, bt=FAKE, bts=10, btw=10,
              starts=FAKE, path=FAKE, path_stride=6, path_width=6, path_lens=FAKE, B=2, stream=None)


@pytest.mark.parametrize("message,change", [
    (b"at most 256", dict(path_width=257)),
    (b"65535", dict(B=65536)),
    (b"bad sizes", dict(row_bytes=0)),
    (b"bad sizes", dict(ps=0)),
    (b"NULL", dict(starts=None)),
    (b"NULL", dict(bt=None)),
])
def test_commits_refuse(message, change):
    assert _call("psk_commit_draft_tokens", list(COMMIT), COMMIT, **change) == ARG
    assert message in _lib.lib().psk_last_error(), _lib.lib().psk_last_error()


def test_commits_of_nothing():
    for empty in (dict(B=0), dict(layers=0), dict(path_width=0)):
        assert _call("psk_commit_draft_tokens", list(COMMIT), COMMIT, **empty) == 0


def test_tensors_on_the_host_are_refused():
    t = torch.zeros(2, 4, 16, 4, 128, dtype=torch.float8_e4m3fn)
    i = torch.zeros(2, 4, dtype=torch.int32)
    with pytest.raises(AssertionError, match="GPU"):
        cache_ops.evict_tokens([t], torch.zeros(2, 2, 4, 64), i, i[:, 0].contiguous(), i + 1, 16)
    with pytest.raises(AssertionError, match="GPU"):
        cache_ops.commit_draft_tokens([t], i, i[:, 0].contiguous(), i, i[:, 0].contiguous())
    with pytest.raises(AssertionError, match="q must be"):
        attention.paged_tree_attention(torch.zeros(2, 4, 128), t[0], t[0], i, i[:, 0].contiguous(),
                                       torch.zeros(2, 1, dtype=torch.int64), None, 1)
    with pytest.raises(AssertionError, match="q must be"):
        attention.accumulate_attention_weights(torch.zeros(2, 4, 64), torch.zeros(2, 4, 128), t[0], torch.zeros(4, 2), i,
                                               i[:, 0].contiguous())


def test_a_broadcast_is_not_written():
    assert _lib.distinct(torch.zeros(3, 4)) and _lib.distinct(torch.zeros(1, 4).expand(1, 4)[:, ::2])
    assert _lib.distinct(torch.zeros(4).expand(1, 4)) and not _lib.distinct(torch.zeros(4).expand(2, 4))


def test_tensors_whose_elements_share_a_place():
    t = torch.zeros(4000)
    at = lambda shape, strides, first=0: torch.as_strided(t, shape, strides, first)  # noqa: E731
    for shape, strides in (((3, 4), (4, 1)), ((3, 4), (9, 1)), ((3, 4), (1, 3)), ((2, 3, 4), (4, 8, 1)), ((2, 3), (3, 2)),
                           ((2, 2, 3), (3, 9, 1)), ((2, 2, 2), (5, 3, 1)), ((0, 4), (1, 1)), ((1, 4), (0, 1)), ((5,), (1,)),
                           ((), ()), ((4, 1), (1, 7))):
        x = at(shape, strides)
        seen = (torch.arange(4000).as_strided(shape, strides)).reshape(-1).tolist()
        assert _lib.distinct(x) and len(set(seen)) == len(seen), (shape, strides)
    for shape, strides in (((3, 4), (3, 1)), ((3, 4), (0, 1)), ((2, 3, 4), (2, 8, 1)), ((2, 2, 2), (3, 2, 1)), ((4, 4), (1, 1)),
                           ((3, 3), (2, 2))):
        assert not _lib.distinct(at(shape, strides)), (shape, strides)
    # rows counted wider than they are
    assert _lib.distinct(at((3, 4), (9, 1)), 9) and not _lib.distinct(at((3, 4), (9, 1)), 10)
    assert _lib.distinct(at((1, 4), (4, 1)), 100) and not _lib.distinct(at((3, 4), (4, 1)), 5)


def test_tensors_that_share_elements():
    t = torch.zeros(2, 3, 2, 100)
    for a, b in ((t, t), (t, t[..., 5:]), (t[..., :60], t[..., 59:]), (t[:1], t), (t[:, 1:], t[:, :2]),
                 (t.view(-1)[:50], t.view(-1)[49:52]), (t[..., ::2], t[..., 2:3])):
        assert _lib.overlap(a, b) and _lib.overlap(b, a)
    for a, b in ((t, t.clone()), (t[..., :50], t[..., 50:]), (t[:, :1], t[:, 1:]), (t[:, ::2], t[:, 1:2]), (t[..., ::2], t[..., 1::2]),
                 (t[:, :, 0], t[:, :, 1]), (t[:0], t), (t.view(-1)[:50], t.view(-1)[50:])):
        assert not _lib.overlap(a, b) and not _lib.overlap(b, a)
