"""What the operators around a decoder's cache refuse, before anything reaches a GPU
(the addresses are no memory), and the tables' frequencies."""
import ctypes as C

import numpy as np
import pytest
import torch

import nnr_amd
import serving_ref as R
from nnr_amd import _lib
from test_decode_cpu import BAD_CACHES, MEM, attention_desc, cache_desc

INVALID, UNSUPPORTED = _lib.NNRH_ERR_INVALID, _lib.NNRH_ERR_UNSUPPORTED


# ---------------------------------------------------------------------------
# rotary positions

def rotary_desc(**kw):
    d = dict(dtype=_lib.F16, batch=2, seq=3, q_heads=4, k_heads=2, head_dim=64, rotary_dim=32, positions_dev=MEM[4],
             table_dev=MEM[5], max_positions=100)
    for t, h in (("q", 4), ("k", 2), ("qy", 4), ("ky", 2)):
        d[f"{t}_token_stride"], d[f"{t}_batch_stride"] = h * 64, 3 * h * 64
    d.update(kw)
    return _lib.RotaryDesc(**d)


def rotary(d, q=MEM[0], k=MEM[1], qy=MEM[2], ky=MEM[3]):
    return _lib.lib().nnrh_rotary(C.byref(d), q, k, qy, ky, None)


@pytest.mark.parametrize("kw,rc", [
    (dict(dtype=_lib.U8), UNSUPPORTED), (dict(batch=-1), INVALID), (dict(seq=-1), INVALID), (dict(q_heads=-1), INVALID),
    (dict(head_dim=0), INVALID), (dict(rotary_dim=33), INVALID), (dict(rotary_dim=66), INVALID), (dict(rotary_dim=-2), INVALID),
    (dict(max_positions=0), INVALID), (dict(positions_dev=None), INVALID), (dict(table_dev=None), INVALID),
    (dict(positions_dev=MEM[4] + 2), INVALID), (dict(table_dev=MEM[5] + 4), INVALID), (dict(q_token_stride=-256), INVALID),
    (dict(qy_token_stride=255), INVALID), (dict(ky_batch_stride=127), INVALID), (dict(k_batch_stride=1 << 39), UNSUPPORTED),
    (dict(batch=1 << 14, seq=1 << 14), UNSUPPORTED), (dict(q_heads=1 << 21), UNSUPPORTED)])
def test_rotary_refuses(kw, rc):
    assert rotary(rotary_desc(**kw)) == rc and b"rotary" in _lib.lib().nnrh_last_error()


def test_rotary_refuses_memory():
    d = rotary_desc()
    size, kv = 2 * 3 * 4 * 64 * 2, 2 * 3 * 2 * 64 * 2
    for kw in (dict(q=None), dict(k=None), dict(qy=None), dict(ky=None), dict(q=MEM[0] + 1), dict(ky=MEM[3] + 1),
               dict(qy=MEM[0] + 16), dict(qy=MEM[0] - size + 2), dict(qy=MEM[1]), dict(ky=MEM[2] + 64), dict(ky=MEM[0]),
               dict(qy=MEM[4]), dict(ky=MEM[4] - kv + 2), dict(qy=MEM[5] + 100 * 32 * 4 - 16)):
        assert rotary(d, **kw) == INVALID, kw
    # in place at other strides
    assert rotary(rotary_desc(qy_token_stride=512, qy_batch_stride=1536), qy=MEM[0]) == INVALID
    # rows of q and k side by side in one tensor, in place, but k's a part of a row too early
    side = dict(q_token_stride=384, k_token_stride=384, qy_token_stride=384, ky_token_stride=384, q_batch_stride=1152,
                k_batch_stride=1152, qy_batch_stride=1152, ky_batch_stride=1152)
    at = MEM[0] + 2 * 256
    assert rotary(rotary_desc(**side), k=at - 16, ky=at - 16, qy=MEM[0]) == INVALID
    # (uneven steps: rows may meet, so it is taken that they do)
    uneven = {**side, **{f"{t}_batch_stride": 1160 for t in ("q", "k", "qy", "ky")}}
    assert rotary(rotary_desc(**uneven), k=at, ky=at, qy=MEM[0]) == INVALID
    # nothing to do is no error
    for kw in (dict(batch=0), dict(seq=0), dict(q_heads=0, k_heads=0)):
        assert rotary(rotary_desc(**kw), None, None, None, None) == 0
    assert _lib.lib().nnrh_rotary(None, MEM[0], MEM[1], MEM[2], MEM[3], None) == INVALID


@pytest.mark.parametrize("scaling,factor", [(None, 1.0), ("none", 1.0), ("linear", 4.0), ("ntk", 8.0), ("yarn", 8.0), ("yarn", 1.0)])
@pytest.mark.parametrize("r", [4, 40, 128])
def test_frequencies(scaling, factor, r):
    f, m = nnr_amd.rotary_frequencies(r, 10000.0, scaling, factor, 4096)
    want, wm = R.frequencies(r, 10000.0, scaling or "none", factor, 4096)
    assert np.abs(f / want - 1).max() < 1e-14 and abs(m - wm) < 1e-14


def test_python_refuses_host_memory():
    """Tensors that no kernel can read"""
    t = torch.zeros((4, 2, 64))
    starts, one = torch.tensor([0, 4], dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    cache = nnr_amd.KVCache(2, 2, 64, page_size=32, device="cpu")
    calls = (lambda: nnr_amd.prompt_attention(t, t, t, starts),
             lambda: nnr_amd.RotaryEmbedding(64, 10, device="cpu"),
             lambda: nnr_amd.copy_pages(cache, one, one),
             lambda: nnr_amd.move_tokens([cache], one[None], one[None], one[None]),
             lambda: cache.attention(t[None], one[None], one, tree=torch.ones((4, 4), dtype=torch.bool)))
    for call in calls:
        with pytest.raises(ValueError, match="not on a GPU"):
            call()


def test_frequencies_refuse():
    for kw in (dict(scaling="cubic"), dict(factor=0.0), dict(base=-1.0), dict(scaling="yarn")):
        with pytest.raises(ValueError):
            nnr_amd.rotary_frequencies(64, **kw)
    for kw in (dict(rotary_dim=63), dict(rotary_dim=66), dict(max_positions=0), dict(frequencies=[1.0]),
               dict(scaling="linear", factor=0.0)):
        with pytest.raises(ValueError):
            nnr_amd.RotaryEmbedding(**{**dict(head_dim=64, max_positions=10, device="cpu"), **kw})


# ---------------------------------------------------------------------------
# attention of prompts

def prompt_desc(**kw):
    d = dict(dtype=_lib.F16, tokens=100, seqs=2, q_heads=8, kv_heads=2, head_dim=64, q_stride=512, k_stride=128, v_stride=128,
             scale=0.1, causal=1, starts_dev=MEM[4])
    d.update(kw)
    return _lib.PromptAttentionDesc(**d)


def prompt(d, q=MEM[0], k=MEM[1], v=MEM[2], y=MEM[3]):
    return _lib.lib().nnrh_prompt_attention(C.byref(d), q, k, v, y, None)


@pytest.mark.parametrize("kw,rc", [
    (dict(dtype=_lib.S8), UNSUPPORTED), (dict(tokens=-1), INVALID), (dict(seqs=-1), INVALID), (dict(q_heads=7), INVALID),
    (dict(q_heads=0), INVALID), (dict(kv_heads=0), INVALID), (dict(head_dim=80), UNSUPPORTED), (dict(head_dim=0), UNSUPPORTED),
    (dict(starts_dev=None), INVALID), (dict(starts_dev=MEM[4] + 2), INVALID), (dict(q_stride=-512), INVALID),
    (dict(k_stride=132), INVALID), (dict(v_stride=(1 << 22) + 8), UNSUPPORTED), (dict(tokens=1 << 28), UNSUPPORTED),
    (dict(seqs=1 << 23), UNSUPPORTED), (dict(kv_heads=40000, q_heads=40000), UNSUPPORTED)])
def test_prompt_refuses(kw, rc):
    assert prompt(prompt_desc(**kw)) == rc and b"prompt_attention" in _lib.lib().nnrh_last_error()


def test_prompt_refuses_memory():
    d = prompt_desc()
    size, kv = 100 * 512 * 2, 100 * 128 * 2
    for kw in (dict(q=None), dict(k=None), dict(v=None), dict(y=None), dict(q=MEM[0] + 8), dict(k=MEM[1] + 2), dict(v=MEM[2] + 4),
               dict(y=MEM[3] + 8), dict(y=MEM[0] + 16), dict(y=MEM[0] - size + 16), dict(y=MEM[1] + kv - 16), dict(y=MEM[2]),
               dict(y=MEM[4]), dict(y=MEM[4] - size + 16)):
        assert prompt(d, **kw) == INVALID, kw
    assert prompt(prompt_desc(q_stride=520), y=MEM[0]) == INVALID       # in place of a q that is not dense
    for kw in (dict(tokens=0), dict(seqs=0)):
        assert prompt(prompt_desc(**kw), None, None, None, None) == 0
    assert _lib.lib().nnrh_prompt_attention(None, MEM[0], MEM[1], MEM[2], MEM[3], None) == INVALID


# ---------------------------------------------------------------------------
# trees of drafts

def tree(a, at=MEM[7], stride=9, cache=None, y=MEM[2], ws=MEM[6]):
    c = cache or cache_desc()
    return _lib.lib().nnrh_kv_tree_attention(C.byref(c), MEM[0], C.byref(a), at, stride, MEM[1], y, ws, None)


def tree_workspace(a, c=None):
    n = C.c_size_t()
    return _lib.lib().nnrh_kv_tree_attention_workspace(C.byref(c or cache_desc()), C.byref(a), C.byref(n)), n.value


def test_tree_workspace():
    """Partial results of rows x (elements + 2) floats, once a part; none where one block sees all of a sequence"""
    L, c, n = _lib.lib(), cache_desc(), C.c_size_t()
    for seq, pages in ((1, 2), (3, 2), (64, 2), (17, 512), (4096, 512), (64, 0)):
        a = attention_desc(seq=seq, q_batch_stride=seq * 1024, q_token_stride=1024, max_pages=pages)
        rc, size = tree_workspace(a)
        rows = a.batch * seq * a.q_heads
        assert rc == 0 and size % (rows * (c.head_dim * 4 + 8)) == 0
        assert size == 0 or size >= 2 * rows * (c.head_dim * 4 + 8)
    assert tree_workspace(attention_desc(seq=0)) == (0, 0) and tree_workspace(attention_desc(batch=0)) == (0, 0)
    for kw, rc in ((dict(seq=4097), UNSUPPORTED), (dict(max_pages=-1), INVALID), (dict(max_pages=1 << 30), INVALID),
                   (dict(dtype=_lib.S8), UNSUPPORTED), (dict(q_heads=7), INVALID)):
        assert tree_workspace(attention_desc(**{**dict(seq=3), **kw}))[0] == rc, kw
    a = attention_desc(seq=3)
    assert L.nnrh_kv_tree_attention_workspace(C.byref(c), C.byref(a), None) == INVALID
    assert L.nnrh_kv_tree_attention_workspace(None, C.byref(a), C.byref(n)) == INVALID
    assert L.nnrh_kv_tree_attention_workspace(C.byref(c), None, C.byref(n)) == INVALID


@pytest.mark.parametrize("kw,rc", [
    (dict(dtype=_lib.S8), UNSUPPORTED), (dict(q_heads=7), INVALID), (dict(prefix_len=-1), INVALID), (dict(batch=-1), INVALID),
    (dict(seq=-1), INVALID), (dict(page_table_dev=None), INVALID), (dict(seq=4097, q_token_stride=1024), UNSUPPORTED)])
def test_tree_refuses(kw, rc):
    assert tree(attention_desc(**{**dict(seq=3), **kw}), stride=0) == rc


@pytest.mark.parametrize("kw,rc", BAD_CACHES)
def test_tree_refuses_caches(kw, rc):
    assert tree(attention_desc(seq=3, q_batch_stride=4096), cache=cache_desc(**kw)) == rc
    assert tree_workspace(attention_desc(seq=3, q_batch_stride=4096), cache_desc(**kw))[0] == rc


def test_tree_refuses_memory():
    a = attention_desc(seq=3)
    for kw in (dict(at=None), dict(stride=8), dict(stride=-9), dict(stride=1), dict(at=MEM[2]), dict(at=MEM[2] - 17),
               dict(at=MEM[6] + 5), dict(y=None), dict(ws=None)):
        assert tree(a, **kw) == INVALID, kw
    assert tree(a, stride=(1 << 38) + 1) == UNSUPPORTED
    for kw in (dict(batch=0), dict(seq=0)):
        assert tree(attention_desc(**kw), at=None) == 0
    c = cache_desc()
    assert _lib.lib().nnrh_kv_tree_attention(C.byref(c), MEM[0], None, MEM[7], 9, MEM[1], MEM[2], MEM[6], None) == INVALID


# ---------------------------------------------------------------------------
# pages and tokens moved

def layers(*at):
    return (C.c_void_p * len(at))(*at)


def copy(c=None, caches=(MEM[0],), n=None, src=MEM[1], dst=MEM[2], count=3):
    c = c or cache_desc()
    return _lib.lib().nnrh_kv_copy_pages(C.byref(c), layers(*caches), len(caches) if n is None else n, src, dst, count, None)


def moves(**kw):
    d = dict(batch=2, count=3, page_table_dev=MEM[1], max_pages=2, source_dev=MEM[2], destination_dev=MEM[3])
    d.update(kw)
    return _lib.KvMoves(**d)


def move(m, c=None, caches=(MEM[0],), n=None):
    c = c or cache_desc()
    return _lib.lib().nnrh_kv_move_tokens(C.byref(c), layers(*caches), len(caches) if n is None else n, C.byref(m), None)


@pytest.mark.parametrize("kw,rc", BAD_CACHES)
def test_moves_refuse_caches(kw, rc):
    assert copy(cache_desc(**kw)) == rc and move(moves(), cache_desc(**kw)) == rc


def test_moves_refuse_memory():
    size = C.c_size_t()
    assert _lib.lib().nnrh_kv_cache_bytes(C.byref(cache_desc()), C.byref(size)) == 0
    for caches in ((None,), (MEM[0] + 8,), (MEM[0], MEM[0]), (MEM[5], MEM[0], MEM[0] + size.value - 16)):
        assert copy(caches=caches) == INVALID and move(moves(), caches=caches) == INVALID
    assert copy(n=-1) == INVALID and move(moves(), n=-1) == INVALID
    assert copy(n=1025, caches=(MEM[0],) * 1025) == UNSUPPORTED
    for kw in (dict(src=None), dict(dst=None), dict(src=MEM[1] + 2), dict(dst=MEM[2] + 1), dict(count=-1), dict(src=MEM[0]),
               dict(dst=MEM[0] + size.value - 4)):
        assert copy(**kw) == INVALID, kw
    L = _lib.lib()
    c = cache_desc()
    assert L.nnrh_kv_copy_pages(C.byref(c), None, 1, MEM[1], MEM[2], 3, None) == INVALID
    assert L.nnrh_kv_move_tokens(C.byref(c), None, 1, C.byref(moves()), None) == INVALID
    assert L.nnrh_kv_move_tokens(C.byref(c), layers(MEM[0]), 1, None, None) == INVALID
    assert copy(count=0, src=None, dst=None) == 0 and copy(caches=(), src=None) == 0


@pytest.mark.parametrize("kw,rc", [
    (dict(batch=-1), INVALID), (dict(count=-1), INVALID), (dict(max_pages=-1), INVALID), (dict(page_table_dev=None), INVALID),
    (dict(source_dev=None), INVALID), (dict(destination_dev=None), INVALID), (dict(source_dev=MEM[2] + 1), INVALID),
    (dict(page_table_dev=MEM[0]), INVALID), (dict(source_dev=MEM[0] + 64), INVALID), (dict(destination_dev=MEM[0]), INVALID),
    (dict(batch=65536), UNSUPPORTED), (dict(count=129), UNSUPPORTED), (dict(max_pages=1 << 25), UNSUPPORTED),
    (dict(batch=0), 0), (dict(count=0), 0), (dict(max_pages=0), 0)])
def test_move_refuses(kw, rc):
    assert move(moves(**kw)) == rc


def test_move_refuses_threads():
    assert move(moves(batch=65535), cache_desc(kv_heads=100)) == UNSUPPORTED
