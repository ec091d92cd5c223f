"""What the decoder operators refuse, before anything reaches a GPU (the
addresses are no memory), and their plain forms' own checks."""
import ctypes as C

import numpy as np
import pytest
import torch

import decode_ref as R
import nnr_amd
from decode_ref import nbits_graph
from nnr_amd import _lib

INVALID, UNSUPPORTED = _lib.NNRH_ERR_INVALID, _lib.NNRH_ERR_UNSUPPORTED
MEM = [0x100000000 * (i + 1) for i in range(8)]


def nbits_desc(**kw):
    d = dict(n=16, k=64, bits=4, block_size=32, dtype=_lib.F32, b=MEM[0], scales=MEM[1])
    d.update(kw)
    return _lib.MatMulNBitsDesc(**d)


@pytest.mark.parametrize("kw,rc", [
    (dict(n=0), INVALID), (dict(k=-1), INVALID), (dict(block_size=48), INVALID), (dict(block_size=0), INVALID),
    (dict(b=None), INVALID), (dict(scales=None), INVALID), (dict(bits=8), UNSUPPORTED),
    (dict(block_size=16), UNSUPPORTED), (dict(dtype=_lib.U8), UNSUPPORTED), (dict(dtype=17), UNSUPPORTED),
    (dict(on_device=1, b=MEM[0] + 2), INVALID), (dict(on_device=1, scales=MEM[1] + 1), INVALID),
    (dict(k=(1 << 22) + 1), UNSUPPORTED), (dict(n=(1 << 31) - 1), UNSUPPORTED)])
def test_nbits_create_refuses(kw, rc):
    h = C.c_void_p(5)
    d = nbits_desc(**kw)
    assert _lib.lib().nnrh_matmul_nbits_create(C.byref(h), C.byref(d)) == rc
    assert h.value is None and b"matmul_nbits" in _lib.lib().nnrh_last_error()


def test_nbits_null():
    L = _lib.lib()
    assert L.nnrh_matmul_nbits_create(None, None) == INVALID
    assert L.nnrh_matmul_nbits_run(None, MEM[0], MEM[1], 1, None) == INVALID
    assert L.nnrh_matmul_nbits_destroy(None) == 0


def cache_desc(**kw):
    d = dict(num_pages=4, page_size=64, kv_heads=2, head_dim=128, bits=8)
    d.update(kw)
    return _lib.KvCacheDesc(**d)


BAD_CACHES = [(dict(page_size=0), INVALID), (dict(kv_heads=0), INVALID), (dict(num_pages=-1), INVALID),
              (dict(head_dim=-64), INVALID), (dict(page_size=16), UNSUPPORTED), (dict(page_size=96), UNSUPPORTED),
              (dict(page_size=8192), UNSUPPORTED), (dict(head_dim=80), UNSUPPORTED), (dict(head_dim=512), UNSUPPORTED),
              (dict(bits=2), UNSUPPORTED), (dict(kv_heads=40000), UNSUPPORTED)]


@pytest.mark.parametrize("kw,rc", BAD_CACHES)
def test_cache_refuses(kw, rc):
    n = C.c_size_t()
    d = cache_desc(**kw)
    assert _lib.lib().nnrh_kv_cache_bytes(C.byref(d), C.byref(n)) == rc


@pytest.mark.parametrize("bits,hd,page,heads", [(8, 64, 32, 1), (8, 256, 128, 3), (4, 128, 64, 8), (4, 96, 4096, 2)])
def test_cache_bytes(bits, hd, page, heads):
    """Codes and bf16 scales, one a token and head at 8 bits, one per 32 elements at 4; past 2^32 too."""
    groups = 1 if bits == 8 else hd // 32
    each = 2 * heads * page * (hd * bits // 8 + 2 * groups)
    for pages in (0, 1, 7, 2_000_000):
        n, d = C.c_size_t(), cache_desc(num_pages=pages, page_size=page, kv_heads=heads, head_dim=hd, bits=bits)
        assert _lib.lib().nnrh_kv_cache_bytes(C.byref(d), C.byref(n)) == 0 and n.value == pages * each


def tokens_desc(**kw):
    d = dict(dtype=_lib.F16, batch=2, seq=3, batch_stride=3 * 256, token_stride=256, page_table_dev=MEM[3],
             max_pages=2, seq_lens_dev=MEM[4])
    d.update(kw)
    return _lib.KvTokens(**d)


BAD_TOKENS = [
    (dict(dtype=_lib.U8), UNSUPPORTED), (dict(batch=-1), INVALID), (dict(seq=-1), INVALID), (dict(max_pages=-1), INVALID),
    (dict(page_table_dev=None), INVALID), (dict(seq_lens_dev=None), INVALID), (dict(page_table_dev=MEM[3] + 2), INVALID),
    (dict(token_stride=257), INVALID), (dict(batch_stride=-8), INVALID), (dict(batch=70000), UNSUPPORTED),
    (dict(max_pages=1 << 25), UNSUPPORTED), (dict(token_stride=1 << 41), UNSUPPORTED)]


@pytest.mark.parametrize("kw,rc", BAD_TOKENS)
def test_cache_calls_refuse(kw, rc):
    L, c, t = _lib.lib(), cache_desc(), tokens_desc(**kw)
    assert L.nnrh_kv_cache_write(C.byref(c), MEM[0], C.byref(t), MEM[1], MEM[2], None) == rc
    assert L.nnrh_kv_cache_read(C.byref(c), MEM[0], C.byref(t), MEM[1], MEM[2], None) == rc


def test_cache_calls_refuse_memory():
    L, c, t = _lib.lib(), cache_desc(), tokens_desc()
    size = C.c_size_t()
    assert L.nnrh_kv_cache_bytes(C.byref(c), C.byref(size)) == 0
    for cache, k, v in ((MEM[0] + 8, MEM[1], MEM[2]), (MEM[0], MEM[1] + 8, MEM[2]), (MEM[0], MEM[1], MEM[2] + 2),
                        (None, MEM[1], MEM[2]), (MEM[0], None, MEM[2]), (MEM[0], MEM[1], None),
                        (MEM[0], MEM[0] + size.value - 16, MEM[2]), (MEM[0], MEM[1], MEM[0] - 16)):
        assert L.nnrh_kv_cache_write(C.byref(c), cache, C.byref(t), k, v, None) == INVALID
        assert L.nnrh_kv_cache_read(C.byref(c), cache, C.byref(t), k, v, None) == INVALID
    # results that lie over each other
    for kw in (dict(token_stride=128), dict(batch_stride=0), dict(batch_stride=256)):
        t = tokens_desc(**kw)
        assert L.nnrh_kv_cache_read(C.byref(c), MEM[0], C.byref(t), MEM[1], MEM[2], None) == INVALID
    t = tokens_desc()
    assert L.nnrh_kv_cache_read(C.byref(c), MEM[0], C.byref(t), MEM[1], MEM[1], None) == INVALID
    # nothing to do is no error
    for kw in (dict(batch=0), dict(seq=0)):
        t = tokens_desc(**kw)
        assert L.nnrh_kv_cache_write(C.byref(c), MEM[0], C.byref(t), None, None, None) == 0


def attention_desc(**kw):
    d = dict(dtype=_lib.F16, batch=2, seq=1, q_heads=8, q_batch_stride=1024, q_token_stride=1024, scale=0.1,
             page_table_dev=MEM[3], max_pages=2, seq_lens_dev=MEM[4], prefix_table_dev=MEM[5], prefix_len=100)
    d.update(kw)
    return _lib.KvAttentionDesc(**d)


@pytest.mark.parametrize("kw,rc", [
    (dict(dtype=_lib.S8), UNSUPPORTED), (dict(q_heads=7), INVALID), (dict(q_heads=0), INVALID),
    (dict(prefix_len=-1), INVALID), (dict(prefix_table_dev=None), INVALID), (dict(prefix_table_dev=MEM[5] + 1), INVALID),
    (dict(page_table_dev=None), INVALID), (dict(seq_lens_dev=None), INVALID), (dict(max_pages=-1), INVALID),
    (dict(q_batch_stride=4), INVALID), (dict(batch=-1), INVALID), (dict(prefix_len=(1 << 30) + 1), UNSUPPORTED),
    (dict(batch=60000, seq=1 << 20), UNSUPPORTED)])
def test_attention_refuses(kw, rc):
    L, c, a = _lib.lib(), cache_desc(), attention_desc(**kw)
    assert L.nnrh_kv_attention(C.byref(c), MEM[0], C.byref(a), MEM[1], MEM[2], MEM[6], None) == rc


@pytest.mark.parametrize("kw,rc", BAD_CACHES)
def test_attention_refuses_caches(kw, rc):
    L, c, a = _lib.lib(), cache_desc(**kw), attention_desc()
    assert L.nnrh_kv_attention(C.byref(c), MEM[0], C.byref(a), MEM[1], MEM[2], MEM[6], None) == rc
    assert L.nnrh_kv_attention_workspace(C.byref(c), C.byref(a), C.byref(C.c_size_t())) == rc


def test_attention_refuses_memory():
    L, c, a = _lib.lib(), cache_desc(), attention_desc()
    run = lambda cache, q, y, ws: L.nnrh_kv_attention(C.byref(c), cache, C.byref(a), q, y, ws, None)
    n = C.c_size_t()
    assert L.nnrh_kv_attention_workspace(C.byref(c), C.byref(a), C.byref(n)) == 0 and n.value > 0
    y = 2 * 8 * 128 * 2
    for args in ((MEM[0] + 1, MEM[1], MEM[2], MEM[6]), (None, MEM[1], MEM[2], MEM[6]), (MEM[0], None, MEM[2], MEM[6]),
                 (MEM[0], MEM[1], None, MEM[6]), (MEM[0], MEM[1] + 8, MEM[2], MEM[6]), (MEM[0], MEM[1], MEM[2] + 4, MEM[6]),
                 (MEM[0], MEM[1], MEM[2], None), (MEM[0], MEM[1], MEM[2], MEM[6] + 128),
                 (MEM[0], MEM[1], MEM[1] + 16, MEM[6]), (MEM[0], MEM[1], MEM[1] - y + 16, MEM[6]),
                 (MEM[0], MEM[1], MEM[0], MEM[6]), (MEM[0], MEM[1], MEM[6], MEM[6]), (MEM[0], MEM[6] + 256, MEM[2], MEM[6])):
        assert run(*args) == INVALID
    a = attention_desc(q_batch_stride=2048)      # y over a q that is not dense
    assert run(MEM[0], MEM[1], MEM[1], MEM[6]) == INVALID
    a = attention_desc(batch=0)
    assert run(MEM[0], None, None, None) == 0


@pytest.mark.parametrize("kw", [dict(n=(1 << 26) + 1), dict(n=1 << 25, k=4096)])
def test_nbits_create_refuses_sizes(kw):
    """Launches that would pass 2^32 threads: from shapes alone, before any pointer is read"""
    d = dict(n=16, k=64, bits=4, block_size=32, dtype=_lib.F16, on_device=1, b=MEM[0], scales=MEM[1])
    h = C.c_void_p()
    assert _lib.lib().nnrh_matmul_nbits_create(C.byref(h), C.byref(_lib.MatMulNBitsDesc(**{**d, **kw}))) == UNSUPPORTED
    assert not h.value


@pytest.mark.parametrize("kw", [dict(seq=(1 << 22) + 1), dict(batch_stride=(1 << 38) + 8)])
def test_calls_refuse_sizes(kw):
    L, c, t = _lib.lib(), cache_desc(), tokens_desc(**kw)
    assert L.nnrh_kv_cache_write(C.byref(c), MEM[0], C.byref(t), MEM[1], MEM[2], None) == UNSUPPORTED
    assert L.nnrh_kv_cache_read(C.byref(c), MEM[0], C.byref(t), MEM[1], MEM[2], None) == UNSUPPORTED


def test_attention_refuses_rows():
    L, c, n = _lib.lib(), cache_desc(kv_heads=1), C.c_size_t()
    for batch, seq, heads, rc in ((64, 4096, 32, 0), (64, 4097, 32, UNSUPPORTED), (1, 1, (1 << 23) + 1, UNSUPPORTED)):
        a = attention_desc(batch=batch, seq=seq, q_heads=heads, q_token_stride=heads * 128, q_batch_stride=seq * heads * 128)
        assert L.nnrh_kv_attention_workspace(C.byref(c), C.byref(a), C.byref(n)) == rc
        if rc:
            assert L.nnrh_kv_attention(C.byref(c), MEM[0], C.byref(a), MEM[1], MEM[2], MEM[6], None) == rc


def test_read_refuses_rows_over_each_other():
    """v's rows may lie between k's, not over them."""
    L, c = _lib.lib(), cache_desc()
    t = tokens_desc(token_stride=1024, batch_stride=4096)
    for at in (-496, -16, 16, 496):
        assert L.nnrh_kv_cache_read(C.byref(c), MEM[0], C.byref(t), MEM[1] + 512, MEM[1] + 512 + at, None) == INVALID


def test_attention_refuses_a_workspace_in_the_cache():
    L, c, a = _lib.lib(), cache_desc(), attention_desc()
    assert L.nnrh_kv_attention(C.byref(c), MEM[0], C.byref(a), MEM[1], MEM[2], MEM[0] + 256, None) == INVALID


def test_python_refuses_types():
    with pytest.raises(TypeError):
        nnr_amd.MatMulNBits(np.zeros((4, 2, 16), np.uint8), torch.zeros(4, 2, dtype=torch.float64), 64, 32)
    with pytest.raises(ValueError):
        nnr_amd.MatMulNBits(np.zeros((4, 2, 15), np.uint8), torch.zeros(4, 2), 64, 32)
    with pytest.raises(nnr_amd.NnrHipError):
        nnr_amd.KVCache(4, 2, 80)


def test_plain_quantizer():
    """The plain form itself on a group worked out by hand"""
    x = torch.tensor([127.0, -63.5, 0.4, 1.5, float("inf"), float("nan"), -float("inf"), 2.5] + [0.0] * 56)
    v, c, s = R.quantize(x, 8)
    assert s.item() == 1.0 and c[:8].tolist() == [127, -64, 0, 2, 127, 0, -127, 2]
    v, c, s = R.quantize(x * 7 / 127, 4)
    assert c[:2].tolist() == [7, -4]
    assert s[1].item() == 0.0


def test_nbits_node_shapes():
    from nnr_amd.graph import Session
    s = Session(nbits_graph(), device=False)
    assert s.tensor_info("y")[2] == (2, 3, 24) and [p["op"] for p in s.plan()] == ["MatMulNBits"]


@pytest.mark.parametrize("kw", [dict(shape=(2, 3, 71)), dict(attrs=dict(K=0)), dict(attrs=dict(N=-1)), dict(dt=np.int8)])
def test_nbits_node_refuses(kw):
    from nnr_amd.graph import Session
    with pytest.raises(RuntimeError):
        Session(nbits_graph(**kw), device=False)
