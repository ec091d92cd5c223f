"""What the decoder operators say of sizes, from the host alone."""
import ctypes as C

import pytest
import torch

import nnr_amd
from decode_ref import nbits_graph
from nnr_amd import _lib

TYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def workspace(cache, t, batch, seq, heads, pages, prefix):
    """What the C function says for a type."""
    a = _lib.KvAttentionDesc(dtype=TYPES[t], batch=batch, seq=seq, q_heads=heads, max_pages=pages, prefix_len=prefix)
    n = C.c_size_t()
    assert _lib.lib().nnrh_kv_attention_workspace(C.byref(cache.desc), C.byref(a), C.byref(n)) == 0
    return n.value


# batch, seq, heads, pages a sequence, prefix
SHAPES = [(32, 1, 32, 8, 4096), (8, 64, 32, 64, 0), (128, 1, 32, 5, 32768), (1, 1024, 32, 128, 0), (1, 1, 32, 4, 0),
          (3, 3, 16, 20, 600), (64, 1, 8, 100, 0)]


@pytest.mark.parametrize("shape", SHAPES)
def test_attention_workspace_by_type(shape):
    """A type's own size where it is named, enough for any type where it is not."""
    cache = nnr_amd.KVCache(1, 8, 128, page_size=64, device="cpu")
    need = {t: workspace(cache, t, *shape) for t in TYPES}
    for t in TYPES:
        assert cache.attention_workspace(*shape, dtype=t) == need[t]
    assert cache.attention_workspace(*shape) == max(need.values())


def test_attention_workspace_differs_by_type():
    """(the shapes above tell the types apart)"""
    cache = nnr_amd.KVCache(1, 8, 128, page_size=64, device="cpu")
    sizes = [[workspace(cache, t, *s) for t in TYPES] for s in SHAPES]
    assert any(f32 < f16 for f32, f16, _ in sizes) and all(f16 == bf16 for _, f16, bf16 in sizes)
    with pytest.raises(TypeError):
        cache.attention_workspace(1, 1, 8, 4, dtype=torch.float64)


BIG = 2 ** 32


def test_whole_numbers_past_32_bits():
    """None is taken for its remainder."""
    for kw in (dict(num_pages=BIG + 4), dict(page_size=BIG + 64), dict(kv_heads=BIG + 8), dict(head_dim=BIG + 128), dict(bits=BIG + 8)):
        with pytest.raises(ValueError, match="32 bits"):
            nnr_amd.KVCache(**{**dict(num_pages=1, kv_heads=8, head_dim=128, page_size=64, bits=8, device="cpu"), **kw})
    b = torch.zeros((1, 1, 1), dtype=torch.uint8).expand(1, (BIG + 64) // 32, 16)
    for k, block in ((BIG + 64, 32), (64, BIG + 32), (64 - BIG, 32)):
        with pytest.raises(ValueError, match="32 bits"):
            nnr_amd.MatMulNBits(b, torch.zeros(1, 1), k, block)


def test_calls_past_32_bits():
    cache = nnr_amd.KVCache(1, 1, 64, page_size=4096, device="cpu")
    one = torch.zeros((1, 1, 1, 64))
    many = one.expand(1, BIG + 1, 1, 64)
    table, lens = torch.zeros((1, 1), dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    pt = torch.zeros(BIG // 4096 + 1, dtype=torch.int32)
    for call in (lambda: cache.write(many, many, table, lens), lambda: cache.attention(many, table, lens, y=many.detach()),
                 lambda: cache.attention(one, table, lens, prefix_table=pt, prefix_len=BIG),
                 lambda: cache.attention(one, table, lens, prefix_table=pt, prefix_len=-BIG)):
        with pytest.raises(ValueError, match="32 bits"):
            call()
    for args in ((BIG + 1, 1, 1, 1), (1, BIG + 1, 1, 1), (1, 1, BIG + 1, 1), (1, 1, 1, BIG + 1), (1, 1, 1, 1, BIG)):
        with pytest.raises(ValueError, match="32 bits"):
            cache.attention_workspace(*args)


@pytest.mark.parametrize("kw", [dict(attrs=dict(K=BIG + 70)), dict(attrs=dict(N=BIG + 24)), dict(shape=(2 ** 20 + 1, 70)),
                                dict(shape=(2 ** 26, 2 ** 6, 70)), dict(attrs=dict(bits=BIG + 4))])
def test_nbits_node_past_its_range(kw):
    from nnr_amd.graph import Session
    with pytest.raises(RuntimeError):
        Session(nbits_graph(**kw), device=False)


@pytest.mark.parametrize("ins", [["x"], ["x", "b"], ["x", "", "s"], ["x", "b", ""]])
def test_nbits_node_without_its_inputs(ins):
    from nnr_amd.graph import Session
    g = nbits_graph()
    node = g.nodes[-1]
    node.inputs[:] = ins
    with pytest.raises(RuntimeError, match="MatMulNBits"):
        Session(g, device=False)


MEM = [0x100000000 * (i + 1) for i in range(8)]


def test_results_over_tables():
    """Tables and lengths are read while a call writes: none may lie in its results."""
    L, inv = _lib.lib(), _lib.NNRH_ERR_INVALID
    c = _lib.KvCacheDesc(4, 64, 2, 128, 8)

    def tokens(table, lens):
        return _lib.KvTokens(dtype=_lib.F16, batch=2, seq=3, batch_stride=768, token_stride=256, page_table_dev=table, max_pages=2,
                             seq_lens_dev=lens)

    def attention(table, lens, prefix):
        return _lib.KvAttentionDesc(dtype=_lib.F16, batch=2, seq=1, q_heads=8, q_batch_stride=1024, q_token_stride=1024, scale=0.1,
                                    page_table_dev=table, max_pages=2, seq_lens_dev=lens, prefix_table_dev=prefix, prefix_len=100)
    last = 2 * 3 * 256 * 2 - 4   # of k's or v's extent
    for at in (MEM[1], MEM[1] + last, MEM[2] + 16):
        for table, lens in ((at, MEM[4]), (MEM[3], at)):
            assert L.nnrh_kv_cache_read(C.byref(c), MEM[0], C.byref(tokens(table, lens)), MEM[1], MEM[2], None) == inv
    for table, lens in ((MEM[0] + 64, MEM[4]), (MEM[3], MEM[0] + 64)):
        assert L.nnrh_kv_cache_write(C.byref(c), MEM[0], C.byref(tokens(table, lens)), MEM[1], MEM[2], None) == inv
    for at in (MEM[2], MEM[2] + 4092, MEM[6] + 256):
        for tables in ((at, MEM[4], MEM[5]), (MEM[3], at, MEM[5]), (MEM[3], MEM[4], at)):
            assert L.nnrh_kv_attention(C.byref(c), MEM[0], C.byref(attention(*tables)), MEM[1], MEM[2], MEM[6], None) == inv


@pytest.mark.parametrize("kw,rc", [
    (dict(num_pages=2 ** 31 - 1, page_size=4096, kv_heads=32767, head_dim=256, bits=8), _lib.NNRH_ERR_UNSUPPORTED),
    (dict(num_pages=2 ** 30, page_size=4096, kv_heads=16384, head_dim=128, bits=4), _lib.NNRH_ERR_UNSUPPORTED),
    (dict(num_pages=2 ** 31 - 1, page_size=32, kv_heads=8, head_dim=128, bits=8), 0)])
def test_cache_bytes_past_64_bits(kw, rc):
    """A cache larger than any memory has no size, and no page of it is taken for one."""
    c, n = _lib.KvCacheDesc(**kw), C.c_size_t(7)
    assert _lib.lib().nnrh_kv_cache_bytes(C.byref(c), C.byref(n)) == rc
    groups = 1 if kw["bits"] == 8 else kw["head_dim"] // 32
    each = 2 * kw["kv_heads"] * kw["page_size"] * (kw["head_dim"] * kw["bits"] // 8 + 2 * groups)
    assert n.value == (7 if rc else kw["num_pages"] * each)
