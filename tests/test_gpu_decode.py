"""Operators of a decoder's step against float64: products with 4-bit weights,
the quantized key/value cache and the attention that reads it."""
import ctypes as C

import numpy as np
import pytest
import torch

import decode_ref as R
import nnr_amd
from nnr_amd import _lib

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def f64(t):
    return t.detach().cpu().double().numpy()


# ---------------------------------------------------------------------------
# 4-bit weights

def weights(seed, n, k, block, t, zp, bias):
    rng = np.random.default_rng(seed)
    nb = -(-k // block)
    b = rng.integers(0, 256, (n, nb, block // 2), dtype=np.uint8)
    s = torch.from_numpy(rng.uniform(0.01, 0.1, (n, nb))).to(t)
    z = rng.integers(0, 256, (n, (nb + 1) // 2), dtype=np.uint8) if zp else None
    c = torch.from_numpy(rng.standard_normal(n)).to(t) if bias else None
    return b, s, z, c


def check_nbits(dev, m, n, k, block, t, zp, bias, a=None):
    b, s, z, c = weights(m + n + k, n, k, block, t, zp, bias)
    if a is None:
        a = torch.from_numpy(np.random.default_rng(k).standard_normal((m, k))).to(t)
    op = nnr_amd.MatMulNBits(b, s, k, block, zero_points=z, bias=c)
    y = f64(op(a.to(dev)))
    ref, mag = R.nbits(f64(a), b, f64(s), k, block, z, None if c is None else f64(c))
    tol = R.nbits_tol(ref, mag, k, t)
    assert R.close(y, ref, tol, t).all(), (np.abs(y - ref) / tol).max()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,n,k,block,zp,bias", [
    (1, 1, 1, 32, False, False), (1, 16, 32, 32, True, True), (1, 17, 33, 32, True, False), (2, 64, 128, 64, False, True),
    (1, 1024, 1024, 32, False, False), (1, 100, 4096, 128, True, True), (5, 65, 130, 32, True, True),
    (15, 48, 384, 256, True, False), (16, 333, 1000, 64, False, True), (17, 80, 257, 32, True, True),
    (31, 96, 512, 128, False, False), (33, 130, 640, 32, True, True), (64, 256, 2048, 32, True, False),
    (65, 67, 96, 512, False, True), (130, 200, 1500, 64, True, True), (300, 512, 1024, 32, False, False),
    (1, 16500, 160, 32, True, True), (3, 20, 8192, 4096, True, False), (2, 16400, 320, 64, True, True),
    # grids of blocks that share rows: few column tiles a wave, many, one piece of K, uneven rounds
    (130, 12300, 200, 32, True, True), (193, 8200, 1160, 128, False, True), (300, 16500, 160, 64, True, False),
    (260, 16400, 64, 32, False, True), (1030, 4200, 640, 256, True, True), (513, 8250, 1096, 32, True, False)])
def test_nbits(dev, t, m, n, k, block, zp, bias):
    check_nbits(dev, m, n, k, block, t, zp, bias)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m", [1, 20, 70, 200])
def test_nbits_unaligned_rows(dev, t, m):
    """a at an address of one element past a 16-byte boundary"""
    n, k, block = 40, 256, 64
    b, s, z, c = weights(7, n, k, block, t, True, True)
    op = nnr_amd.MatMulNBits(b, s, k, block, zero_points=z, bias=c)
    buf = torch.randn(m * k + 1, generator=torch.Generator().manual_seed(1)).to(t).to(dev)
    a = buf[1:].view(m, k)
    y = f64(op(a))
    ref, mag = R.nbits(f64(a), b, f64(s), k, block, z, f64(c))
    assert (np.abs(y - ref) <= R.nbits_tol(ref, mag, k, t)).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m", [7, 90])
def test_nbits_rows_do_not_mix(dev, t, m):
    """A row with an infinity or a NaN is that row's alone; an infinity keeps its sign."""
    n, k, block = 50, 320, 32
    b, s, z, c = weights(3, n, k, block, t, False, False)
    b[:, 0, 0] = 0x9b      # k 0: q 11 (a weight above 0), k 1: q 9
    op = nnr_amd.MatMulNBits(b, s, k, block)
    a = torch.randn(m, k, generator=torch.Generator().manual_seed(2)).to(t)
    clean = op(a.to(dev))
    bad = a.clone()
    bad[2, 0], bad[4, 5] = float("inf"), float("nan")
    y = op(bad.to(dev))
    assert torch.isnan(y[4]).all() and (y[2] == float("inf")).all()
    rows = [i for i in range(m) if i not in (2, 4)]
    assert torch.equal(y[rows], clean[rows])


@pytest.mark.parametrize("t", TYPES)
def test_nbits_extreme_activations(dev, t):
    """The largest and smallest numbers of a type, whose sums fp32 still holds."""
    n, k, block = 32, 64, 32
    top = {torch.float32: 1e36, torch.float16: 65504.0, torch.bfloat16: 1e36}[t]
    a = torch.full((4, k), top).to(t)
    a[1] = torch.finfo(t).tiny
    a[2, ::2] *= -1
    a[3, 1:] = 1e-4
    check_nbits(dev, 4, n, k, block, t, True, False, a=a)


@pytest.mark.parametrize("t", TYPES)
def test_nbits_weights_on_the_device(dev, t):
    """The same handle from host and device memory, at odd addresses too"""
    b, s, z, c = weights(11, 70, 300, 64, t, True, True)
    x = torch.randn((9, 300), generator=torch.Generator().manual_seed(4)).to(t).to(dev)
    ref = nnr_amd.MatMulNBits(b, s, 300, 64, zero_points=z, bias=c)(x)
    odd = torch.empty(b.size + 1, dtype=torch.uint8, device=dev)[1:].reshape(b.shape)
    odd.copy_(torch.from_numpy(b))
    for w in (torch.from_numpy(b).to(dev), odd):
        op = nnr_amd.MatMulNBits(w, s.to(dev), 300, 64, zero_points=torch.from_numpy(z).to(dev), bias=c.to(dev))
        w.fill_(0)
        assert torch.equal(op(x), ref)


def test_nbits_empty_and_shapes(dev):
    b, s, z, c = weights(1, 24, 96, 32, torch.float16, False, True)
    op = nnr_amd.MatMulNBits(b, s, 96, 32, bias=c)
    assert op(torch.empty((0, 96), dtype=torch.float16, device=dev)).shape == (0, 24)
    a = torch.randn((2, 3, 96), device=dev).half()
    y = op(a)
    assert y.shape == (2, 3, 24) and torch.equal(y.reshape(6, 24), op(a.reshape(6, 96)))
    # columns of a wider tensor
    wide = torch.randn((5, 200), device=dev).half()
    assert torch.equal(op(wide[:, 3:99]), op(wide[:, 3:99].contiguous()))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("block", [32, 64, 256])
@pytest.mark.parametrize("m,n,k", [(450, 3201, 191), (200, 6401, 65), (1700, 2500, 193)])
def test_nbits_many_unaligned_rows(dev, t, block, m, n, k):
    """Rows of odd lengths where blocks share rows: a chunk of 64 k whole, cut short, and with nothing left in it"""
    check_nbits(dev, m, n, k, block, t, True, block == 64)


@pytest.mark.parametrize("t,k", [(torch.float32, 33), (torch.float16, 64)])
def test_nbits_most_rows(dev, t, k):
    """2^20 rows, the most that a call takes, by row loads of either kind; one more is refused."""
    b, s, z, c = weights(2, 16, k, 32, t, True, True)
    op = nnr_amd.MatMulNBits(b, s, k, 32, zero_points=z, bias=c)
    a = torch.randn(((1 << 20) + 1, k), device=dev).to(t)
    y = op(a[:-1])
    for i in (0, 77777, (1 << 20) - 300):
        ref = op(a[i:i + 300])   # both: k 2^-24 of the terms' sum, and half a step of y
        assert ((y[i:i + 300] - ref).abs() <= 1e-2 * ref.abs() + 1e-2).all()
    with pytest.raises(nnr_amd.NnrHipError):
        op(a)


def test_calls_on_a_given_stream(dev):
    """Each call by a stream's handle while the current stream is busy: copies of
    rows and tables that the call makes are made on that stream."""
    st = torch.cuda.Stream()
    H, hd, page, B, S = 2, 64, 32, 2, 40
    b, s, z, c = weights(5, 24, 96, 32, torch.float16, True, True)
    op = nnr_amd.MatMulNBits(b, s, 96, 32, zero_points=z, bias=c)
    a = torch.randn((5, 200), device=dev).half()[:, 3:99]
    caches = [filled(dev, 8, H, hd, page_size=page) for _ in "ab"]
    k, v = (x.to(dev) for x in tokens(1, B, S, H, hd, torch.float16))
    k, v = k.transpose(1, 2).contiguous().transpose(1, 2), v.transpose(1, 2).contiguous().transpose(1, 2)
    q = torch.randn((B, 4 * H, S, hd), device=dev).half().transpose(1, 2)
    td = torch.arange(16, dtype=torch.int32, device=dev).reshape(8, 2)[:, 0].reshape(2, 4).t()[:2]
    lens = torch.tensor([40, 9, 33, 9], dtype=torch.int32, device=dev)[::2]
    td = torch.stack((td[:, 0] // 2, td[:, 1] // 2 + 1), 1).t().contiguous().t()

    def run(cache, **kw):
        y = op(a, **kw)
        cache.write(k, v, td, lens, **kw)
        return (y, *cache.read(S, td, lens, torch.float16, **kw), cache.attention(q, td, lens, **kw),
                cache.attention(q, td, lens, prefix_table=td[1], prefix_len=33, **kw))
    ref = run(caches[0])
    torch.cuda.synchronize()
    torch.cuda._sleep(50_000_000)
    got = run(caches[1], stream=st.cuda_stream)
    st.synchronize()
    torch.cuda.synchronize()
    for x, y in zip(got, ref):
        assert torch.equal(x, y)


def test_nbits_streams_share_a_handle(dev):
    b, s, z, c = weights(5, 512, 1024, 32, torch.bfloat16, True, False)
    op = nnr_amd.MatMulNBits(b, s, 1024, 32, zero_points=z)
    xs = [torch.randn((m, 1024), device=dev).bfloat16() for m in (1, 40, 300, 8)]
    ref = [op(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    out = []
    for _ in range(5):
        for x, st in zip(xs, streams):
            with torch.cuda.stream(st):
                out.append(op(x))
    torch.cuda.synchronize()
    for i, y in enumerate(out):
        assert torch.equal(y, ref[i % 4])


@pytest.mark.parametrize("dt", [np.float32, np.float16])
@pytest.mark.parametrize("kw", [dict(), dict(zp=False, bias=False), dict(block=128, K=300, N=70, shape=(5, 300)),
                                dict(shape=(70,))])
@pytest.mark.parametrize("onnx", [False, True])
def test_nbits_node(dev, dt, kw, onnx, tmp_path):
    """The node in a graph, from memory and from an ONNX file; run twice (the
    second time as a captured graph)"""
    from nnr_amd import onnx_io
    from nnr_amd.graph import Session
    g = R.nbits_graph(dt=dt, **kw)
    if onnx:
        onnx_io.save(g, str(tmp_path / "m.onnx"))
        s = Session(None, onnx=str(tmp_path / "m.onnx"))
    else:
        s = Session(g)
    i, t = g.initializers, torch.float32 if dt == np.float32 else torch.float16
    K, block = kw.get("K", 70), kw.get("block", 32)
    for seed in (1, 2, 3):
        x = np.random.default_rng(seed).standard_normal(g.inputs["x"][1]).astype(dt)
        s.set_input("x", x)
        s.run()
        y = s.output("y")[0].astype(np.float64).reshape(-1, i["s"].shape[0])
        ref, mag = R.nbits(x.reshape(-1, K), i["b"], i["s"], K, block, i.get("z"), i["c"].astype(np.float64) if "c" in i else None)
        assert R.close(y, ref, R.nbits_tol(ref, mag, K, t), t).all()


@pytest.mark.parametrize("kw", [dict(block=16), dict(scale_dt=np.float16), dict(drop=1), dict(attrs=dict(bits=8)),
                                dict(attrs=dict(block_size=48))])
def test_nbits_node_refuses(dev, kw):
    from nnr_amd.graph import Session
    with pytest.raises(RuntimeError, match="MatMulNBits|matmul_nbits"):
        Session(R.nbits_graph(**kw))


# ---------------------------------------------------------------------------
# the cache

def tables(rng, counts, page, spare=2, per=None):
    """Page tables over shuffled pages: [len(counts)][per], number of pages."""
    per = max(1, max(-(-n // page) for n in counts)) if per is None else per
    order = rng.permutation(len(counts) * per + spare).astype(np.int32)
    return torch.from_numpy(order[:len(counts) * per].reshape(len(counts), per).copy()), len(order), \
        torch.from_numpy(order[len(counts) * per:].copy())


def tokens(seed, B, S, H, hd, t):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn((B, S, H, hd), generator=g) * torch.exp(torch.randn((H, hd), generator=g))).to(t) for _ in "kv"]


def filled(dev, *args, **kw):
    """A cache whose memory holds what memory may hold: NaN scales among it."""
    c = nnr_amd.KVCache(*args, **kw)
    c.data.fill_(255)
    return c


def expect(x, bits, t):
    return R.quantize(x, bits)[0].to(t)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd,H,page", [(64, 3, 32), (96, 1, 64), (128, 2, 64), (256, 1, 128)])
def test_cache_values(dev, t, bits, hd, H, page):
    """Prompts of several lengths, padded at the front, then single tokens; every value as the formula has it."""
    lens = [70, 1, 33, 128]
    B, S = len(lens), 128
    rng = np.random.default_rng(hd)
    table, pages, _ = tables(rng, [n + 3 for n in lens], page)
    k, v = tokens(hd + bits, B, S + 3, H, hd, t)
    k[2, S - 5, 0, 3], v[2, S - 6, 0, 1] = float("nan"), float("inf")
    v[3, 7] = 0
    cache = filled(dev, pages, H, hd, page_size=page, bits=bits)
    td = table.to(dev)
    cache.write(k[:, :S].to(dev), v[:, :S].to(dev), td, torch.tensor(lens, dtype=torch.int32, device=dev))
    for i in range(3):
        cache.write(k[:, S + i:S + i + 1].to(dev), v[:, S + i:S + i + 1].to(dev), td,
                    torch.tensor([n + 1 + i for n in lens], dtype=torch.int32, device=dev))
    ks, vs = cache.read(S + 3, td, torch.tensor([n + 3 for n in lens], dtype=torch.int32, device=dev), t)
    for b, n in enumerate(lens):
        for got, x in ((ks, k), (vs, v)):
            assert torch.equal(got[b, S - n:].cpu(), expect(x[b, S - n:], bits, t))
            assert not got[b, :S - n].any()


@pytest.mark.parametrize("bits", [8, 4])
def test_cache_write_leaves_the_rest(dev, bits):
    """A write into the middle of a sequence changes those tokens alone."""
    H, hd, page = 2, 64, 32
    table, pages, _ = tables(np.random.default_rng(2), [100, 100], page)
    cache, td = filled(dev, pages, H, hd, page_size=page, bits=bits), table.to(dev)
    full = torch.tensor([100, 100], dtype=torch.int32, device=dev)
    k, v = (x.to(dev) for x in tokens(1, 2, 100, H, hd, torch.float32))
    cache.write(k, v, td, full)
    before = cache.data.clone()
    k2, v2 = (x.to(dev) for x in tokens(2, 2, 7, H, hd, torch.float32))
    cache.write(k2, v2, td, torch.tensor([60, 3], dtype=torch.int32, device=dev))
    k[0, 53:60], v[0, 53:60], k[1, :3], v[1, :3] = k2[0], v2[0], k2[1, 4:], v2[1, 4:]
    ks, vs = cache.read(100, td, full, torch.float32)
    for got, x in ((ks, k), (vs, v)):
        assert torch.equal(got.cpu(), expect(x.cpu(), bits, torch.float32))
    # and none of the pages that no table names
    named = set(table.reshape(-1).tolist())
    pb = cache.data.numel() // pages
    for p in set(range(pages)) - named:
        assert torch.equal(cache.data[p * pb:(p + 1) * pb], before[p * pb:(p + 1) * pb])


@pytest.mark.parametrize("bits", [8, 4])
def test_cache_without_pages(dev, bits):
    """Entries outside the cache, positions behind the last page, lengths below 0: nothing written, zeros read."""
    H, hd, page = 1, 96, 32
    cache = filled(dev, 3, H, hd, page_size=page, bits=bits)
    td = torch.tensor([[0, -1, 1], [7, 2, 3]], dtype=torch.int32, device=dev)
    k, v = tokens(4, 2, 110, H, hd, torch.float16)
    lens = torch.tensor([110, 96], dtype=torch.int32, device=dev)
    cache.write(k.to(dev), v.to(dev), td, lens)
    ks, vs = cache.read(110, td, lens, torch.float16)
    for got, x in ((ks.cpu(), k), (vs.cpu(), v)):
        e = expect(x, bits, torch.float16)
        e[0, 32:64] = 0          # page -1
        e[0, 96:] = 0            # no fourth page
        e[1, :14] = 0            # padding
        e[1, 14:46] = 0          # page 7
        e[1, 78:] = 0            # page 3
        assert torch.equal(got, e)
    before = cache.data.clone()
    cache.write(k.to(dev), v.to(dev), td, torch.tensor([0, -5], dtype=torch.int32, device=dev))
    assert torch.equal(cache.data, before)


def test_cache_strides(dev):
    """k and v as slices of one projection's output"""
    H, hd, page = 2, 128, 64
    table, pages, _ = tables(np.random.default_rng(3), [50, 50], page)
    cache, td = filled(dev, pages, H, hd, page_size=page), table.to(dev)
    qkv = torch.randn((2, 40, 8 * hd), device=dev).bfloat16()
    k, v = (qkv[..., i * H * hd:(i + 1) * H * hd].unflatten(-1, (H, hd)) for i in (2, 3))
    lens = torch.tensor([45, 50], dtype=torch.int32, device=dev)
    cache.write(k, v, td, lens)
    ks, vs = cache.read(40, td, lens, torch.bfloat16)
    assert torch.equal(ks.cpu(), expect(k.cpu(), 8, torch.bfloat16))
    assert torch.equal(vs.cpu(), expect(v.cpu(), 8, torch.bfloat16))


@pytest.mark.parametrize("bits", [8, 4])
def test_cache_borders(dev, bits):
    """Quotients next to a border between two codes, and scales next to one between two bf16 numbers."""
    L = 127 if bits == 8 else 7
    hd = 64
    rng = np.random.default_rng(8)
    n = 512
    x = np.zeros((n, hd), np.float32)
    top = (rng.integers(129, 256, n) / 128.0 * 2.0 ** rng.integers(-20, 20, n) * L).astype(np.float32)
    half = (rng.integers(257, 511, n) | 1) / 256.0 * L          # amax / L between two bf16 numbers
    top[::2] = half[::2].astype(np.float32)
    top = np.nextafter(top, np.float32(np.inf) * rng.choice([-1, 1], n).astype(np.float32)).astype(np.float32)
    s = (top.astype(np.float64) / L)
    for g in range(hd // 32):
        x[:, 32 * g] = top
        c = rng.integers(-L, L, (n, 31)) + 0.5
        b = torch.from_numpy(s).bfloat16().double().numpy()
        x[:, 32 * g + 1:32 * g + 32] = (c * b[:, None]).astype(np.float32)
        up = rng.integers(-1, 2, (n, 31))
        y = x[:, 32 * g + 1:32 * g + 32]
        y[up > 0] = np.nextafter(y[up > 0], np.float32(np.inf))
        y[up < 0] = np.nextafter(y[up < 0], np.float32(-np.inf))
    x = torch.from_numpy(x)[None, :, None]
    x = torch.minimum(torch.maximum(x, -x.abs()[..., :1]), x.abs()[..., :1])
    cache = filled(dev, n // 32, 1, hd, page_size=32, bits=bits)
    td = torch.arange(n // 32, dtype=torch.int32, device=dev)[None]
    lens = torch.tensor([n], dtype=torch.int32, device=dev)
    cache.write(x.to(dev), -x.to(dev), td, lens)
    ks, vs = cache.read(n, td, lens, torch.float32)
    assert torch.equal(ks.cpu(), expect(x, bits, torch.float32))
    assert torch.equal(vs.cpu(), expect(-x, bits, torch.float32))


@pytest.mark.parametrize("bits", [8, 4])
def test_cache_small_values(dev, bits):
    """Groups whose scale would be no normal number, and just is one"""
    x = torch.zeros(1, 4, 1, 64)
    L = 127 if bits == 8 else 7
    x[0, 0], x[0, 1, 0, 5], x[0, 2] = 1e-40, 1e-45, 2.0 ** -126 * L * 1.1
    x[0, 3, 0, 0] = 3e38
    cache = filled(dev, 1, 1, 64, page_size=32, bits=bits)
    td, lens = torch.zeros((1, 1), dtype=torch.int32, device=dev), torch.tensor([4], dtype=torch.int32, device=dev)
    cache.write(x.to(dev), x.to(dev), td, lens)
    for got in cache.read(4, td, lens, torch.float32):
        assert torch.equal(got.cpu(), expect(x, bits, torch.float32))


# ---------------------------------------------------------------------------
# attention

def check_attention(dev, t, bits, hd, H, G, S, lens, prefix, page, seed=0, qscale=1.0, per=None, scale=None):
    B = len(lens)
    rng = np.random.default_rng(seed + hd)
    pre_pages = -(-prefix // page)
    table, pages, spare = tables(rng, [max(n, 1) for n in lens], page, spare=pre_pages + 1, per=per)
    cache, td = filled(dev, pages, H, hd, page_size=page, bits=bits), table.to(dev)
    n = max(max(lens), 1)
    k, v = tokens(seed + 1, B, n, H, hd, t)
    ld = torch.tensor(lens, dtype=torch.int32, device=dev)
    cache.write(k.to(dev), v.to(dev), td, ld)
    pt = spare[:pre_pages].to(dev)
    pk, pv = tokens(seed + 2, 1, prefix, H, hd, t)
    if prefix:
        cache.write(pk.to(dev), pv.to(dev), pt[None], torch.tensor([prefix], dtype=torch.int32, device=dev))
    q = (torch.randn((B, S, H * G, hd), generator=torch.Generator().manual_seed(seed + 3)) * qscale).to(t)
    y = cache.attention(q.to(dev), td, ld, scale=scale, prefix_table=pt, prefix_len=prefix).cpu()
    sc = np.float32(hd ** -0.5 if scale is None else scale).item()
    worst = 0.0
    for h in range(H):
        pkx, pvx = (R.quantize(x[0, :, h], bits)[0] for x in (pk, pv))
        for b in range(B):
            kx = torch.cat((pkx, R.quantize(k[b, n - lens[b]:, h], bits)[0]))
            vx = torch.cat((pvx, R.quantize(v[b, n - lens[b]:, h], bits)[0]))
            vis = [prefix + max(0, lens[b] - S + s + 1) for s in range(S)]
            qs = q[b, :, h * G:(h + 1) * G]
            ref, tol = R.attention(qs, kx, vx, sc, vis)
            mag, _ = R.attention(qs, kx, vx.abs(), sc, vis)
            err = (y[b, :, h * G:(h + 1) * G].double() - ref).abs()
            tol = R.attention_tol(ref, tol, mag, t)
            assert not torch.isnan(err).any()
            worst = max(worst, (err / tol).max().item())
    assert worst <= 1.0, worst


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd,H,G,S,lens,prefix,page", [
    (64, 1, 1, 1, [1], 0, 32),
    (64, 2, 3, 1, [0, 5, 32, 33, 64, 257], 0, 32),
    (128, 2, 4, 1, [700, 1, 129], 0, 64),
    (128, 1, 8, 1, [40] * 5 + [3], 300, 64),
    (96, 2, 1, 4, [4, 9, 2, 0], 37, 64),
    (256, 1, 4, 5, [60, 5, 100], 70, 128),
    (64, 1, 2, 40, [40, 90, 33], 0, 64),
    (256, 1, 1, 1, [1500], 1, 256),
    (128, 1, 32, 2, [200, 2], 64, 32),
    (64, 3, 1, 1, [0, 0], 500, 32),
    (96, 1, 2, 3, [0, 1], 0, 32)])
def test_attention(dev, t, bits, hd, H, G, S, lens, prefix, page):
    check_attention(dev, t, bits, hd, H, G, S, lens, prefix, page)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bits", [8, 4])
def test_attention_long(dev, t, bits):
    check_attention(dev, t, bits, 128, 1, 4, 1, [9000, 17, 4000], 5000, 64)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd", [64, 256])
def test_attention_many_rows(dev, bits, hd):
    """Rows of the prefix in several groups, the last not full"""
    check_attention(dev, torch.float16, bits, hd, 2, 3, 3, [7, 3, 20, 0, 64, 100, 1, 2, 90, 33, 31], 400, 32)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bits", [8, 4])
def test_attention_large_scores(dev, t, bits):
    """Scores of several hundred; a negative scale"""
    check_attention(dev, t, bits, 64, 1, 2, 1, [300, 40], 100, 32, qscale=30.0)
    check_attention(dev, t, bits, 64, 1, 2, 2, [65, 40], 0, 32, scale=-0.3)


@pytest.mark.parametrize("bits", [8, 4])
def test_attention_more_pages_than_tokens(dev, bits):
    """A table with room for far longer sequences"""
    check_attention(dev, torch.bfloat16, bits, 128, 2, 2, 1, [65, 10], 0, 32, per=120)


@pytest.mark.parametrize("bits", [8, 4])
def test_attention_pages_that_do_not_exist(dev, bits):
    """An entry outside the cache holds no tokens."""
    H, hd, page = 1, 64, 32
    cache = filled(dev, 4, H, hd, page_size=page, bits=bits)
    good = torch.tensor([[3, 0, 2]], dtype=torch.int32, device=dev)
    bad = torch.tensor([[3, 99, 2]], dtype=torch.int32, device=dev)
    k, v = tokens(3, 1, 90, H, hd, torch.float32)
    lens = torch.tensor([90], dtype=torch.int32, device=dev)
    cache.write(k.to(dev), v.to(dev), good, lens)
    q = torch.randn((1, 1, 2, hd), generator=torch.Generator().manual_seed(1))
    y = cache.attention(q.to(dev), bad, lens).cpu()
    keep = [i for i in range(90) if not 32 <= i < 64]
    kx, vx = (R.quantize(x[0, keep, 0], bits)[0] for x in (k, v))
    ref, tol = R.attention(q[0], kx, vx, np.float32(hd ** -0.5).item(), [len(keep)])
    mag, _ = R.attention(q[0], kx, vx.abs(), np.float32(hd ** -0.5).item(), [len(keep)])
    assert ((y[0].double() - ref).abs() <= R.attention_tol(ref, tol, mag, torch.float32)).all()
    none = cache.attention(q.to(dev), torch.tensor([[-1, 4, 5]], dtype=torch.int32, device=dev), lens)
    assert not none.any()


@pytest.mark.parametrize("hd,S,heads,prefix", [(64, 1, 1, 0), (128, 1, 8, 40), (128, 40, 2, 40), (256, 9, 4, 100)])
def test_attention_without_keys(dev, hd, S, heads, prefix):
    """No pages at all, and tables of no pages: zeros for every query."""
    q = torch.randn((3, S, heads, hd), device=dev).half()
    lens = torch.tensor([0, 50, 2 ** 31 - 1], dtype=torch.int32, device=dev)
    pt = torch.tensor([0, 1, 5, -1], dtype=torch.int32, device=dev)
    for pages, per in ((0, 4), (0, 0), (2, 0)):
        cache = filled(dev, pages, 1, hd, page_size=32)
        td = torch.zeros((3, per), dtype=torch.int32, device=dev)
        assert not cache.attention(q, td, lens).any()
        if pages == 0 and prefix:
            assert not cache.attention(q, td, lens, prefix_table=pt, prefix_len=prefix).any()
        k = torch.randn((3, S, 1, hd), device=dev)
        cache.write(k, k, td, lens)
        assert not any(x.any() for x in cache.read(S, td, lens, torch.float32))


@pytest.mark.parametrize("bits", [8, 4])
def test_attention_splits_in_a_graph(dev, bits):
    """Prefix, many rows and splits captured; replays after the lengths and the
    queries changed, eager calls between, two graphs over one workspace in turn."""
    H, hd, page, B, S, G = 2, 128, 64, 3, 3, 8
    cache = filled(dev, 70, H, hd, page_size=page, bits=bits)
    td = torch.arange(60, dtype=torch.int32, device=dev).reshape(3, 20)
    pt = torch.arange(60, 70, dtype=torch.int32, device=dev)
    lens = torch.tensor([1280, 700, 64], dtype=torch.int32, device=dev)
    for tab, n in ((td, 1280), (pt.reshape(1, 10), 640)):
        k, v = (x.to(dev) for x in tokens(n, len(tab), n, H, hd, torch.float16))
        cache.write(k, v, tab, torch.full((len(tab),), n, dtype=torch.int32, device=dev))
    q = torch.randn((B, S, H * G, hd), device=dev).half()
    size = cache.attention_workspace(B, S, H * G, 20, 600)
    assert size > 0
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    cache.attention(q, td, lens, prefix_table=pt, prefix_len=600, workspace=ws)
    torch.cuda.synchronize()
    graphs, ys = [], []
    for prefix in (600, 64):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ys.append(cache.attention(q, td, lens, prefix_table=pt, prefix_len=prefix, workspace=ws))
        graphs.append(g)
    for i in range(4):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(i)).half())
        lens.copy_(torch.tensor([1280 - 100 * i, 3 + i, 64 * i], dtype=torch.int32))
        for g in graphs:
            g.replay()
        for y, prefix in zip(ys, (600, 64)):
            assert torch.equal(y, cache.attention(q, td, lens, prefix_table=pt, prefix_len=prefix))
        torch.cuda.synchronize()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bits", [8, 4])
def test_attention_rows_do_not_mix(dev, t, bits):
    """A query with a NaN or an infinity is NaN alone."""
    H, hd, page, G = 1, 128, 32, 4
    table, pages, _ = tables(np.random.default_rng(1), [70, 70], page)
    cache, td = filled(dev, pages, H, hd, page_size=page, bits=bits), table.to(dev)
    k, v = tokens(5, 2, 70, H, hd, t)
    lens = torch.tensor([70, 41], dtype=torch.int32, device=dev)
    cache.write(k.to(dev), v.to(dev), td, lens)
    q = torch.randn((2, 3, G, hd), device=dev).to(t)
    clean = cache.attention(q, td, lens)
    bad = q.clone()
    bad[0, 1, 2, 5], bad[1, 2, 0, 0] = float("nan"), float("inf")
    y = cache.attention(bad, td, lens)
    assert torch.isnan(y[0, 1, 2]).all() and torch.isnan(y[1, 2, 0]).all()
    rows = torch.ones(2, 3, G, dtype=torch.bool)
    rows[0, 1, 2] = rows[1, 2, 0] = False
    assert torch.equal(y[rows], clean[rows])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bits", [8, 4])
def test_attention_values_of_all_sizes(dev, t, bits):
    """Tokens whose values differ by many orders, and a sequence of zeros"""
    H, hd, page, n = 1, 64, 32, 200
    cache = filled(dev, 8, H, hd, page_size=page, bits=bits)
    td = torch.arange(7, dtype=torch.int32, device=dev)[None]
    k, v = tokens(6, 1, n, H, hd, torch.float32)
    v = v * torch.logspace(-4, 4, n)[None, :, None, None] if t == torch.float16 else \
        v * torch.logspace(-30, 30, n)[None, :, None, None]
    k, v = k.to(t), v.to(t)
    lens = torch.tensor([n], dtype=torch.int32, device=dev)
    q = (0.1 * torch.randn((1, 1, 1, hd), generator=torch.Generator().manual_seed(1))).to(t)
    sc = np.float32(hd ** -0.5).item()
    for flip in (False, True):     # the unit grows, and is large from the start
        vv = v.flip(1) if flip else v
        cache.write(k.to(dev), vv.to(dev), td, lens)
        y = cache.attention(q.to(dev), td, lens).cpu()
        kx, vx = R.quantize(k[0, :, 0], bits)[0], R.quantize(vv[0, :, 0], bits)[0]
        ref, tol = R.attention(q[0], kx, vx, sc, [n])
        mag, _ = R.attention(q[0], kx, vx.abs(), sc, [n])
        assert ((y[0].double() - ref).abs() <= R.attention_tol(ref, tol, mag, t)).all()
    cache.write(k.to(dev), torch.zeros_like(v).to(dev), td, lens)
    assert not cache.attention(q.to(dev), td, lens).any()


def test_attention_strided_and_in_place(dev):
    H, hd, page, G = 2, 64, 32, 2
    table, pages, _ = tables(np.random.default_rng(1), [70, 70], page)
    cache, td = filled(dev, pages, H, hd, page_size=page), table.to(dev)
    k, v = tokens(5, 2, 70, H, hd, torch.float16)
    lens = torch.tensor([70, 41], dtype=torch.int32, device=dev)
    cache.write(k.to(dev), v.to(dev), td, lens)
    qkv = torch.randn((2, 3, 8 * hd), device=dev).half()
    q = qkv[..., 2 * hd:6 * hd].unflatten(-1, (4, hd))
    ref = cache.attention(q.contiguous(), td, lens)
    assert torch.equal(cache.attention(q, td, lens), ref)
    over = q.contiguous()
    assert cache.attention(over, td, lens, y=over) is over and torch.equal(over, ref)


def test_attention_beyond_32_bits(dev):
    """Pages whose bytes lie past 2^32"""
    H, hd, page = 8, 256, 128
    pages = 9000      # 4.7 GB
    cache = nnr_amd.KVCache(pages, H, hd, page_size=page)
    assert cache.data.numel() > 2 ** 32
    table = torch.tensor([[pages - 1, 0], [pages - 2, pages - 3]], dtype=torch.int32, device=dev)
    small = nnr_amd.KVCache(4, H, hd, page_size=page)
    stable = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=dev)
    k, v = (x.to(dev) for x in tokens(1, 2, 200, H, hd, torch.float16))
    lens = torch.tensor([200, 190], dtype=torch.int32, device=dev)
    q = torch.randn((2, 1, 8, hd), device=dev).half()
    out = []
    for c, tb in ((cache, table), (small, stable)):
        c.write(k, v, tb, lens)
        out.append((c.attention(q, tb, lens), *c.read(200, tb, lens, torch.float16)))
    for a, b in zip(*out):
        assert torch.equal(a, b)


# ---------------------------------------------------------------------------
# together

class Layer:
    """A decoder layer's attention: 4-bit q, k, v projections in one, cache, attention, 4-bit output projection."""

    def __init__(self, seed, hidden, H, G, hd, t):
        self.H, self.G, self.hd, self.t = H, G, hd, t
        wide = (H * G + 2 * H) * hd
        self.w = weights(seed, wide, hidden, 32, t, True, True)
        self.o = weights(seed + 1, hidden, H * G * hd, 64, t, False, False)
        scale = lambda w, k: (w[0], (w[1].float() * 3 / k ** 0.5).to(t), *w[2:])
        self.w, self.o = scale(self.w, hidden), scale(self.o, H * G * hd)
        self.qkv = nnr_amd.MatMulNBits(*self.w[:2], hidden, 32, zero_points=self.w[2], bias=self.w[3])
        self.out = nnr_amd.MatMulNBits(*self.o[:2], H * G * hd, 64)

    def step(self, x, cache, td, lens, **kw):
        B, S, _ = x.shape
        y = self.qkv(x)
        cut = self.H * self.G * self.hd
        q = y[..., :cut].unflatten(-1, (self.H * self.G, self.hd))
        k = y[..., cut:cut + self.H * self.hd].unflatten(-1, (self.H, self.hd))
        v = y[..., cut + self.H * self.hd:].unflatten(-1, (self.H, self.hd))
        cache.write(k, v, td, lens)
        return self.out(cache.attention(q, td, lens, **kw).flatten(-2)), (q, k, v)

    def exact(self, x):
        f = lambda a, w, k, blk: R.nbits(a, w[0], f64(w[1]), k, blk, w[2], None if w[3] is None else f64(w[3]))[0]
        return f(x, self.w, x.shape[-1], 32)

    def exact_out(self, a):
        return R.nbits(a, self.o[0], f64(self.o[1]), a.shape[-1], 64, None, None)[0]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bits", [8, 4])
def test_decoder_layer(dev, t, bits):
    """A shared prompt, then three steps of four sequences, in float64 beside it:
    each operator's result within its own tolerance given its actual inputs."""
    hidden, H, G, hd, page, B, P = 256, 2, 2, 64, 32, 4, 75
    layer = Layer(3, hidden, H, G, hd, t)
    pre = torch.tensor([5, 1, 8], dtype=torch.int32, device=dev)
    td = torch.tensor([[0], [2], [3], [4]], dtype=torch.int32, device=dev)
    cache = filled(dev, 10, H, hd, page_size=page, bits=bits)
    g = torch.Generator().manual_seed(9)
    x = torch.randn((1, P, hidden), generator=g).to(t).to(dev)
    _, (q, k, v) = layer.step(x, cache, pre[None], torch.tensor([P], dtype=torch.int32, device=dev))
    ref, mag = R.nbits(f64(x[0]), layer.w[0], f64(layer.w[1]), hidden, 32, layer.w[2], f64(layer.w[3]))
    y = np.concatenate([f64(z.flatten(-2))[0] for z in (q, k, v)], -1)
    assert (np.abs(y - ref) <= R.nbits_tol(ref, mag, hidden, t)).all()
    hist = [[k.cpu(), v.cpu()]]
    own = [[], []]
    for i in range(3):
        x = torch.randn((B, 1, hidden), generator=g).to(t).to(dev)
        lens = torch.full((B,), i + 1, dtype=torch.int32, device=dev)
        out, (q, k, v) = layer.step(x, cache, td, lens, prefix_table=pre, prefix_len=P)
        own[0].append(k.cpu())
        own[1].append(v.cpu())
        att = cache.attention(q, td, lens, prefix_table=pre, prefix_len=P)
        sc = np.float32(hd ** -0.5).item()
        for b in range(B):
            for h in range(H):
                kx, vx = (R.quantize(torch.cat((hist[0][j][0, :, h], torch.cat(own[j], 1)[b, :, h])), bits)[0] for j in (0, 1))
                qs = q[b, :, h * G:(h + 1) * G].cpu()
                ref, tol = R.attention(qs, kx, vx, sc, [P + i + 1])
                wt, _ = R.attention(qs, kx, vx.abs(), sc, [P + i + 1])
                err = (att[b, :, h * G:(h + 1) * G].cpu().double() - ref).abs()
                assert (err <= R.attention_tol(ref, tol, wt, t)).all()
        a = f64(att.flatten(-2))[:, 0]
        ref, mag = R.nbits(a, layer.o[0], f64(layer.o[1]), a.shape[-1], 64, None, None)
        assert (np.abs(f64(out)[:, 0] - ref) <= R.nbits_tol(ref, mag, a.shape[-1], t)).all()


@pytest.mark.parametrize("bits", [8, 4])
def test_decoder_layer_in_a_graph(dev, bits):
    """The step captured once and replayed as the sequences grow, with eager work
    between; the same results as eager steps."""
    t, hidden, H, G, hd, page, B = torch.float16, 128, 2, 2, 64, 32, 3
    layer = Layer(4, hidden, H, G, hd, t)
    td = torch.arange(3 * 12, dtype=torch.int32, device=dev).reshape(3, 12)
    caches = [filled(dev, 36, H, hd, page_size=page, bits=bits) for _ in "ab"]
    x = torch.zeros((B, 1, hidden), dtype=t, device=dev)
    lens = torch.tensor([1, 30, 200], dtype=torch.int32, device=dev)
    k, v = (z.to(dev) for z in tokens(1, B, 200, H, hd, t))
    for c in caches:
        c.write(k, v, td, lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c in caches:          # (it writes the last token)
            layer.step(x, c, td, lens)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, _ = layer.step(x, caches[0], td, lens)
    for i in range(5):
        x.copy_(torch.randn((B, 1, hidden), generator=torch.Generator().manual_seed(i)).to(t))
        lens += 1
        graph.replay()
        got = y.clone()
        ref, _ = layer.step(x, caches[1], td, lens)
        assert torch.equal(got, ref)
        torch.cuda.synchronize()
    a, b = (c.read(210, td, lens, t) for c in caches)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
