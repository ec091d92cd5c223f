"""Operators of a decoder's step where ranges, sizes and rows are far apart, against float64."""
import numpy as np
import pytest
import torch

import decode_range_ref as D
import decode_ref as R
import nnr_amd

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("typed", [False, True])
def test_workspace_made_before_the_call(dev, t, typed):
    """A workspace of the size that attention_workspace names serves the call, which
    writes nothing behind it; shapes at which the types' sizes differ."""
    H, hd, page = 8, 128, 64
    for B, S, heads, per, prefix in ((8, 64, 32, 64, 0), (32, 1, 32, 8, 4096)):
        pages = prefix // page + 4
        cache = nnr_amd.KVCache(pages, H, hd, page_size=page)
        td = torch.full((B, per), pages - 1, dtype=torch.int32, device=dev)
        pt = torch.arange(prefix // page, dtype=torch.int32, device=dev)
        lens = torch.full((B,), S, dtype=torch.int32, device=dev)
        k = torch.randn((1, S, H, hd), device=dev).to(t)
        cache.write(k, k, td[:1], lens[:1])
        q = torch.randn((B, S, heads, hd), device=dev).to(t)
        n = cache.attention_workspace(B, S, heads, per, prefix, **(dict(dtype=t) if typed else {}))
        buf = torch.full((n + 4096,), 77, dtype=torch.uint8, device=dev)
        kw = dict(prefix_table=pt, prefix_len=prefix)
        y = cache.attention(q, td, lens, workspace=buf[:n], **kw)
        assert torch.equal(y, cache.attention(q, td, lens, **kw))
        assert (buf[n:] == 77).all()


def run_attention(dev, t, bits, shape, q, k, v, pk, pv, scale=None):
    """(result, float64's, how far it may be off), each [rows, hd]"""
    lens, S, H, G, hd, P, per = D.sizes(shape)
    B, n, page = len(lens), max(lens), 32
    pre = -(-P // page)
    order = torch.randperm(B * per + pre + 1, generator=torch.Generator().manual_seed(5)).to(torch.int32)
    td, pt = order[:B * per].reshape(B, per).to(dev), order[B * per:B * per + pre].to(dev)
    cache = nnr_amd.KVCache(len(order), H, hd, page_size=page, bits=bits)
    cache.data.fill_(255)
    ld = torch.tensor(lens, dtype=torch.int32, device=dev)
    cache.write(k.to(dev), v.to(dev), td, ld)
    if P:
        cache.write(pk.to(dev), pv.to(dev), pt[None], torch.tensor([P], dtype=torch.int32, device=dev))
    y = cache.attention(q.to(dev), td, ld, scale=scale, prefix_table=pt, prefix_len=P).cpu()
    sc = torch.tensor(hd ** -0.5 if scale is None else scale, dtype=torch.float32).item()
    out = []
    for h in range(H):
        pkx, pvx = (R.quantize(x[0, :, h], bits)[0] for x in (pk, pv))
        for b in range(B):
            kx = torch.cat((pkx, R.quantize(k[b, n - lens[b]:, h], bits)[0]))
            vx = torch.cat((pvx, R.quantize(v[b, n - lens[b]:, h], bits)[0]))
            vis = [P + max(0, lens[b] - S + s + 1) for s in range(S)]
            ref, tol = D.attention(q[b, :, h * G:(h + 1) * G], kx, vx, sc, vis, bits)
            out.append([x.reshape(-1, hd) for x in (y[b, :, h * G:(h + 1) * G].double(), ref, tol)])
    return [torch.cat(x) for x in zip(*out)]


@pytest.mark.parametrize("shape", list(D.SHAPES))
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bits", [8, 4])
def test_attention_large_values(dev, t, bits, shape):
    """Results that fit their type, of values next to its largest number"""
    lens, S, H, G, hd, P, _ = D.sizes(shape)
    top = {torch.float32: 3e38, torch.float16: 6e4, torch.bfloat16: 3e38}[t]
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.rand(s, generator=g, dtype=torch.float64) * 2 - 1
    q, k, pk = r(len(lens), S, H * G, hd), r(len(lens), max(lens), H, hd), r(1, P, H, hd)
    v, pv = r(len(lens), max(lens), H, hd) * top, r(1, P, H, hd) * top
    # (a token's largest element stands for up to 2^-8 more than it is)
    v, pv = v.clamp(-0.95 * top, 0.95 * top), pv.clamp(-0.95 * top, 0.95 * top)
    y, ref, tol = run_attention(dev, t, bits, shape, *(x.to(t) for x in (q, k, v, pk, pv)))
    assert torch.isfinite(y).all()
    assert ((y - ref).abs() <= tol).all(), ((y - ref).abs() / tol).max()


@pytest.mark.parametrize("shape", list(D.SHAPES))
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("size", [1e-30, 1e25, 1e36])
def test_attention_large_and_small_keys(dev, t, bits, shape, size):
    """Scores of ordinary size out of keys and queries that are not"""
    lens, S, H, G, hd, P, _ = D.sizes(shape)
    q, k, v, pk, pv = D.inputs("", shape, torch.float64)
    y, ref, tol = run_attention(dev, t, bits, shape, (q / size).to(t), *(x.to(t) for x in (k * size, v, pk * size, pv)))
    assert ((y - ref).abs() <= tol).all(), ((y - ref).abs() / tol).max()


@pytest.mark.parametrize("shape", list(D.SHAPES))
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("pattern", D.PATTERNS)
def test_attention_sizes_far_apart(dev, t, bits, shape, pattern):
    """Groups, tokens and rows that another's size may not cost their bits"""
    y, ref, tol = run_attention(dev, t, bits, shape, *D.inputs(pattern, shape, t))
    assert torch.isfinite(ref).all() and ((y - ref).abs() <= tol).all(), ((y - ref).abs() / tol).max()


@pytest.mark.parametrize("shape", ["one block", "splits", "prompt"])
@pytest.mark.parametrize("bits", [8, 4])
def test_attention_sizes_far_apart_repeats(dev, bits, shape):
    """Such rows too: the same from call to call, over their own queries, and in a
    graph whose values grow apart and come together again"""
    lens, S, H, G, hd, P, per = D.sizes(shape)
    B, n, t = len(lens), max(lens), torch.bfloat16
    cache = nnr_amd.KVCache(B * per + 8, H, hd, page_size=32, bits=bits)
    td = torch.arange(B * per, dtype=torch.int32, device=dev).reshape(B, per)
    pt = torch.arange(B * per, B * per + 7, dtype=torch.int32, device=dev)
    ld = torch.tensor(lens, dtype=torch.int32, device=dev)

    def fill(pattern):
        q, k, v, pk, pv = (x.to(dev) for x in D.inputs(pattern, shape, t))
        cache.write(k, v, td, ld)
        if P:
            cache.write(pk, pv, pt[None], torch.tensor([P], dtype=torch.int32, device=dev))
        return q
    q = fill("value tokens")
    kw = dict(prefix_table=pt, prefix_len=P)
    first = cache.attention(q, td, ld, **kw)
    for _ in range(3):
        assert torch.equal(cache.attention(q, td, ld, **kw), first)
    over = q.clone()
    assert torch.equal(cache.attention(over, td, ld, y=over, **kw), first)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = cache.attention(q, td, ld, **kw)
    for pattern in ("", "key tokens", "value tokens", "", "seen later"):
        q.copy_(fill(pattern))
        graph.replay()
        got = y.clone()
        assert torch.equal(got, cache.attention(q, td, ld, **kw))
        torch.cuda.synchronize()


def test_nbits_rows_past_32_bits(dev):
    """Refused, not taken for their remainder"""
    op = nnr_amd.MatMulNBits(torch.zeros((1, 1, 16), dtype=torch.uint8), torch.ones((1, 1), dtype=torch.float16), 1, 32)
    with pytest.raises(ValueError, match="32 bits"):
        op(torch.empty((2 ** 32 + 5, 1), dtype=torch.float16, device=dev))


# ---------------------------------------------------------------------------
# sizes that the kernels tell apart

@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("k,block", [(33, 32), (64, 32), (96, 64)])
def test_nbits_most_rows_values(dev, t, k, block):
    """2^20 rows against float64, at both ends, in the middle and across a block's end"""
    m, n = 1 << 20, 20
    rng = np.random.default_rng(k)
    nb = -(-k // block)
    b, z = rng.integers(0, 256, (n, nb, block // 2), dtype=np.uint8), rng.integers(0, 256, (n, (nb + 1) // 2), dtype=np.uint8)
    s, c = torch.from_numpy(rng.uniform(0.01, 0.1, (n, nb))).to(t), torch.from_numpy(rng.standard_normal(n)).to(t)
    op = nnr_amd.MatMulNBits(b, s, k, block, zero_points=z, bias=c)
    a = torch.randn((m, k), device=dev).to(t)
    y = op(a)
    for i in (0, 77777, (1 << 19) - 150, m - 300):
        f = lambda x: x.detach().cpu().double().numpy()
        ref, mag = R.nbits(f(a[i:i + 300]), b, f(s), k, block, z, f(c))
        tol = R.nbits_tol(ref, mag, k, t)
        assert R.close(f(y[i:i + 300]), ref, tol, t).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd", [64, 96, 128])
@pytest.mark.parametrize("lens,S,G,prefix", [
    ([300], 300, 1, 0),                  # a prompt: rows of 128 a block and what is left of them
    ([520, 417], 260, 2, 0),             # the second part of one, 520 rows
    ([64, 70, 33], 50, 4, 190),          # 600 rows of a prefix, 200 of each sequence
    ([5] * 130, 1, 2, 130),              # 260 rows of a prefix, few of each sequence
    ([129], 129, 1, 0), ([128], 128, 1, 1)])
def test_attention_prompts(dev, t, bits, hd, lens, S, G, prefix):
    """More rows of a head than a block holds"""
    shape = (lens, S, 1, G, hd, prefix, -(-max(lens) // 32))
    y, ref, tol = run_attention(dev, t, bits, shape, *D.inputs("", shape, t))
    assert ((y - ref).abs() <= tol).all(), ((y - ref).abs() / tol).max()


@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits", [8, 4])
def test_attention_long_prompt(dev, t, bits):
    """1200 new tokens over splits of their own and of a prefix"""
    shape = ([1200], 1200, 1, 2, 128, 700, 40)
    y, ref, tol = run_attention(dev, t, bits, shape, *D.inputs("", shape, t))
    assert ((y - ref).abs() <= tol).all(), ((y - ref).abs() / tol).max()


@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("bits", [8, 4])
def test_attention_weights_next_to_ties(dev, bits, own):
    """Weights of fp32 tensors in two pieces: their sum is the weight also where it
    lies beside the middle of two fp16 numbers. Two keys, the second's value 0, so
    that nothing hides the first's weight; 2^16 of them."""
    hd, n = 64, 1 << 16
    g = torch.Generator().manual_seed(2)
    k, v = torch.randn((1, 2, 1, hd), generator=g), torch.randn((1, 2, 1, hd), generator=g)
    v[:, 1] = 0
    cache = nnr_amd.KVCache(1, 1, hd, page_size=32, bits=bits)
    two = torch.full((1,), 2, dtype=torch.int32, device=dev)
    cache.write(k.to(dev), v.to(dev), torch.zeros((1, 1), dtype=torch.int32, device=dev), two)
    kx, vx = (R.quantize(x[0, :, 0], bits)[0] for x in (k, v))
    if own:     # 16384 sequences of those tokens, 4 queries each
        q, lens = 0.3 * torch.randn((n // 4, 1, 4, hd), generator=g), torch.full((n // 4,), 2, dtype=torch.int32, device=dev)
        y = cache.attention(q.to(dev), torch.zeros((n // 4, 1), dtype=torch.int32, device=dev), lens)
    else:       # a prefix that 2^16 queries see
        q, lens = 0.3 * torch.randn((1, n // 4, 4, hd), generator=g), torch.zeros(1, dtype=torch.int32, device=dev)
        y = cache.attention(q.to(dev), torch.zeros((1, 1), dtype=torch.int32, device=dev), lens,
                            prefix_table=torch.zeros(1, dtype=torch.int32, device=dev), prefix_len=2)
    q, y = q.reshape(n, hd).double(), y.reshape(n, hd).cpu().double()
    p = torch.softmax(q @ kx.T * hd ** -0.5, -1)[:, :1]
    # of both keys' scores, each in p and in the total; the weight's two pieces and what is left of
    # the second (2^-21); maximum, exponential, total, division and result, an operation each
    e = hd ** -0.5 * ((hd + 16) * R.U + 2.0 ** -22) * (q.abs() @ kx.abs().T).sum(-1, keepdim=True)
    tol = (2 * e + 2.0 ** -21 + 16 * R.U) * (p * vx[0]).abs()
    assert tol.max() < 2.0 ** -12 * vx.abs().max()
    assert ((y - p * vx[0]).abs() <= tol).all(), ((y - p * vx[0]).abs() / tol).nan_to_num(0).max()
