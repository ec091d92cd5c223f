"""Operators around a decoder's cache against float64: rotary positions, attention
of packed prompts, of trees of drafts over the cache, pages and tokens moved."""
import numpy as np
import pytest
import torch

import decode_ref as D
import nnr_amd
import serving_ref as R
from nnr_amd import _lib

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def ints(dev, x):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def near(y, ref, tol, t):
    y = y.detach().cpu().double()
    ok = torch.from_numpy(D.close(y.numpy(), ref.numpy(), tol.numpy(), t)) | (y.isnan() & ref.isnan())
    assert ok.all(), ((y - ref).abs() / tol)[~ok].max()


# ---------------------------------------------------------------------------
# rotary positions

def check_rotary(dev, t, B, S, Hq, Hk, hd, r, interleaved, first=0, seed=0, wide=0, **scaling):
    held = 70000
    rope = nnr_amd.RotaryEmbedding(hd, held, base=10000.0, rotary_dim=r, interleaved=interleaved, device=dev, **scaling)
    if scaling:
        f, m = R.frequencies(r, 10000.0, scaling["scaling"], scaling["factor"], held / scaling["factor"])
    else:
        f, m = R.frequencies(r, 10000.0)
    # slices of one projection's output, `wide` elements further apart
    rows = (torch.randn((B, S, (Hq + Hk) * hd + wide), generator=gen(seed)) * 3).to(t).to(dev)
    q, k = rows[..., :Hq * hd].unflatten(-1, (Hq, hd)), rows[..., Hq * hd:(Hq + Hk) * hd].unflatten(-1, (Hk, hd))
    pos = torch.randint(first, held, (B, S), generator=gen(seed + 1)).to(torch.int32)
    before = rows.clone()
    out = rope(q, k, pos.to(dev))
    assert torch.equal(rows, before)
    for x, y in zip((q, k), out):
        assert y.shape == x.shape and y.dtype == t and y.is_contiguous()
        near(y, *R.rotate(x.cpu(), pos, f, m, interleaved, held), t)
        assert torch.equal(y[..., r:], x[..., r:])
    # in place: the same, and nothing else of the rows changed
    rope(q, k, pos.to(dev), out=(q, k))
    assert torch.equal(q, out[0]) and torch.equal(k, out[1])
    assert torch.equal(rows[..., (Hq + Hk) * hd:], before[..., (Hq + Hk) * hd:])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,S,Hq,Hk,hd,r,wide", [
    (1, 1, 1, 1, 64, 64, 0), (3, 1, 32, 8, 128, 128, 0), (2, 37, 4, 2, 128, 64, 128), (5, 33, 3, 3, 96, 40, 96),
    (1, 257, 8, 1, 256, 256, 0), (2, 5, 2, 2, 80, 80, 0), (2, 5, 2, 1, 64, 6, 0), (1, 9, 2, 1, 10, 6, 3), (2, 3, 1, 1, 7, 2, 1),
    (2, 4, 3, 2, 64, 0, 0)])
def test_rotary(dev, t, interleaved, B, S, Hq, Hk, hd, r, wide):
    check_rotary(dev, t, B, S, Hq, Hk, hd, r, interleaved, wide=wide, seed=hd + r)


@pytest.mark.parametrize("scaling", ["linear", "ntk", "yarn"])
@pytest.mark.parametrize("factor", [2.0, 16.0])
def test_rotary_scaled(dev, scaling, factor):
    check_rotary(dev, torch.float32, 2, 50, 4, 2, 128, 128, False, first=60000, scaling=scaling, factor=factor)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_positions(dev, t, interleaved):
    """Padding is left as it is, the last position turned, what lies beyond gives NaN."""
    held = 50
    rope = nnr_amd.RotaryEmbedding(64, held, rotary_dim=48, interleaved=interleaved, device=dev)
    pos = torch.tensor([[-1, 0, 49, 50, 2 ** 31 - 1, -2 ** 31]], dtype=torch.int32)
    q, k = (torch.randn((1, 6, h, 64), generator=gen(h)).to(t).to(dev) for h in (2, 1))
    f, m = R.frequencies(48, 10000.0)
    for x, y in zip((q, k), rope(q, k, pos.to(dev))):
        near(y, *R.rotate(x.cpu(), pos, f, m, interleaved, held), t)
        assert torch.equal(y[0, [0, 5]], x[0, [0, 5]]) and y[0, 3:5, :, :48].isnan().all()
        assert torch.equal(y[0, 1], x[0, 1]) and torch.equal(y[..., 48:], x[..., 48:])


def test_rotary_frequencies_given(dev):
    f = np.array([0.5, 0.25, 1e-3])
    rope = nnr_amd.RotaryEmbedding(8, 100, rotary_dim=6, frequencies=f, magnitude=1.25, device=dev)
    q = torch.randn((1, 20, 2, 8), generator=gen(1))
    pos = torch.arange(80, 100, dtype=torch.int32)[None]
    near(rope(q.to(dev), q.to(dev), pos.to(dev))[1], *R.rotate(q, pos, f, 1.25, False, 100), torch.float32)


def test_rotary_streams_and_graphs(dev):
    """On a given stream; captured and replayed with new positions, in place of eager calls between."""
    rope = nnr_amd.RotaryEmbedding(128, 4096, device=dev)
    q, k = (torch.randn((2, 3, h, 128), generator=gen(h)).to(dev) for h in (4, 2))
    pos = ints(dev, [[5, 6, 7], [1000, 1001, 1002]])
    want = rope(q, k, pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = rope(q, k, pos, stream=side.cuda_stream)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.cuda.stream(side):
        rope(q, k, pos)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rope(q, k, pos)
    for i in range(3):
        pos += i
        want = rope(q, k, pos)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_rotary_refuses(dev):
    rope = nnr_amd.RotaryEmbedding(64, 100, device=dev)
    rows = torch.zeros((2, 3, 6 * 64 + 8), device=dev)
    q, k = rows[..., :256].unflatten(-1, (4, 64)), rows[..., 256:384].unflatten(-1, (2, 64))
    pos = torch.zeros((2, 3), dtype=torch.int32, device=dev)
    for bad in (lambda: rope(q[..., :32], k, pos), lambda: rope(q, k.half(), pos), lambda: rope(q, k, pos.long()),
                lambda: rope(q, k, pos[:1]), lambda: rope(q, k[:1], pos), lambda: rope(q, k, pos.cpu()),
                lambda: rope(q, k, pos, out=(q, k.cpu())), lambda: rope(q, k, pos, out=(q.half(), k)),
                lambda: rope(q, k, pos, out=(q, k.transpose(1, 2).contiguous().transpose(1, 2)))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        rope(q.double(), k.double(), pos)
    with pytest.raises(nnr_amd.NnrHipError):
        rope(q, q, pos, out=(q, q))
    # a result a part of a head further, over k's rows, over itself
    for qy, ky in ((rows[..., 8:264].unflatten(-1, (4, 64)), k), (q, rows[..., 128:256].unflatten(-1, (2, 64))),
                   (q, torch.zeros((2, 2, 64), device=dev)[:, None].expand(2, 3, 2, 64))):
        with pytest.raises(nnr_amd.NnrHipError):
            rope(q, k, pos, out=(qy, ky))


# ---------------------------------------------------------------------------
# attention of prompts

def prompts(seed, lens, Hq, Hk, hd, t, size=1.0):
    T = sum(lens)
    g = gen(seed)
    spread = torch.cat((torch.full((Hq, hd), size), torch.exp(0.5 * torch.randn((2 * Hk, hd), generator=g))))
    rows = (torch.randn((T, Hq + 2 * Hk, hd), generator=g) * spread).to(t)
    return rows, np.concatenate(([0], np.cumsum(lens))).tolist()


def parts(rows, Hq, Hk):
    return rows[:, :Hq], rows[:, Hq:Hq + Hk], rows[:, Hq + Hk:]


def check_prompt(dev, t, lens, Hq, Hk, hd, causal=True, scale=None, seed=0, size=1.0):
    rows, starts = prompts(seed + hd, lens, Hq, Hk, hd, t, size)
    q, k, v = parts(rows.to(dev), Hq, Hk)
    y = nnr_amd.prompt_attention(q, k, v, ints(dev, starts), causal=causal, scale=scale)
    assert y.shape == q.shape and y.dtype == t
    sc = np.float32(hd ** -0.5 if scale is None else scale).item()
    near(y, *R.prompt(*parts(rows, Hq, Hk), starts, sc, causal), t)
    return y


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("lens,Hq,Hk", [
    ([1], 1, 1), ([2], 4, 1), ([0, 3, 0, 1], 2, 2), ([31, 33], 3, 1), ([64, 32, 65], 2, 2), ([127, 1, 128, 129], 4, 4),
    ([200, 0, 61], 12, 4), ([300], 8, 1), ([5] * 70, 2, 1), ([1] * 130, 1, 1), ([513], 5, 1)])
def test_prompt(dev, t, hd, lens, Hq, Hk):
    check_prompt(dev, t, lens, Hq, Hk, hd)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [64, 96, 128, 256])
def test_prompt_all_tokens(dev, t, hd):
    """Not causal: the last tile of every row ends inside a tile."""
    check_prompt(dev, t, [1, 63, 64, 65, 190], 4, 2, hd, causal=False)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0, 5.0])
def test_prompt_scales(dev, t, scale):
    check_prompt(dev, t, [150, 40], 4, 2, 64, scale=scale, seed=3)


@pytest.mark.parametrize("t", TYPES)
def test_prompt_long(dev, t):
    check_prompt(dev, t, [2100, 17, 1025], 2, 1, 128, seed=5)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_prompt_scores_grow(dev, t, hd):
    """Later keys score higher than all before by more than a weight's range: the maximum moves at every tile."""
    n = 400
    rows, starts = prompts(1, [n], 2, 2, hd, t)
    q, k, v = parts(rows, 2, 2)
    q[:], k[:] = 0, 0
    q[:, :, 0] = 1
    k[:, :, 0] = torch.arange(n).float()[:, None] * 2.0      # exact in every type up to 256; steps of 4 beyond in bf16
    y = nnr_amd.prompt_attention(q.to(dev), k.to(dev), v.to(dev), ints(dev, starts), scale=1.0)
    near(y, *R.prompt(q, k, v, starts, 1.0, True), t)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd,Hq,Hk,lens", [(256, 2, 1, [400, 33]), (256, 40, 40, [300, 300, 300]), (96, 2, 2, [400])])
def test_prompt_scores_grow_by_little(dev, t, hd, Hq, Hk, lens):
    """Scores that grow by 2^8 of a weight every 32 tokens (the maximum moves at some of the tiles, in some of the rows), over
    random ones; few blocks and more than the chip holds at once"""
    rows, starts = prompts(6, lens, Hq, Hk, hd, t)
    q, k, v = parts(rows, Hq, Hk)
    q[:, :, 0] = 1
    for b, n in enumerate(lens):
        k[starts[b]:starts[b + 1], :, 0] = (torch.arange(n) // 32).float()[:, None] * 5.5
    q[1::3, :, 0] = 0
    y = nnr_amd.prompt_attention(q.to(dev), k.to(dev), v.to(dev), ints(dev, starts), scale=1.0)
    near(y, *R.prompt(q, k, v, starts, 1.0, True), t)


@pytest.mark.parametrize("t", TYPES)
def test_prompt_large_values(dev, t):
    """The largest numbers of a type as values, whose sums pass them where their means do not"""
    rows, starts = prompts(2, [300], 2, 1, 64, t)
    q, k, v = parts(rows, 2, 1)
    v[:] = torch.finfo(t).max * (0.5 if t != torch.float16 else 1.0)
    y = nnr_amd.prompt_attention(q.to(dev), k.to(dev), v.to(dev), ints(dev, starts))
    near(y, *R.prompt(q, k, v, starts, 0.125, True), t)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [64, 96, 256])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), float("-inf")])
def test_prompt_unseen_values(dev, t, hd, what):
    """A NaN or infinity among the values: rows that do not see it are as without it, of the others that element alone
    is not finite; a token before and one behind a sequence have no effect either."""
    lens, Hq, Hk = [70, 200, 40], 4, 2
    rows, starts = prompts(4, lens, Hq, Hk, hd, t)
    q, k, v = parts(rows, Hq, Hk)
    sd = ints(dev, starts)
    clean = nnr_amd.prompt_attention(q.to(dev), k.to(dev), v.to(dev), sd).cpu()
    bad = v.clone()
    at = {0: 69, 1: starts[1] + 100, 2: starts[2] + 3}
    for b, tok in at.items():
        bad[tok, 1, 5 + b] = what
    y = nnr_amd.prompt_attention(q.to(dev), k.to(dev), bad.to(dev), sd).cpu()
    touched = torch.zeros(y.shape, dtype=torch.bool)
    for b, tok in at.items():
        touched[tok:starts[b + 1], 2:, 5 + b] = True
    assert torch.equal(y[~touched], clean[~touched])
    assert (y[touched].isnan() if what != what else y[touched] == what).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_prompt_unseen_values_of_many(dev, t, hd):
    """The same with more blocks than the chip holds at once (a block has more rows then)"""
    lens, H, at = [300] * 3, 100, 437
    rows, starts = prompts(7, lens, H, H, hd, t)
    q, k, v = (x.to(dev) for x in parts(rows, H, H))
    sd = ints(dev, starts)
    clean = nnr_amd.prompt_attention(q, k, v, sd)
    for what in (float("nan"), float("-inf")):
        bad = v.clone()
        bad[at, 60, 9] = what
        y = nnr_amd.prompt_attention(q, k, bad, sd)
        hit = torch.zeros(y.shape, dtype=torch.bool, device=dev)
        hit[at:600, 60, 9] = True
        assert torch.equal(y[~hit], clean[~hit])
        assert (y[hit].isnan() if what != what else y[hit] == what).all()


@pytest.mark.parametrize("t", TYPES)
def test_prompt_unseen_kinds(dev, t):
    """Infinities of both signs and NaNs side by side, beside values of both signs."""
    n, hd = 100, 64
    rows, starts = prompts(6, [n], 1, 1, hd, t)
    q, k, v = parts(rows, 1, 1)
    inf = float("inf")
    v[40, 0, 0], v[50, 0, 0] = inf, -inf
    v[41, 0, 1], v[45, 0, 1] = inf, inf
    v[42, 0, 2], v[60, 0, 2] = -inf, float("nan")
    y = nnr_amd.prompt_attention(q.to(dev), k.to(dev), v.to(dev), ints(dev, starts)).cpu()[:, 0].float()
    assert y[:40].isfinite().all() and y[:, 3:].isfinite().all()
    assert (y[40:50, 0] == inf).all() and y[50:, 0].isnan().all()
    assert (y[41:, 1] == inf).all() and y[40, 1].isfinite()
    assert (y[42:60, 2] == -inf).all() and y[60:, 2].isnan().all()


@pytest.mark.parametrize("t", TYPES)
def test_prompt_unseen_keys(dev, t):
    """A NaN, and the lowest number, among the keys: rows before it are as without it."""
    lens, hd = [130], 128
    rows, starts = prompts(8, lens, 2, 1, hd, t)
    q, k, v = parts(rows, 2, 1)
    sd = ints(dev, starts)
    clean = nnr_amd.prompt_attention(q.to(dev), k.to(dev), v.to(dev), sd).cpu()
    for what in (float("nan"), torch.finfo(t).min, float("inf")):
        bad = k.clone()
        bad[77] = what
        y = nnr_amd.prompt_attention(q.to(dev), bad.to(dev), v.to(dev), sd).cpu()
        assert torch.equal(y[:77], clean[:77])
        if what != what:
            assert y[77:].isnan().all()


@pytest.mark.parametrize("t", TYPES)
def test_prompt_rows_do_not_mix(dev, t):
    rows, starts = prompts(9, [90], 4, 2, 64, t)
    q, k, v = parts(rows, 4, 2)
    sd = ints(dev, starts)
    clean = nnr_amd.prompt_attention(q.to(dev), k.to(dev), v.to(dev), sd).cpu()
    q[33, 1] = float("nan")
    y = nnr_amd.prompt_attention(q.to(dev), k.to(dev), v.to(dev), sd).cpu()
    assert y[33, 1].isnan().all()
    y[33, 1] = clean[33, 1]
    assert torch.equal(y, clean)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [64, 256])
def test_prompt_other_tokens(dev, t, hd):
    """Tokens before the first sequence and behind the last: not read (they hold NaN), not written."""
    lens = [10, 50, 33, 40]
    rows, starts = prompts(10, lens, 2, 1, hd, t)
    rows[:10], rows[-40:] = float("nan"), float("nan")
    q, k, v = parts(rows.to(dev), 2, 1)
    y = torch.full(q.shape, 7.0, dtype=t, device=dev)
    starts = starts[1:-1]
    assert nnr_amd.prompt_attention(q, k, v, ints(dev, starts), y=y) is y
    assert (y[:10] == 7).all() and (y[-40:] == 7).all()
    ref, tol = R.prompt(*parts(rows, 2, 1), starts, np.float32(hd ** -0.5).item(), True)
    near(y[10:-40], ref[10:-40], tol[10:-40], t)


def test_prompt_nothing(dev):
    q, k = torch.randn((5, 2, 64), device=dev), torch.randn((5, 1, 64), device=dev)
    y = torch.full((5, 2, 64), 3.0, device=dev)
    for starts in ([0], [2, 2], [0, 0, 0], [5, 5]):
        nnr_amd.prompt_attention(q, k, k, ints(dev, starts), y=y)
        assert (y == 3).all()
    assert nnr_amd.prompt_attention(q[:0], k[:0], k[:0], ints(dev, [0, 0])).shape == (0, 2, 64)


def test_prompt_many_sequences(dev):
    """More sequences than a wave looks at in one step, or two, empty ones among them"""
    rng = np.random.default_rng(1)
    lens = rng.integers(0, 4, 5000)
    rows, starts = prompts(11, lens.tolist(), 1, 1, 64, torch.float16)
    q, k, v = parts(rows.to(dev), 1, 1)
    y = nnr_amd.prompt_attention(q, k, v, ints(dev, starts))
    near(y, *R.prompt(*parts(rows, 1, 1), starts, 0.125, True), torch.float16)


@pytest.mark.parametrize("t", TYPES)
def test_prompt_layouts(dev, t):
    """Slices at odd places, heads that are not dense, q in place of y, another stream."""
    Hq, Hk, hd = 4, 2, 64
    rows, starts = prompts(12, [77, 20], Hq, Hk, hd, t)
    sd = ints(dev, starts)
    q, k, v = (x.contiguous() for x in parts(rows.to(dev), Hq, Hk))
    want = nnr_amd.prompt_attention(q, k, v, sd)
    odd = torch.empty(k.numel() + 1, dtype=t, device=dev)[1:].view(k.shape)
    odd.copy_(k)
    apart = v.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(nnr_amd.prompt_attention(q, odd, apart, sd), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = nnr_amd.prompt_attention(q, k, v, sd, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(got, want)
    assert nnr_amd.prompt_attention(q, k, v, sd, y=q) is q and torch.equal(q, want)


def test_prompt_graph(dev):
    """Captured; replayed with other lengths and values."""
    rows, _ = prompts(13, [300], 4, 2, 128, torch.bfloat16)
    rows = rows.to(dev)
    q, k, v = parts(rows, 4, 2)
    starts = ints(dev, [0, 100, 300])
    y = torch.zeros((300, 4, 128), dtype=torch.bfloat16, device=dev)
    nnr_amd.prompt_attention(q, k, v, starts, y=y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        nnr_amd.prompt_attention(q, k, v, starts, y=y)
    for middle in (150, 1, 299):
        starts[1] = middle
        rows.mul_(0.9)
        want = nnr_amd.prompt_attention(q, k, v, starts)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_prompt_refuses(dev):
    f = nnr_amd.prompt_attention
    q, k, s = torch.zeros((6, 4, 64), device=dev), torch.zeros((6, 2, 64), device=dev), ints(dev, [0, 6])
    for bad in (lambda: f(q, k, k[:5], s), lambda: f(q[:5], k, k, s), lambda: f(q, k, k.half(), s), lambda: f(q, k, k, s.long()),
                lambda: f(q, k, k, s[:0]), lambda: f(q, k, k, s.cpu()), lambda: f(q, k.cpu(), k, s), lambda: f(q[0], k, k, s),
                lambda: f(q, k, k, s, y=q[:5]), lambda: f(q, k, k, s, y=q.half())):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: f(q[:, :3], k, k, s), lambda: f(q[..., :32], k[..., :32], k[..., :32], s), lambda: f(k, k, k, s, y=k)):
        with pytest.raises(nnr_amd.NnrHipError):
            bad()
    with pytest.raises(TypeError):
        f(q.double(), k.double(), k.double(), s)


# ---------------------------------------------------------------------------
# trees of drafts

def tables(rng, batch, per, spare):
    order = rng.permutation(batch * per + spare).astype(np.int32)
    return torch.from_numpy(order[:batch * per].reshape(batch, per).copy()), len(order), torch.from_numpy(order[batch * per:].copy())


def tokens(seed, B, S, H, hd, t):
    g = gen(seed)
    return [(torch.randn((B, S, H, hd), generator=g) * torch.exp(0.5 * torch.randn((H, hd), generator=g))).to(t) for _ in "kv"]


def cache_of(dev, *args, **kw):
    c = nnr_amd.KVCache(*args, **kw)
    c.data.fill_(255)     # what memory may hold: NaN scales among it
    return c


def check_tree(dev, t, bits, hd, H, G, tree, lens, prefix, page, seed=0, vscale=None, per=None):
    """tree bool [S, S] or [B, S, S]"""
    B, S = len(lens), tree.shape[-1]
    rng = np.random.default_rng(seed + hd)
    pre_pages = -(-prefix // page)
    per = max(1, max(-(-n // page) for n in lens)) if per is None else per
    table, pages, spare = tables(rng, B, per, pre_pages + 1)
    cache, td, ld = cache_of(dev, pages, H, hd, page_size=page, bits=bits), table.to(dev), ints(dev, lens)
    n = max(max(lens), 1)
    k, v = tokens(seed + 1, B, n, H, hd, t)
    if vscale is not None:
        v *= vscale(B, n).to(t)
    cache.write(k.to(dev), v.to(dev), td, ld)
    pt = spare[:pre_pages].to(dev)
    pk, pv = tokens(seed + 2, 1, prefix, H, hd, t)
    if prefix:
        cache.write(pk.to(dev), pv.to(dev), pt[None], ints(dev, [prefix]))
    q = torch.randn((B, S, H * G, hd), generator=gen(seed + 3)).to(t)
    args = (q.to(dev), td, ld)
    y = cache.attention(*args, prefix_table=pt, prefix_len=prefix, tree=tree.to(dev)).cpu()
    sc = np.float32(hd ** -0.5).item()
    cap = per * page
    for b in range(B):
        have = min(lens[b], cap)
        line = tree[b] if tree.dim() == 3 else tree
        sees = torch.ones((S, prefix + max(have, 0)), dtype=torch.bool)
        for j in range(S):
            at = lens[b] - S + j
            if 0 <= at < have:
                sees[:, prefix + at] = line[:, j]
        for h in range(H):
            kx, vx = (torch.cat((D.quantize(p[0, :, h], bits)[0], D.quantize(x[b, n - lens[b]:n - lens[b] + have, h], bits)[0]))
                      for p, x in ((pk, k), (pv, v)))
            ref, w, tol = R.attend(q[b, :, h * G:(h + 1) * G], kx, vx, sc, sees, R.CACHE_FLOOR[t])
            # a row's queries meet the keys with a power of two in common
            top = q[b, :, h * G:(h + 1) * G].double().abs().amax((1, 2))[:, None, None]
            low = 2.0 ** -39 * top * (kx.abs().sum(-1).amax() if len(kx) else 0.0) * sc
            near(y[b, :, h * G:(h + 1) * G], ref, R.rounded(ref, w, tol + 2 * low * w, t, R.CACHE_WEIGHTS[t]), t)
    return y


def random_tree(rng, S, B=None):
    m = np.zeros((B or 1, S, S), bool)
    for b in range(B or 1):
        for i in range(S):
            m[b, i, i] = True
            if i:
                m[b, i] |= m[b, rng.integers(max(0, i - 4), i)]
    return torch.from_numpy(m if B else m[0])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd,H,G,S,lens,prefix,page,each", [
    (64, 1, 1, 1, [1, 40], 0, 32, False), (64, 2, 4, 3, [3, 35, 64], 0, 32, True), (128, 1, 4, 15, [15, 200, 47], 70, 64, True),
    (96, 2, 3, 7, [7, 33, 90], 0, 64, False), (128, 2, 2, 64, [64, 97, 300], 100, 64, True), (256, 1, 2, 9, [100, 9], 33, 32, False),
    (96, 1, 4, 40, [40, 55], 31, 32, True), (256, 1, 1, 33, [64, 41], 0, 64, True), (64, 1, 8, 130, [700, 131], 40, 128, False),
    (128, 1, 8, 2, [5000], 0, 64, True)])
def test_tree(dev, t, bits, hd, H, G, S, lens, prefix, page, each):
    rng = np.random.default_rng(S)
    check_tree(dev, t, bits, hd, H, G, random_tree(rng, S, len(lens) if each else None), lens, prefix, page, seed=S)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("S,prefix", [(5, 0), (5, 40), (40, 0), (40, 40)])
def test_tree_any_relation(dev, t, bits, S, prefix):
    """Drafts that see later ones, not themselves, or none; padding at the front; lengths behind the last page; a length
    of 0. A row that sees nothing at all gives 0."""
    rng = np.random.default_rng(S + prefix)
    tree = torch.from_numpy(rng.random((5, S, S)) < 0.3)
    tree[:, 1] = False
    lens = [S, S - 3, S + 50, 1, 0]
    y = check_tree(dev, t, bits, 64, 2, 2, tree, lens, prefix, 32, seed=S)
    if not prefix:
        assert not y[0, 1].any() and not y[4].any()
    check_tree(dev, t, bits, 64, 2, 2, tree, lens, prefix, 32, seed=S, per=2)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("S", [3, 40])
def test_tree_scales_far_apart(dev, t, bits, S):
    """Values of 1e3 that some drafts do not see beside such of 1e-3 (rows that are computed again)"""
    rng = np.random.default_rng(3)
    tree = random_tree(rng, S)
    tree[2] = False
    tree[2, 2] = True

    def vscale(B, n):
        x = torch.full((B, n, 1, 1), 1e-3)
        x[:, n - S + 1] = 3e4 if t == torch.float16 else 1e6
        return x
    check_tree(dev, t, bits, 64, 1, 2, tree, [S, 90], 0, 32, seed=9, vscale=vscale)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd", [64, 96, 128])
def test_tree_scales_far_apart_in_parts(dev, t, bits, hd):
    """As before, behind a prefix, over several parts of prefix and sequence, with more rows than a block has"""
    S = 40
    tree = random_tree(np.random.default_rng(4), S)
    tree[:, 1] = False
    tree[1, 1] = tree[5, 1] = True

    def vscale(B, n):
        x = torch.full((B, n, 1, 1), 1e-3)
        x[:, n - S + 1] = 3e4 if t == torch.float16 else 1e6
        return x
    check_tree(dev, t, bits, hd, 1, 4, tree, [S, 700, 230], 300, 64, seed=11, vscale=vscale)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("S", [4, 33])
def test_tree_of_a_chain_is_causal(dev, bits, S):
    """A tree without branches gives what the causal call gives. Both are within a tolerance of the 64-bit result, so
    they are within twice that of each other (they may join a different number of tiles at a time)."""
    B, H, G, hd, page = 3, 2, 4, 128, 64
    table, pages, spare = tables(np.random.default_rng(1), B, 5, 3)
    cache, td, ld = cache_of(dev, pages, H, hd, page_size=page, bits=bits), table.to(dev), ints(dev, [300, S, 77])
    k, v = tokens(1, B, 300, H, hd, torch.float16)
    cache.write(k.to(dev), v.to(dev), td, ld)
    q = torch.randn((B, S, H * G, hd), generator=gen(5)).half().to(dev)
    chain = torch.ones((S, S), dtype=torch.bool, device=dev).tril()
    causal, want = cache.attention(q, td, ld).cpu(), cache.attention(q, td, ld, tree=chain)
    for b, n in enumerate((300, S, 77)):
        sees = torch.cat((torch.ones((S, n - S), dtype=torch.bool), chain.cpu()), -1)
        for h in range(H):
            at = (b, slice(None), slice(h * G, (h + 1) * G))
            kx, vx = (D.quantize(x[b, 300 - n:, h], bits)[0] for x in (k, v))
            ref, w, tol = R.attend(q[at].cpu(), kx, vx, np.float32(hd ** -0.5).item(), sees, R.CACHE_FLOOR[torch.float16])
            near(want[at], causal[at].double(), 2 * R.rounded(ref, w, tol, torch.float16, R.CACHE_WEIGHTS[torch.float16]),
                 torch.float16)
    assert torch.equal(cache.attention(q, td, ld, tree=chain.expand(B, S, S)), want)
    assert torch.equal(cache.attention(q, td, ld, tree=chain[None].repeat(B, 1, 1)), want)
    # a mask that is a view, another stream, a workspace of the call's
    wide = torch.zeros((S, 2 * S), dtype=torch.bool, device=dev)
    wide[:, ::2] = chain
    ws = torch.empty(cache.attention_workspace(B, S, H * G, 5, dtype=torch.float16, tree=True), dtype=torch.uint8, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = cache.attention(q, td, ld, tree=wide[:, ::2], workspace=ws, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(got, want)


def test_tree_graph(dev):
    """Captured; replayed with other lengths and another tree."""
    B, S, H, G, hd = 2, 12, 1, 4, 64
    table, pages, _ = tables(np.random.default_rng(2), B, 4, 1)
    cache, td, ld = cache_of(dev, pages, H, hd, page_size=64), table.to(dev), ints(dev, [200, 100])
    k, v = tokens(3, B, 256, H, hd, torch.bfloat16)
    cache.write(k.to(dev), v.to(dev), td, ints(dev, [256, 256]))
    q = torch.randn((B, S, H * G, hd), generator=gen(5)).bfloat16().to(dev)
    tree = random_tree(np.random.default_rng(4), S).to(dev)
    y = cache.attention(q, td, ld, tree=tree)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = cache.attention(q, td, ld, tree=tree)
    for i in range(3):
        ld += 9
        tree.copy_(random_tree(np.random.default_rng(40 + i), S))
        want = cache.attention(q, td, ld, tree=tree)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_tree_refuses(dev):
    cache = nnr_amd.KVCache(2, 1, 64, page_size=32, device=dev)
    q, td, ld = torch.zeros((2, 3, 2, 64), device=dev), ints(dev, [[0], [1]]), ints(dev, [5, 6])
    ok = torch.ones((3, 3), dtype=torch.bool, device=dev)
    for bad in (ok[:2], ok.int(), ok.cpu(), ok[None], ok.expand(3, 3, 3), ok[0]):
        with pytest.raises(ValueError):
            cache.attention(q, td, ld, tree=bad)


# ---------------------------------------------------------------------------
# pages and tokens moved

@pytest.mark.parametrize("bits,hd,H,page,layers,n", [(8, 128, 8, 64, 1, 1), (4, 96, 3, 32, 3, 7), (8, 64, 1, 32, 2, 20),
                                                     (4, 256, 2, 4096, 1, 3), (8, 96, 5, 128, 70, 2)])
def test_copy_pages(dev, bits, hd, H, page, layers, n):
    pages = 2 * n + 3
    rng = np.random.default_rng(n)
    caches = [nnr_amd.KVCache(pages, H, hd, page_size=page, bits=bits) for _ in range(layers)]
    for i, c in enumerate(caches):
        c.data.copy_(torch.randint(0, 256, c.data.shape, generator=gen(i), dtype=torch.uint8))
    want = [c.data.view(pages, -1).clone() for c in caches]
    order = rng.permutation(pages).astype(np.int32)
    src, dst = order[:n].copy(), order[n:2 * n].copy()
    src[n // 2] = src[0]      # one source for two
    for w in want:
        w[torch.from_numpy(dst).long()] = w[torch.from_numpy(src).long()]
    # pairs without a page, and of a page with itself
    src = np.concatenate((src, [-1, pages, 0, 1, order[-1]])).astype(np.int32)
    dst = np.concatenate((dst, [order[-1], order[-1], -5, 2 ** 31 - 1, order[-1]])).astype(np.int32)
    nnr_amd.copy_pages(caches if layers > 1 else caches[0], ints(dev, src), ints(dev, dst))
    for c, w in zip(caches, want):
        assert torch.equal(c.data.view(pages, -1), w)


def test_copy_pages_many(dev):
    """More pairs than a grid's second dimension holds"""
    n = 70000
    cache = nnr_amd.KVCache(2 * n, 1, 64, page_size=32, bits=4)
    data = cache.data.view(2 * n, -1)
    data.copy_(torch.randint(0, 256, data.shape, dtype=torch.uint8, device=dev))
    want = data[:n].clone()
    i = torch.arange(n, dtype=torch.int32, device=dev)
    nnr_amd.copy_pages(cache, i, i + n)
    assert torch.equal(data[n:], want) and torch.equal(data[:n], want)
    nnr_amd.copy_pages(cache, i[:0], i[:0])


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd,H,page,layers", [(64, 1, 32, 1), (96, 3, 64, 2), (128, 2, 32, 66), (256, 1, 128, 1)])
def test_move_tokens(dev, t, bits, hd, H, page, layers):
    """Permutations, moves to the front, sequences that move fewer, tokens that are read twice; everything else stays."""
    rng = np.random.default_rng(hd)
    B, n, per = 4, 9, 3
    total = min(per * page, 90)
    table, pages, _ = tables(rng, B, per, 2)
    td, full = table.to(dev), ints(dev, [total] * B)
    caches, toks = [], []
    for i in range(layers):
        caches.append(cache_of(dev, pages, H, hd, page_size=page, bits=bits))
        toks.append(tokens(i, B, total, H, hd, t))
        caches[-1].write(toks[-1][0].to(dev), toks[-1][1].to(dev), td, full)
    src = np.stack([rng.permutation(total)[:n] for _ in range(B)])
    dst = np.stack([rng.permutation(src[0]), 20 + np.arange(n), rng.permutation(total)[:n], rng.permutation(total)[:n]])
    src[1] = 20 + np.sort(rng.permutation(40)[:n])
    src[2, 4] = src[2, 3]
    src[2, [0, 5]], dst[2, 6] = (-1, 2 ** 31 - 1), -2 ** 31
    src[3, 2:] = -1
    before = [c.data.clone() for c in caches]
    nnr_amd.move_tokens(caches, td, ints(dev, src), ints(dev, dst))
    for c, (k, v) in zip(caches, toks):
        ks, vs = c.read(total, td, full, t)
        for got, x in ((ks, k), (vs, v)):
            want = D.quantize(x, bits)[0].to(t)
            old = want.clone()
            for b in range(B):
                for i in range(n):
                    if 0 <= src[b, i] < per * page and dst[b, i] >= 0:
                        want[b, dst[b, i]] = old[b, src[b, i]]
            assert torch.equal(got.cpu(), want)
    # and back: a permutation undone leaves every byte as it was
    c = caches[0]
    c.data.copy_(before[0])
    s0, d0 = ints(dev, src[:1]), ints(dev, dst[:1])
    nnr_amd.move_tokens(c, td[:1], s0, d0)
    assert not torch.equal(c.data, before[0])
    nnr_amd.move_tokens(c, td[:1], d0, s0)
    assert torch.equal(c.data, before[0])


@pytest.mark.parametrize("bits", [8, 4])
def test_move_most_tokens(dev, bits):
    """128 tokens of a sequence, over pages one of which does not exist; no tokens at all"""
    H, hd, page = 2, 256, 64
    cache = cache_of(dev, 4, H, hd, page_size=page, bits=bits)
    td, full = ints(dev, [[2, -1, 0, 3]]), ints(dev, [256])
    k, v = tokens(1, 1, 256, H, hd, torch.float16)
    cache.write(k.to(dev), v.to(dev), td, full)
    src = torch.randperm(256, generator=gen(2))[:128].to(torch.int32)
    dst = torch.randperm(256, generator=gen(3))[:128].to(torch.int32)
    old = cache.read(256, td, full, torch.float16)
    nnr_amd.move_tokens(cache, td, src[None].to(dev), dst[None].to(dev))
    for got, x in zip(cache.read(256, td, full, torch.float16), old):
        want = x.clone()
        for s, d in zip(src.tolist(), dst.tolist()):
            if s // 64 != 1 and d // 64 != 1:
                want[0, d] = x[0, s]
        assert torch.equal(got, want)
    before = cache.data.clone()
    empty = torch.zeros((1, 0), dtype=torch.int32, device=dev)
    nnr_amd.move_tokens(cache, td, empty, empty)
    nnr_amd.move_tokens(cache, td[:0], src[:0, None].to(dev), src[:0, None].to(dev))
    assert torch.equal(cache.data, before)


def test_moves_in_a_graph(dev):
    """Both captured, replayed with other pages and positions, on caches that eager calls use between"""
    caches = [nnr_amd.KVCache(8, 2, 64, page_size=32, bits=4) for _ in range(2)]
    td, full = ints(dev, [[0, 1], [2, 3]]), ints(dev, [64, 64])
    src, dst = ints(dev, [0, 1]), ints(dev, [4, 5])
    fr, to = ints(dev, [[40, 50], [63, 62]]), ints(dev, [[33, 34], [40, 41]])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        nnr_amd.copy_pages(caches, src, dst)
        nnr_amd.move_tokens(caches, td, fr, to)
    for i in range(3):
        for c in caches:
            k, v = tokens(i, 2, 64, 2, 64, torch.float32)
            c.write(k.to(dev), v.to(dev), td, full)
        src.fill_(i), dst.copy_(ints(dev, [5 + i % 2, 7])), fr.sub_(1)
        want = [c.data.clone() for c in caches]
        graph.replay()
        torch.cuda.synchronize()
        got = [c.data.clone() for c in caches]
        for c, w in zip(caches, want):
            c.data.copy_(w)
        nnr_amd.copy_pages(caches, src, dst)
        nnr_amd.move_tokens(caches, td, fr, to)
        assert all(torch.equal(c.data, g) for c, g in zip(caches, got))


def test_moves_refuse(dev):
    a, b = nnr_amd.KVCache(4, 2, 64, page_size=32), nnr_amd.KVCache(4, 2, 64, page_size=32, bits=4)
    one, td = ints(dev, [0]), ints(dev, [[0, 1]])
    for bad in (lambda: nnr_amd.copy_pages([], one, one), lambda: nnr_amd.copy_pages([a, b], one, one),
                lambda: nnr_amd.copy_pages(a, one.long(), one), lambda: nnr_amd.copy_pages(a, one, ints(dev, [1, 2])),
                lambda: nnr_amd.copy_pages(a, one.cpu(), one), lambda: nnr_amd.copy_pages(a, one[None], one[None]),
                lambda: nnr_amd.move_tokens(a, td, one, one), lambda: nnr_amd.move_tokens(a, td, td, td[:, :1]),
                lambda: nnr_amd.move_tokens(a, td, td.repeat(2, 1), td.repeat(2, 1)),
                lambda: nnr_amd.move_tokens([a, b], td, td, td)):
        with pytest.raises(ValueError):
            bad()
    many = torch.zeros((1, 129), dtype=torch.int32, device=dev)
    for bad in (lambda: nnr_amd.copy_pages([a, a], one, one), lambda: nnr_amd.move_tokens([a, a], td, td, td),
                lambda: nnr_amd.move_tokens(a, td, many, many)):
        with pytest.raises(nnr_amd.NnrHipError):
            bad()


# ---------------------------------------------------------------------------
# together

@pytest.mark.parametrize("bits", [8, 4])
def test_a_step_with_drafts(dev, bits):
    """Prompts, then a tree of drafts whose accepted path moves to the front, then a fork: the next step's attention is that
    of a cache that was written token by token."""
    t, L, Hq, Hk, hd, page = torch.float16, 2, 8, 2, 64, 32
    rope = nnr_amd.RotaryEmbedding(hd, 1000, device=dev)
    lens, B = [40, 61], 2
    starts = ints(dev, [0, 40, 101])
    # parents and depths of 7 drafts; the path 0 - 2 - 5 is accepted
    parent, path = [-1, 0, 0, 1, 1, 2, 2], [0, 2, 5]
    S, tree, depth = len(parent), torch.eye(7, dtype=torch.bool), [0] * 7
    for i, p in enumerate(parent):
        if p >= 0:
            tree[i] |= tree[p]
            depth[i] = depth[p] + 1
    tree = tree.to(dev)
    caches = [nnr_amd.KVCache(12, Hk, hd, page_size=page, bits=bits) for _ in range(L)]
    plain = [nnr_amd.KVCache(12, Hk, hd, page_size=page, bits=bits) for _ in range(L)]
    td = ints(dev, [[0, 3, 5], [4, 1, 2]])
    g = gen(1)
    for layer in range(L):
        rows = torch.randn((101, Hq + 2 * Hk, hd), generator=g).to(t).to(dev)
        pos = torch.cat([torch.arange(n, dtype=torch.int32) for n in lens]).to(dev)
        q, k, v = (x[None] for x in parts(rows, Hq, Hk))
        rope(q, k, pos[None], out=(q, k))
        y = nnr_amd.prompt_attention(q[0], k[0], v[0], starts)
        ref, tol = R.prompt(q[0].cpu(), k[0].cpu(), v[0].cpu(), [0, 40, 101], 0.125, True)
        near(y, ref, tol, t)
        for c in (caches[layer], plain[layer]):
            for b, (s, e) in enumerate(((0, 40), (40, 101))):
                c.write(k[:, s:e], v[:, s:e], td[b:b + 1], ints(dev, [e - s]))
    now = ints(dev, lens)
    pos = now[:, None] + ints(dev, depth)
    accepted = []
    for layer in range(L):
        q, k = (torch.randn((B, S, h, hd), generator=g).to(t).to(dev) for h in (Hq, Hk))
        v = torch.randn((B, S, Hk, hd), generator=g).to(t).to(dev)
        q, k = rope(q, k, pos)
        caches[layer].write(k, v, td, now + S)
        y = caches[layer].attention(q, td, now + S, tree=tree)
        # each draft of the path as if its ancestors alone were written
        for i, d in enumerate(path):
            plain[layer].write(k[:, d:d + 1], v[:, d:d + 1], td, now + i + 1)
            alone = plain[layer].attention(q[:, d:d + 1], td, now + i + 1)
            assert (y[:, d:d + 1].float() - alone.float()).abs().max() <= 2 * 2.0 ** -11 * 4
    first = now[:, None]
    nnr_amd.move_tokens(caches, td, first + ints(dev, path), first + ints(dev, [0, 1, 2]))
    now = now + 3
    for a, b in zip(caches, plain):
        for x, z in zip(a.read(64, td, now, t), b.read(64, td, now, t)):
            assert torch.equal(x, z)
    # sequence 0 forked: its last page copied, the others shared
    nnr_amd.copy_pages(caches, td[0, 1:2], ints(dev, [9]))
    forked = torch.cat((td, ints(dev, [[0, 9, 10]])))
    lens3 = torch.cat((now, now[:1]))
    k, v = (torch.randn((3, 1, Hk, hd), generator=g).to(t).to(dev) for _ in "kv")
    q = torch.randn((3, 1, Hq, hd), generator=g).to(t).to(dev)
    for a, b in zip(caches, plain):
        a.write(k, v, forked, lens3 + 1)
        y = a.attention(q, forked, lens3 + 1)
        b.write(k[:2], v[:2], td, now + 1)
        assert torch.equal(y[:2], b.attention(q[:2], td, now + 1))
        b.write(k[2:], v[2:], td[:1], now[:1] + 1)
        assert torch.equal(y[2:], b.attention(q[2:], td[:1], now[:1] + 1))
