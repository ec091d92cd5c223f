"""Operators around a decoder's cache where a part, a page, a length or a step has its end: against float64,
like test_gpu_serving.py."""
import numpy as np
import pytest
import torch

import decode_ref as D
import nnr_amd
import serving_ref as R
from test_gpu_serving import TYPES, cache_of, gen, ints, near, parts, prompts, random_tree, tables, tokens

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# trees of drafts

def tree_parts(cache, batch, S, Hq, per, prefix, t, length):
    """Tiles [first, end) of a sequence's parts: the prefix's, then its own, in parts of equal length whose number the
    workspace tells."""
    size = cache.attention_workspace(batch, S, Hq, per, prefix, dtype=t, tree=True)
    count = max(1, size // (batch * S * Hq * (cache.head_dim * 4 + 8)))
    tiles = -(-prefix // 32) + -(-length // 32)
    each, more = divmod(tiles, count)
    ends = np.cumsum([each + (i < more) for i in range(count)]).tolist()
    return list(zip([0] + ends[:-1], ends))


def check_computed_again(dev, t, bits, hd, S, G, prefix, lens, far_pre, far_own, in_parts):
    """A few large values that no row gives weight to, beside such of 1e-3: rows of the parts that hold them are computed
    again in fp32. in_parts: those parts hold tokens of the prefix at the positions that drafts have in their sequence.
    The tree's first line hides all drafts but one."""
    H, page = 1, 32
    tree = random_tree(np.random.default_rng(4), S)
    B, pre_pages, per = len(lens), -(-prefix // page), max(-(-n // page) for n in lens)
    table, pages, spare = tables(np.random.default_rng(hd), B, per, pre_pages + 1)
    cache = cache_of(dev, pages, H, hd, page_size=page, bits=bits)
    for b, n in enumerate(lens if in_parts else []):
        found = False
        for first, end in tree_parts(cache, B, S, H * G, per, prefix, t, n):
            far = any(first <= p // 32 < end for p in far_pre) or any(first <= -(-prefix // 32) + p // 32 < end for p in far_own)
            found |= far and any(first <= p // 32 < end for p in range(n - S + 1, min(n, prefix)))
        assert found, "no part is computed again that the drafts' positions meet in the prefix"
    most = max(lens)
    k, v = tokens(1, B, most, H, hd, t)
    pk, pv = tokens(2, 1, prefix, H, hd, t)
    q = torch.randn((B, S, H * G, hd), generator=gen(3)).to(t)
    big = 3e4 if t == torch.float16 else 1e6
    q[..., 0] = 4
    small_v = [x * 1e-3 for x in (v, pv)]
    v[:], pv[:] = small_v
    for x, y, at in ((pk, pv, [(0, p) for p in far_pre]), (k, v, [(b, most - n + p) for b, n in enumerate(lens) for p in far_own])):
        for b, p in at:
            x[b, p], x[b, p, :, 0] = 0, -8 * hd ** 0.5      # a score 32 less than one of 0
            y[b, p] = big
    cache.write(k.to(dev), v.to(dev), table.to(dev), ints(dev, lens))
    pt = spare[:pre_pages].to(dev)
    cache.write(pk.to(dev), pv.to(dev), pt[None], ints(dev, [prefix]))
    y = cache.attention(q.to(dev), table.to(dev), ints(dev, lens), prefix_table=pt, prefix_len=prefix, tree=tree.to(dev)).cpu()
    sc = np.float32(hd ** -0.5).item()
    for b, n in enumerate(lens):
        sees = torch.ones((S, prefix + n), dtype=torch.bool)
        sees[:, prefix + n - S:] = tree
        kx, vx = (torch.cat([D.quantize(x, bits)[0] for x in (p[0, :, 0], o[b, most - n:, 0])]) for p, o in ((pk, k), (pv, v)))
        ref, w, tol = R.attend(q[b], kx, vx, sc, sees, 0.0)
        # Parts without a large value are the products': weights of 2^-11 and steps of small ones in parts of what
        # those hold at most, queries with a common power of two. (A part with one rounds no weight.)
        low = 2.0 ** -39 * q[b].double().abs().amax((1, 2))[:, None, None] * kx.abs().sum(-1).amax() * sc
        steps = len(vx) * R.CACHE_FLOOR[t] * max(x.double().abs().amax().item() for x in small_v)
        near(y[b], ref, R.rounded(ref, w, tol + 2 * low * w + steps, t, R.CACHE_WEIGHTS[t]), t)


FAR = [(300, [40, 200], [20, 180], []), (64, [40, 60], [], [5]), (300, [300, 290], [], [10]), (33, [41], [32], [])]


@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd", [64, 96, 128])
@pytest.mark.parametrize("prefix,lens,far_pre,far_own", FAR)
def test_tree_computed_again_behind_a_prefix(dev, t, bits, hd, prefix, lens, far_pre, far_own):
    check_computed_again(dev, t, bits, hd, 40, 4, prefix, lens, far_pre, far_own, True)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("t,hd,S,G", [(torch.float32, 64, 40, 4), (torch.float32, 256, 40, 2), (torch.bfloat16, 256, 40, 2),
                                      (torch.float16, 128, 3, 2), (torch.float32, 96, 3, 1), (torch.float16, 256, 5, 3)])
@pytest.mark.parametrize("prefix,lens,far_pre,far_own", FAR)
def test_tree_computed_again_elsewhere(dev, bits, t, hd, S, G, prefix, lens, far_pre, far_own):
    """The same of other types, wide heads and few rows, whose prefix is a block's of its own"""
    check_computed_again(dev, t, bits, hd, S, G, prefix, lens, far_pre, far_own, False)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("S", [2, 40])
def test_tree_over_a_cache_without_pages(dev, t, bits, hd, S):
    """Nothing to see, and no memory behind the cache: zeros. So it is with lengths of 0 and tables without columns."""
    q, tree = torch.randn((2, S, 4, hd), generator=gen(1)).to(t).to(dev), torch.ones((S, S), dtype=torch.bool, device=dev)
    none = nnr_amd.KVCache(0, 2, hd, page_size=32, bits=bits, device=dev)
    for per in (0, 1, 40):
        for prefix in (0, 70):
            y = none.attention(q, ints(dev, [[0] * per] * 2).view(2, per), ints(dev, [S, 1000]), prefix_table=ints(dev, [0, 0, 0]),
                               prefix_len=prefix, tree=tree)
            assert not y.any()
    some = cache_of(dev, 3, 2, hd, page_size=32, bits=bits)
    assert not some.attention(q, ints(dev, [[0], [1]]), ints(dev, [0, -5]), tree=tree).any()
    assert not some.attention(q, ints(dev, [[], []]).view(2, 0), ints(dev, [S, 9]), tree=tree).any()


# ---------------------------------------------------------------------------
# attention of prompts

@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n", [1, 3])
def test_prompt_tokens_far_apart(dev, t, n):
    """Tokens at steps past 2^22 elements: the last ones of long sequences. A single token's step says nothing."""
    S, H, hd = 1060, 32, 128
    x = torch.zeros((n, S, 3 * H, hd), dtype=t, device=dev)
    x[:, -1] = torch.randn((n, 3 * H, hd), generator=gen(n)).to(t).to(dev)
    q, k, v = (x[:, -1, i * H:(i + 1) * H] for i in range(3))
    assert q.stride(0) > 1 << 22
    starts = ints(dev, [0, n])
    want = nnr_amd.prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), starts)
    assert torch.equal(nnr_amd.prompt_attention(q, k, v, starts), want)
    near(want, *R.prompt(q.cpu(), k.cpu(), v.cpu(), [0, n], np.float32(hd ** -0.5).item(), True), t)
    if n == 1:
        assert torch.equal(want, v)
        y = q[0, :, :].unsqueeze(0)      # in place
        assert nnr_amd.prompt_attention(y, k, v, starts, y=y) is y and torch.equal(y, want)


@pytest.mark.parametrize("t", TYPES)
def test_prompt_of_one_token_many_heads(dev, t):
    """A row of more than 2^22 elements is no step either."""
    q, k, v = torch.randn((3, 1, 17000, 256), device=dev).to(t).unbind(0)
    assert torch.equal(nnr_amd.prompt_attention(q, k, v, ints(dev, [0, 1])), v)


# ---------------------------------------------------------------------------
# rotary positions

@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("lay", ["part", "tokens first", "part of tokens first", "side by side"])
def test_rotary_in_place_of_rows(dev, t, lay):
    """Queries and keys of one projection's output turned in place: its first tokens of a longer buffer, or with tokens
    before sequences in memory, or two such. What is not theirs stays."""
    B, S, most, Hq, Hk, hd = 3, 5, 9, 4, 2, 64
    rope = nnr_amd.RotaryEmbedding(hd, 100, device=dev)
    width = (Hq + 2 * Hk) * hd
    whole = torch.randn((2, B, most, width), generator=gen(1)).to(t).to(dev)
    if lay == "part":
        rows = whole[0, :, 2:2 + S]
    elif lay == "side by side":      # sequences a token's step apart from each other
        rows = whole[0].reshape(-1)[:S * B * width].view(S, B, width).transpose(0, 1)
    else:
        rows = whole[0].view(most, B, width).transpose(0, 1)[:, :S] if lay == "tokens first" else \
            whole.view(-1)[:most * 2 * B * width].view(most, 2 * B, width).transpose(0, 1)[1:1 + B, 1:1 + S]
    pos = torch.randint(0, 100, (B, S), generator=gen(2)).to(torch.int32).to(dev)
    q, k = rows[..., :Hq * hd].unflatten(-1, (Hq, hd)), rows[..., Hq * hd:(Hq + Hk) * hd].unflatten(-1, (Hk, hd))
    want, before = rope(q, k, pos), whole.clone()
    f, m = R.frequencies(hd, 10000.0)
    for x, y in zip((q, k), want):
        near(y, *R.rotate(x.cpu(), pos.cpu(), f, m, False, 100), t)
    out = rope(q, k, pos, out=(q, k))
    assert out[0] is q and torch.equal(q, want[0]) and torch.equal(k, want[1])
    q.zero_(), k.zero_()
    after = whole.clone()
    whole.copy_(before)
    q.zero_(), k.zero_()
    assert torch.equal(whole, after)      # but for theirs as before


def test_rotary_refuses_rows_that_meet(dev):
    """Of a longer buffer too: keys' rows that begin within queries', a step that is no multiple of the other."""
    rope = nnr_amd.RotaryEmbedding(64, 100, device=dev)
    buffer = torch.zeros(4000, device=dev)
    pos = ints(dev, [[0, 1, 2]] * 2)
    at = lambda first, heads, bs, ts: buffer.as_strided((2, 3, heads, 64), (bs, ts, 64, 1), first)
    q, k = at(0, 2, 5 * 192, 192), at(128, 1, 5 * 192, 192)
    assert rope(q, k, pos, out=(q, k))[0] is q
    for k in (at(64, 1, 5 * 192, 192), at(127, 1, 5 * 192, 192), at(129, 1, 5 * 192, 192), at(128, 1, 5 * 192 + 64, 192)):
        with pytest.raises(nnr_amd.NnrHipError):
            rope(q, k, pos, out=(q, k))


@pytest.mark.parametrize("t,e", [(torch.float32, e) for e in (-95, -105, -126)] + [(torch.bfloat16, e) for e in (-95, -110, -126)] +
                         [(torch.float16, e) for e in (-14, -23)])
@pytest.mark.parametrize("hd,Hq,Hk,lens", [(64, 2, 1, [300, 20]), (128, 4, 2, [150]), (256, 2, 1, [70, 3]), (256, 40, 40, [90] * 4)])
def test_prompt_small_values(dev, t, e, hd, Hq, Hk, lens):
    """Values whose weighted sums are small. Sums are of 2^-30 p v in fp32 and bf16: steps of the smallest fp32 numbers,
    2^-149, are 2^-119 of a result (its weights' total is 1 and more). A key rounds, or cuts, its product and a sum, a tile of
    32 the sums once more, and joined groups of waves a few times."""
    rows, starts = prompts(hd, lens, Hq, Hk, hd, t)
    q, k, v = parts(rows, Hq, Hk)
    v[:] = torch.ldexp(1 + torch.rand(v.shape, generator=gen(5), dtype=torch.float64), torch.tensor(e)).to(t)
    y = nnr_amd.prompt_attention(q.to(dev), k.to(dev), v.to(dev), ints(dev, starts))
    ref, tol = R.prompt(q, k, v, starts, np.float32(hd ** -0.5).item(), True)
    if t != torch.float16:
        tol = tol + (2.25 * max(lens) + 8) * 2.0 ** -119
    near(y, ref, tol, t)
    if e >= -95:      # hardly more than such results round anyway (fp16's of 2^-23 to half of its least step, 2^-25)
        assert ((y.cpu().double() - ref).abs() <= ref * (D.HALF[t] + R.PROMPT_WEIGHTS[t] + 2.0 ** -17) + D.TINY[t]).all()


# ---------------------------------------------------------------------------
# nothing to do

def test_empty_calls(dev):
    """No sequences (with a tree that is expanded over them), no tokens, no heads of queries or keys"""
    cache = nnr_amd.KVCache(2, 1, 64, page_size=32, device=dev)
    tree = torch.ones((3, 3), dtype=torch.bool, device=dev)
    q, td, ld = torch.zeros((2, 3, 2, 64), device=dev), ints(dev, [[0], [1]]), ints(dev, [5, 6])
    for mask in (tree, tree.expand(0, 3, 3), tree.repeat(0, 1, 1)):
        assert cache.attention(q[:0], td[:0], ld[:0], tree=mask).shape == (0, 3, 2, 64)
    for mask in (tree[:0, :0], tree[:0, :0].expand(2, 0, 0)):
        assert cache.attention(q[:, :0], td, ld, tree=mask).shape == (2, 0, 2, 64)
    rope, pos = nnr_amd.RotaryEmbedding(64, 100, device=dev), ints(dev, [[1, 2, 3], [4, 5, 6]])
    k = torch.randn((2, 3, 1, 64), device=dev)
    want = rope(q, k, pos)[1]
    for inplace in (False, True):
        x = k.clone()
        none, y = rope(q[:, :, :0], x, pos, out=(q[:, :, :0], x) if inplace else None)
        assert none.shape == (2, 3, 0, 64) and torch.equal(y, want)
        x = k.clone()
        assert torch.equal(rope(x, q[:, :, :0], pos, out=(x, q[:, :, :0]) if inplace else None)[0], want)
    assert rope(q[:0], k[:0], pos[:0])[0].shape == (0, 3, 2, 64) and rope(q[:, :0], k[:, :0], pos[:, :0])[1].shape == (2, 0, 1, 64)


# ---------------------------------------------------------------------------
# large sizes, results in place

@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("S", [3, 40])
def test_tree_in_place(dev, t, bits, S):
    """Rows that are computed again read their queries a second time, when others' results lie where queries were."""
    B, H, G, hd, page = 2, 2, 4, 64, 32
    table, pages, _ = tables(np.random.default_rng(S), B, 3, 1)
    cache, td, ld = cache_of(dev, pages, H, hd, page_size=page, bits=bits), table.to(dev), ints(dev, [S, 90])
    k, v = tokens(1, B, 96, H, hd, t)
    v *= 1e-3
    v[:, 96 - S + 1] = 1e4
    cache.write(k.to(dev), v.to(dev), td, ld)
    q = torch.randn((B, S, H * G, hd), generator=gen(2)).to(t).to(dev)
    tree = random_tree(np.random.default_rng(3), S)
    tree[2:, 1] = False
    want = cache.attention(q, td, ld, tree=tree.to(dev))
    assert cache.attention_workspace(B, S, H * G, 3, dtype=t, tree=True) == 0
    assert cache.attention(q, td, ld, tree=tree.to(dev), y=q) is q and torch.equal(q, want)


@pytest.mark.parametrize("t", [torch.float32, torch.float16])
@pytest.mark.parametrize("S,n", [(4096, 4096), (1000, 1777)])
def test_tree_of_many_drafts(dev, t, S, n):
    """As many as a tree may have: a chain, against the causal call, both within a tolerance of the 64-bit result."""
    H, G, hd, page, bits = 1, 2, 64, 128, 8
    per = -(-n // page)
    table, pages, _ = tables(np.random.default_rng(1), 1, per, 2)
    cache, td, ld = cache_of(dev, pages, H, hd, page_size=page, bits=bits), table.to(dev), ints(dev, [n])
    k, v = tokens(1, 1, n, H, hd, t)
    cache.write(k.to(dev), v.to(dev), td, ld)
    q = torch.randn((1, S, H * G, hd), generator=gen(2)).to(t)
    chain = torch.ones((S, S), dtype=torch.bool).tril()
    y = cache.attention(q.to(dev), td, ld, tree=chain.to(dev))
    some = torch.tensor([0, 1, 31, 64, S // 2, S - 2, S - 1])
    sees = torch.cat((torch.ones((len(some), n - S), dtype=torch.bool), chain[some]), -1)
    kx, vx = (D.quantize(x[0, :, 0], bits)[0] for x in (k, v))
    ref, w, tol = R.attend(q[0, some], kx, vx, np.float32(hd ** -0.5).item(), sees, R.CACHE_FLOOR[t])
    low = 2.0 ** -39 * q.double().abs().amax() * kx.abs().sum(-1).amax() * hd ** -0.5
    tol = R.rounded(ref, w, tol + 2 * low * w, t, R.CACHE_WEIGHTS[t])
    near(y[0, some.to(dev)], ref, tol, t)
    near(cache.attention(q.to(dev), td, ld)[0, some.to(dev)], ref, tol, t)


@pytest.mark.parametrize("bits", [8, 4])
def test_cache_past_32_bits(dev, bits):
    """Pages whose bytes begin past 2^32: written, copied, moved within and attended to as those at the front are."""
    H, hd, page, t = 8, 128, 4096, torch.float16
    size = 2 * H * page * (hd * bits // 8 + 2 * (1 if bits == 8 else hd // 32))
    pages = (5 << 30) // size
    far = nnr_amd.KVCache(pages, H, hd, page_size=page, bits=bits, device=dev)
    near_ = nnr_amd.KVCache(4, H, hd, page_size=page, bits=bits, device=dev)
    assert (pages - 2) * size > 1 << 32
    k, v = (torch.randn((1, 5000, H, hd), generator=gen(i)).to(t).to(dev) for i in (1, 2))
    ld, S = ints(dev, [5000]), 40
    q, tree = torch.randn((1, S, 2 * H, hd), generator=gen(3)).to(t).to(dev), random_tree(np.random.default_rng(1), S).to(dev)
    at = {}
    for c, own, to in ((near_, [0, 1], [2, 3]), (far, [pages - 1, 2], [pages - 2, pages - 3])):
        td = ints(dev, [own])
        c.write(k, v, td, ld)
        nnr_amd.copy_pages(c, ints(dev, own), ints(dev, to))
        moved = ints(dev, [[4990, 7, 4100]]), ints(dev, [[4970, 4971, 8]])
        nnr_amd.move_tokens(c, ints(dev, [to]), *moved)
        at[c] = [c.attention(q, ints(dev, [x]), ld, tree=tree) for x in (own, to)] + \
            [x for p in (own, to) for x in c.read(5000, ints(dev, [p]), ld, t)]
    assert all(torch.equal(a, b) for a, b in zip(at[near_], at[far])) and not torch.equal(at[far][0], at[far][1])


def test_prompts_past_32_bits(dev):
    """Tokens whose elements begin past 2^32, of queries, keys and values and of results"""
    T, H, hd, t = 1_200_000, 16, 256, torch.bfloat16
    rows = torch.empty((T, 3 * H, hd), dtype=t, device=dev)
    rows[-900:] = torch.randn((900, 3 * H, hd), generator=gen(1)).to(t).to(dev)
    y = torch.empty((T, H, hd), dtype=t, device=dev)
    y[-1000:] = 7
    q, k, v = rows[:, :H], rows[:, H:2 * H], rows[:, 2 * H:]
    nnr_amd.prompt_attention(q, k, v, ints(dev, [T - 900, T - 300, T - 299, T]), y=y)
    want = nnr_amd.prompt_attention(q[-900:], k[-900:], v[-900:], ints(dev, [0, 600, 601, 900]))
    assert (y[-1000:-900] == 7).all()
    near(y[-300:, :2], *R.prompt(*(x[-300:, :2].cpu() for x in (q, k, v)), [0, 1, 300], 1 / 16, True), t)
    # (other numbers of blocks, and so other groups of waves: twice the rounding of weights, of values at most, and of results)
    assert ((y[-900:].float() - want.float()).abs() <= 2.0 ** -7 * (v[-900:].abs().max() + want.float().abs())).all()


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_prompt_of_a_long_document(dev, t):
    n, hd = 70001, 64
    q, k, v = (torch.randn((n, 1, hd), generator=gen(i)).to(t) for i in range(3))
    y = nnr_amd.prompt_attention(*(x.to(dev) for x in (q, k, v)), ints(dev, [0, n]))
    for i in (0, 1, 63, 4097, 65535, 65536, n - 1):
        ref, w, tol = R.attend(q[i:i + 1], k[:i + 1, 0], v[:i + 1, 0], 0.125, torch.ones((1, i + 1), dtype=torch.bool), R.PROMPT_FLOOR[t])
        near(y[i:i + 1], ref, R.rounded(ref, w, tol, t, R.PROMPT_WEIGHTS[t]), t)


def test_rotary_past_32_bits(dev):
    """Sequences 2^31 elements and more apart, in place"""
    step = (1 << 31) + 64
    rows = torch.empty(2 * step + 3 * 192, dtype=torch.float16, device=dev).as_strided((3, 2, 3, 64), (step, 192, 64, 1))
    rows.copy_(torch.randn((3, 2, 3, 64), generator=gen(1)))
    rope, pos = nnr_amd.RotaryEmbedding(64, 100, device=dev), ints(dev, [[1, 2], [50, 51], [98, 99]])
    q, k = rows[:, :, :2], rows[:, :, 2:]
    want = rope(q.contiguous(), k.contiguous(), pos)
    out = rope(q, k, pos)
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    f, m = R.frequencies(64, 10000.0)
    near(out[0], *R.rotate(q.cpu(), pos.cpu(), f, m, False, 100), torch.float16)
    alone = q.contiguous(), k.contiguous()
    assert rope(q, alone[1], pos, out=(q, alone[1]))[0] is q and torch.equal(q, want[0]) and torch.equal(alone[1], want[1])
