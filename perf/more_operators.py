"""The operators around a decoder's cache, as cases that can be timed and checked.

A case is a dict of plain values. `kind` selects the operator:
  rotary  queries and keys turned by their tokens' positions, before the cache takes the keys
  prompt  causal attention of whole prompts to themselves, packed one behind another
  tree    attention of drafted tokens, which form a tree, over a paged, quantised cache
  copy    pages of several layers' caches copied (a sequence that is forked, a cache that is compacted)
  move    the accepted drafts' keys and values moved to the front of the drafts, several layers at once

`own` False computes them with elementary torch operations in 32 bits, True through the framework. Tables and
caches are made before the pass, as a serving program holds them.

A cache stands for these values. A group is a head's elements of one token (8 bits) or 32 of them (4 bits),
L is 127 or 7:
  scale = bf16(max |x| / L), code = clamp(round_half_even(x / scale), -L, L), value = code * scale
A page holds codes and bf16 scales of its tokens, keys and values of every head; in which order is the cache's own.
"""
import math

import torch

own = False

_T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---------------------------------------------------------------------------
# the cases

def listed():
    return [
        # a decoding step's queries and keys: a launch and little else; neighbours in pairs, half of the head
        dict(name="rotary_b4_s1", kind="rotary", batch=4, seq=1, q_heads=32, kv_heads=8, hd=128, rotary=64,
             interleaved=True, base=500000.0, scaling="linear", factor=4.0, positions=131072, dtype="f32"),
        # a long prompt of odd length, frequencies stretched past the length that a model was trained at
        dict(name="rotary_s8191", kind="rotary", batch=1, seq=8191, q_heads=32, kv_heads=8, hd=128, rotary=128,
             interleaved=False, base=10000.0, scaling="yarn", factor=8.0, positions=65536, dtype="bf16"),
        # a short question
        dict(name="prompt_37", kind="prompt", seqs=1, shortest=37, longest=37, q_heads=12, kv_heads=12, hd=64,
             dtype="f32"),
        # questions of a batch, packed
        dict(name="prompt_9_packed", kind="prompt", seqs=9, shortest=61, longest=1531, q_heads=32, kv_heads=8, hd=128,
             dtype="f16"),
        # a document
        dict(name="prompt_8192", kind="prompt", seqs=1, shortest=8192, longest=8192, q_heads=32, kv_heads=8, hd=128,
             dtype="bf16"),
        # wide heads that share one key/value head
        dict(name="prompt_3_hd256", kind="prompt", seqs=3, shortest=777, longest=2001, q_heads=8, kv_heads=1, hd=256,
             dtype="bf16"),
        # a conversation's drafts
        dict(name="tree_b1_s15", kind="tree", batch=1, seq=15, q_heads=32, kv_heads=8, hd=128, bits=8, page=64,
             prefix=0, longest=1800, each=False, dtype="f16"),
        # drafts of a batch, a tree of its own each, after instructions that all share
        dict(name="tree_b24_s64", kind="tree", batch=24, seq=64, q_heads=32, kv_heads=8, hd=128, bits=8, page=64,
             prefix=1000, longest=4096, each=True, dtype="bf16"),
        # a beam's forks: the last pages of a few sequences
        dict(name="copy_6", kind="copy", layers=2, pages=40, count=6, kv_heads=8, hd=128, bits=8, page=32),
        # a cache's pages brought together
        dict(name="copy_700", kind="copy", layers=8, pages=1500, count=700, kv_heads=4, hd=128, bits=4, page=64),
        # one conversation's accepted drafts
        dict(name="move_b1_n4", kind="move", layers=2, batch=1, drafts=15, count=4, kv_heads=8, hd=128, bits=8,
             page=64, longest=900, dtype="f16"),
        # a batch's, in several layers, 4 bits
        dict(name="move_b64_n7", kind="move", layers=8, batch=64, drafts=64, count=7, kv_heads=8, hd=128, bits=4,
             page=64, longest=500, dtype="bf16"),
    ]


def _logint(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rotary", "prompt", "prompt", "prompt", "tree", "tree", "copy", "move"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    hd, kv_heads, group = rng.choice([64, 96, 128, 128, 256]), rng.choice([1, 2, 4, 8, 12]), rng.choice([1, 2, 3, 4, 4, 8])
    bits, page, layers = rng.choice([8, 4]), rng.choice([32, 64, 128]), rng.choice([1, 2, 4, 8])
    if kind == "rotary":
        batch, seq = _logint(rng, 1, 64), _logint(rng, 1, 8192)
        while batch * seq * kv_heads * (group + 1) * hd * _SIZE[dtype] > 8192 * 40 * 128 * 2:
            batch, seq = max(1, batch // 2), max(1, seq // 2)
        scaling = rng.choice(["none", "linear", "ntk", "yarn"])
        return dict(kind=kind, batch=batch, seq=seq, q_heads=kv_heads * group, kv_heads=kv_heads, hd=hd,
                    rotary=hd if rng.random() < 0.5 else 2 * _logint(rng, 8, hd // 2),
                    interleaved=rng.random() < 0.5, base=rng.choice([10000.0, 500000.0]), scaling=scaling,
                    factor=1.0 if scaling == "none" else rng.choice([2.0, 4.0, 16.0]),
                    positions=seq + _logint(rng, 1, 131072), dtype=dtype)
    if kind == "prompt":
        seqs, longest = _logint(rng, 1, 24), _logint(rng, 1, 8192)
        # no more than a quarter of the largest listed case's products (an eighth in fp32)
        most = (16 if dtype == "f32" else 4) * 8192 * 8192 * 32 * 128 // 64
        while seqs * longest * longest * kv_heads * group * hd > most:
            seqs, longest = max(1, seqs // 2), max(1, longest * 4 // 5)
        return dict(kind=kind, seqs=seqs, shortest=_logint(rng, 1, longest), longest=longest,
                    q_heads=kv_heads * group, kv_heads=kv_heads, hd=hd, dtype=dtype)
    if kind == "tree":
        batch, seq = _logint(rng, 1, 48), _logint(rng, 2, 128)
        prefix = 0 if rng.random() < 0.5 else _logint(rng, 16, 8192)
        longest = seq + _logint(rng, 1, 4096)
        # no more than the largest listed case's products and keys
        while batch > 1 and (batch * seq * kv_heads * group * hd * (prefix + longest) > 24 * 64 * 32 * 128 * 5096 or
                             batch * longest * kv_heads * hd > 24 * 4096 * 8 * 128):
            batch //= 2
        return dict(kind=kind, batch=batch, seq=seq, q_heads=kv_heads * group, kv_heads=kv_heads, hd=hd, bits=bits,
                    page=page, prefix=prefix, longest=longest, each=rng.random() < 0.5, dtype=dtype)
    if kind == "copy":
        count = _logint(rng, 1, 700)
        while count > 1 and layers * count * _page_bytes(kv_heads, hd, bits, page) > 8 * 700 * 36864:
            count //= 2
        return dict(kind=kind, layers=layers, pages=2 * count + rng.randrange(1, 40), count=count, kv_heads=kv_heads,
                    hd=hd, bits=bits, page=page)
    batch, drafts = _logint(rng, 1, 64), _logint(rng, 3, 128)
    return dict(kind="move", layers=layers, batch=batch, drafts=drafts, count=rng.randrange(2, max(3, min(10, drafts // 2 + 1))),
                kv_heads=kv_heads, hd=hd, bits=bits, page=page, longest=drafts + _logint(rng, 1, 600), dtype=dtype)


# ---------------------------------------------------------------------------
# inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, g):
    return torch.randn(shape, generator=g, device="cuda")


def _tokens(shape, g, t):
    """Keys or values [..., heads, hd]: normal, a few channels several times as large."""
    return (_randn(shape, g) * torch.exp(0.6 * _randn(shape[-2:], g))).to(t)


def _projection(case, tokens, g):
    """Queries, keys and values as slices of one projection's output [tokens, (q_heads + 2 kv_heads) hd]."""
    hq, hk, d = case["q_heads"], case["kv_heads"], case["hd"]
    spread = torch.cat((torch.ones((hq, d), device="cuda"), torch.exp(0.6 * _randn((2 * hk, d), g))))
    rows = (_randn((tokens, hq + 2 * hk, d), g) * spread).to(_T[case["dtype"]])
    return rows[:, :hq], rows[:, hq:hq + hk], rows[:, hq + hk:]


def _frequencies(case):
    """(angles a position of the pairs, a factor for cosines and sines), in 64 bits."""
    r, base, s = case["rotary"], case["base"], case["factor"]
    i = torch.arange(0, r, 2, dtype=torch.float64, device="cuda")
    if case["scaling"] == "ntk":
        base = base * s ** (r / (r - 2))
    f = base ** (-i / r)
    if case["scaling"] == "linear":
        return f / s, 1.0
    if case["scaling"] == "yarn":
        # turns within the original length: over 32 as they are, under 1 stretched, a ramp between
        turns = f * (case["positions"] / s) / (2 * math.pi)
        keep = ((turns - 1) / 31).clamp(0, 1)
        return f / s * (1 - keep) + f * keep, 0.1 * math.log(s) + 1
    return f, 1.0


def _rotary_inputs(case, seed):
    g = _gen(seed)
    B, S = case["batch"], case["seq"]
    q, k, _ = _projection(case, B * S, g)
    first = torch.randint(0, case["positions"] - S + 1, (B, 1), generator=g, device="cuda")
    pos = (first + torch.arange(S, device="cuda")).to(torch.int32)
    return dict(q=q.unflatten(0, (B, S)), k=k.unflatten(0, (B, S)), pos=pos)


def _lengths(case, seed):
    n, lo, hi = case["seqs"], case["shortest"], case["longest"]
    lens = [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]
    order = torch.randperm(n, generator=torch.Generator().manual_seed(seed)).tolist()
    return [lens[i] for i in order]


def _prompt_inputs(case, seed):
    lens = _lengths(case, seed)
    q, k, v = _projection(case, sum(lens), _gen(seed))
    starts = torch.tensor([0, *lens]).cumsum(0).to("cuda", torch.int32)
    return dict(q=q, k=k, v=v, starts=starts, lens=lens)


def _groups(case):
    return 1 if case["bits"] == 8 else case["hd"] // 32


def _page_bytes(kv_heads, hd, bits, page):
    return 2 * kv_heads * page * (hd * bits // 8 + 2 * (1 if bits == 8 else hd // 32))


def _tables(case, g, count, prefix):
    """Page tables of `count` sequences and of the prefix, over pages in no order."""
    per, pre = -(-case["longest"] // case["page"]), -(-prefix // case["page"])
    order = torch.randperm(count * per + pre + 3, generator=g, device="cuda").to(torch.int32)
    return order[:count * per].reshape(count, per).contiguous(), order[count * per:count * per + pre].contiguous()


def _tree(case, g):
    """Who sees whom: a draft itself and the drafts that led to it. [seq, seq], or one a sequence."""
    n, s = (case["batch"] if case["each"] else 1), case["seq"]
    mask = torch.eye(s, dtype=torch.bool, device="cuda").repeat(n, 1, 1)
    parent = torch.rand((n, s), generator=g, device="cuda")
    rows = torch.arange(n, device="cuda")
    for i in range(1, s):
        # mostly one of the last few
        p = (i - 1 - (parent[:, i] ** 3 * i).long()).clamp(0, i - 1)
        mask[:, i] |= mask[rows, p]
    return mask if case["each"] else mask[0]


def _tree_inputs(case, seed):
    g, t, B = _gen(seed), _T[case["dtype"]], case["batch"]
    table, prefix = _tables(case, g, B, case["prefix"])
    lens = torch.randint(case["seq"], case["longest"] + 1, (B,), generator=g, device="cuda").to(torch.int32)
    lens[0] = case["longest"]
    own_shape, pre_shape = (B, case["longest"], case["kv_heads"], case["hd"]), (1, case["prefix"], case["kv_heads"], case["hd"])
    x = dict(table=table, prefix=prefix, lens=lens, tree=_tree(case, g))
    x.update(k=_tokens(own_shape, g, t), v=_tokens(own_shape, g, t), pk=_tokens(pre_shape, g, t), pv=_tokens(pre_shape, g, t))
    x["q"] = _randn((B, case["seq"], case["q_heads"], case["hd"]), g).to(t)
    x["pages"] = table.numel() + prefix.numel() + 3
    return x


def _copy_inputs(case, seed):
    g = _gen(seed)
    size = (case["layers"], case["pages"], _page_bytes(case["kv_heads"], case["hd"], case["bits"], case["page"]))
    order = torch.randperm(case["pages"], generator=g, device="cuda").to(torch.int32)
    n = case["count"]
    return dict(data=torch.randint(0, 256, size, generator=g, device="cuda", dtype=torch.uint8), src=order[:n], dst=order[n:2 * n])


def _move_inputs(case, seed):
    """Drafts at the end of every sequence. The accepted path starts at the first draft; those that it goes on with
    lie behind the positions that it takes, and some sequences accept fewer (-1: none)."""
    g, t, B, n, s = _gen(seed), _T[case["dtype"]], case["batch"], case["count"], case["drafts"]
    table, _ = _tables(case, g, B, 0)
    lens = torch.randint(s, case["longest"] + 1, (B,), generator=g, device="cuda").to(torch.int32)
    path = torch.rand((B, s - n), generator=g, device="cuda").argsort(-1)[:, :n - 1].sort(-1).values + n
    path = torch.cat((torch.zeros((B, 1), dtype=torch.int64, device="cuda"), path), -1)
    base = lens.long()[:, None] - s
    taken = torch.randint(1, n + 1, (B, 1), generator=g, device="cuda")
    i = torch.arange(n, device="cuda")
    src = torch.where(i < taken, base + path, -1).to(torch.int32)
    shape = (case["layers"], B, s, case["kv_heads"], case["hd"])
    return dict(table=table, lens=lens, src=src, dst=(base + i).to(torch.int32), end=(base[:, 0] + n).to(torch.int32),
                k=_tokens(shape, g, t), v=_tokens(shape, g, t), pages=table.numel() + 3)


class _PlainCaches:
    """Codes and scales of several layers' paged caches, one byte a code whatever the bits."""

    def __init__(self, case, layers, pages):
        self.limit, self.page, self.groups = (127 if case["bits"] == 8 else 7), case["page"], _groups(case)
        shape = (layers, pages, case["page"], case["kv_heads"])
        self.codes = [torch.zeros((*shape, case["hd"]), dtype=torch.int8, device="cuda") for _ in "kv"]
        self.scales = [torch.zeros((*shape, self.groups), dtype=torch.float32, device="cuda") for _ in "kv"]

    def where(self, table, pos):
        """Page and offset of positions [B, S] of the sequences of a table."""
        return torch.gather(table.long(), 1, pos // self.page), pos % self.page

    def write(self, k, v, table, pos):
        """k, v [layers, B, S, heads, hd]"""
        page, off = self.where(table, pos)
        for i, x in enumerate((k, v)):
            x = x.float().unflatten(-1, (self.groups, -1))
            # a quotient may lie next to a border between two codes
            s = (x.abs().amax(-1, keepdim=True).double() / self.limit).float().bfloat16().float()
            c = (x.double() / torch.where(s > 0, s, 1.0).double()).round().clamp(-self.limit, self.limit)
            self.codes[i][:, page, off] = c.flatten(-2).to(torch.int8)
            self.scales[i][:, page, off] = s.squeeze(-1)

    def read(self, i, table, pos):
        page, off = self.where(table, pos)
        c = self.codes[i][:, page, off].float().unflatten(-1, (self.groups, -1))
        return (c * self.scales[i][:, page, off].unsqueeze(-1)).flatten(-2)

    def move(self, table, src, dst):
        batch, at = torch.nonzero((src >= 0) & (dst >= 0), as_tuple=True)
        table, src, dst = table[batch], src[batch, at].long()[:, None], dst[batch, at].long()[:, None]
        (page, off), (to, to_off) = self.where(table, src), self.where(table, dst)
        for x in (*self.codes, *self.scales):
            x[:, to[:, 0], to_off[:, 0]] = x[:, page[:, 0], off[:, 0]]


def _positions(lens, seq):
    return lens.long()[:, None] - seq + torch.arange(seq, device="cuda")


def _caches(case, layers, pages):
    if own:
        import nnr_amd
        return [nnr_amd.KVCache(pages, case["kv_heads"], case["hd"], page_size=case["page"], bits=case["bits"])
                for _ in range(layers)]
    return _PlainCaches(case, layers, pages)


def _fill(caches, k, v, table, lens):
    """Newest tokens k, v [layers, B, S, heads, hd] into the caches."""
    if own:
        for c, kl, vl in zip(caches, k, v):
            c.write(kl, vl, table, lens)
    else:
        caches.write(k, v, table, _positions(lens, k.shape[2]))


def prepare(case, seed):
    kind = case["kind"]
    if kind == "rotary":
        x = _rotary_inputs(case, seed)
        if own:
            import nnr_amd
            x["rope"] = nnr_amd.RotaryEmbedding(case["hd"], case["positions"], base=case["base"],
                                                rotary_dim=case["rotary"], interleaved=case["interleaved"],
                                                scaling=case["scaling"], factor=case["factor"])
        else:
            f, m = _frequencies(case)
            angles = torch.arange(case["positions"], dtype=torch.float64, device="cuda")[:, None] * f
            x["cos"], x["sin"] = (angles.cos() * m).float(), (angles.sin() * m).float()
        return dict(case=case, **x)
    if kind == "prompt":
        return dict(case=case, **_prompt_inputs(case, seed))
    if kind == "copy":
        x = _copy_inputs(case, seed)
        if own:
            caches = _caches(case, case["layers"], case["pages"])
            for c, data in zip(caches, x["data"]):
                c.data.copy_(data.flatten())
            return dict(case=case, caches=caches, src=x["src"], dst=x["dst"])
        return dict(case=case, **x)
    if kind == "move":
        x = _move_inputs(case, seed)
        caches = _caches(case, case["layers"], x["pages"])
        _fill(caches, x["k"], x["v"], x["table"], x["lens"])
        return dict(case=case, caches=caches, **{n: x[n] for n in ("table", "src", "dst", "end")})
    x = _tree_inputs(case, seed)
    cache = _caches(case, 1, x["pages"])
    full = torch.full((case["batch"],), case["longest"], dtype=torch.int32, device="cuda")
    _fill(cache, x["k"][None], x["v"][None], x["table"], full)
    if case["prefix"]:
        _fill(cache, x["pk"][None], x["pv"][None], x["prefix"][None], torch.full((1,), case["prefix"], dtype=torch.int32, device="cuda"))
    return dict(case=case, cache=cache, **{n: x[n] for n in ("q", "table", "lens", "prefix", "tree")})


# ---------------------------------------------------------------------------
# one pass

def _plain_rotary(s, x):
    r = s["case"]["rotary"]
    pos = s["pos"].long()
    cos, sin = s["cos"][pos].unsqueeze(2), s["sin"][pos].unsqueeze(2)
    y, t = x.float().clone(), x[..., :r].float()
    if s["case"]["interleaved"]:
        a, b = t[..., 0::2], t[..., 1::2]
        y[..., :r] = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = t[..., :r // 2], t[..., r // 2:]
        y[..., :r] = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return y.to(x.dtype)


def _plain_prompt(s):
    q, k, v = s["q"], s["k"], s["v"]
    H, D = k.shape[1:]
    G, y, at = q.shape[1] // H, torch.empty(q.shape, dtype=q.dtype, device="cuda"), 0
    for n in s["lens"]:
        rows = q[at:at + n].float().reshape(n, H, G, D).permute(1, 2, 0, 3).reshape(H, G * n, D) / math.sqrt(D)
        keys = k[at:at + n].float().permute(1, 2, 0).contiguous()
        scores = torch.matmul(rows, keys).reshape(H, G, n, n)
        later = torch.ones((n, n), dtype=torch.bool, device="cuda").triu_(1)
        scores.masked_fill_(later, float("-inf"))
        e = (scores - scores.amax(-1, keepdim=True)).exp_()
        total = e.sum(-1, keepdim=True)
        out = torch.matmul(e.reshape(H, G * n, n), v[at:at + n].float().transpose(0, 1).contiguous())
        y[at:at + n] = (out.reshape(H, G, n, D) / total).permute(2, 0, 1, 3).reshape(n, H * G, D).to(q.dtype)
        at += n
    return y


def _plain_tree(s):
    case, cache, q, lens = s["case"], s["cache"], s["q"], s["lens"].long()
    B, S, H, G, D = case["batch"], case["seq"], case["kv_heads"], case["q_heads"] // case["kv_heads"], case["hd"]
    n, p = case["longest"], case["prefix"]
    qs = q.float().reshape(B, S, H, G, D) / math.sqrt(D)
    pos = torch.arange(n, device="cuda").expand(B, n)
    k, v = (cache.read(i, s["table"], pos)[0].permute(0, 2, 1, 3).contiguous() for i in (0, 1))   # B H n D
    kt = k.transpose(-1, -2).contiguous()
    scores = torch.matmul(qs.permute(0, 2, 1, 3, 4).reshape(B, H, S * G, D), kt).reshape(B, H, S, G, n)
    draft = pos - (lens - S)[:, None]                                                             # B n
    tree = s["tree"].expand(B, S, S)
    sees = torch.gather(tree, 2, draft.clamp(0, S - 1)[:, None].expand(B, S, n)) & (draft < S)[:, None]
    sees = sees | (draft < 0)[:, None]
    scores = scores.masked_fill(~sees[:, None, :, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    if p:
        at = torch.arange(p, device="cuda")[None]
        pk, pv = (cache.read(i, s["prefix"][None], at)[0, 0].permute(1, 0, 2).contiguous() for i in (0, 1))   # H p D
        pkt = pk.transpose(-1, -2).contiguous()
        pscores = torch.matmul(qs.permute(2, 0, 1, 3, 4).reshape(H, B * S * G, D), pkt)
        top = torch.maximum(top, pscores.amax(-1, keepdim=True).reshape(H, B, S, G, 1).transpose(0, 1))
        pe = torch.exp(pscores - top.transpose(0, 1).reshape(H, B * S * G, 1))
    e = torch.exp(scores - top)
    total = e.sum(-1, keepdim=True)
    y = torch.matmul(e.reshape(B, H, S * G, n), v).reshape(B, H, S, G, D)
    if p:
        total = total + pe.sum(-1).reshape(H, B, S, G, 1).transpose(0, 1)
        y = y + torch.matmul(pe, pv).reshape(H, B, S, G, D).transpose(0, 1)
    return (y / total).permute(0, 2, 1, 3, 4).reshape(B, S, H * G, D).to(q.dtype)


def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if own:
        import nnr_amd
    if kind == "rotary":
        q, k = state["q"], state["k"]
        return state["rope"](q, k, state["pos"]) if own else (_plain_rotary(state, q), _plain_rotary(state, k))
    if kind == "prompt":
        if own:
            return nnr_amd.prompt_attention(state["q"], state["k"], state["v"], state["starts"])
        return _plain_prompt(state)
    if kind == "tree":
        if own:
            return state["cache"][0].attention(state["q"], state["table"], state["lens"], prefix_table=state["prefix"],
                                               prefix_len=case["prefix"], tree=state["tree"])
        return _plain_tree(state)
    if kind == "copy":
        if own:
            nnr_amd.copy_pages(state["caches"], state["src"], state["dst"])
            return [c.data.view(case["pages"], -1) for c in state["caches"]]
        state["data"][:, state["dst"].long()] = state["data"][:, state["src"].long()]
        return list(state["data"].unbind(0))
    # the moved tokens are read back as the values that they stand for
    caches, n, table, end, t = state["caches"], case["count"], state["table"], state["end"], _T[case["dtype"]]
    if own:
        nnr_amd.move_tokens(caches, table, state["src"], state["dst"])
        return [x for c in caches for x in c.read(n, table, end, t)]
    caches.move(table, state["src"], state["dst"])
    k, v = (caches.read(i, table, _positions(end, n)).to(t) for i in (0, 1))
    return [x for pair in zip(k, v) for x in pair]


# ---------------------------------------------------------------------------
# what a pass cannot do without

def work(case):
    kind = case["kind"]
    if kind == "copy":
        moved = 2 * case["layers"] * case["count"] * _page_bytes(case["kv_heads"], case["hd"], case["bits"], case["page"])
        return dict(bytes=moved + 8 * case["count"], flops=0)
    if kind == "move":
        # tokens read and written (as many as a sequence takes on average), then read and written as values
        token = _page_bytes(case["kv_heads"], case["hd"], case["bits"], 1)
        n, rows = case["count"], case["layers"] * case["batch"]
        values = 2 * case["kv_heads"] * case["hd"]
        return dict(bytes=int(rows * (2 * token * (n + 1) / 2 + n * (token + values * _SIZE[case["dtype"]]))),
                    flops=rows * n * values)
    e, D, hq, hk = _SIZE[case["dtype"]], case["hd"], case["q_heads"], case["kv_heads"]
    if kind == "rotary":
        tokens = case["batch"] * case["seq"]
        return dict(bytes=tokens * (2 * (hq + hk) * D * e + 4 * case["rotary"] + 4),
                    flops=3 * tokens * (hq + hk) * case["rotary"])
    if kind == "prompt":
        lens = _lengths(case, 0)
        return dict(bytes=sum(lens) * 2 * (hq + hk) * D * e, flops=sum(2 * n * (n + 1) for n in lens) * hq * D)
    B, S = case["batch"], case["seq"]
    # lengths are uniform from seq to longest; half of a tree's pairs at most are seen
    keys = B * (S + case["longest"]) / 2 + case["prefix"]
    row = case["prefix"] + (case["longest"] - S) / 2 + (S + 1) / 4
    return dict(bytes=int(2 * B * S * hq * D * e + keys * _page_bytes(hk, D, case["bits"], 1) + (B if case["each"] else 1) * S * S),
                flops=int(4 * B * S * hq * D * row))


# ---------------------------------------------------------------------------
# the definitions in 64 bits

def _round_bf16(x):
    """x >= 0 rounded to 8 significant bits, ties to even: by the bits of a 64-bit number, of which 45 go."""
    bits = x.contiguous().view(torch.int64)
    return ((bits + (1 << 44) - 1 + (bits >> 45 & 1)) >> 45 << 45).view(torch.float64)


def _exact_values(case, x):
    """What the cache holds for x [..., hd]: code * scale, in 64 bits."""
    limit = 127.0 if case["bits"] == 8 else 7.0
    size = case["hd"] if case["bits"] == 8 else 32
    parts = []
    for at in range(0, case["hd"], size):
        part = x[..., at:at + size].double()
        scale = _round_bf16(part.abs().max(-1, keepdim=True).values / limit)
        code = torch.clamp(torch.round(part / torch.where(scale == 0, torch.ones_like(scale), scale)), -limit, limit)
        parts.append(code * scale)
    return torch.cat(parts, -1)


def _exact_turn(case, x, pos):
    """The pairs as complex numbers, times m e^(i position frequency)."""
    r, s = case["rotary"], case["factor"]
    freqs, m = [], 1.0
    for j in range(r // 2):
        f = math.exp(-2 * j / r * math.log(case["base"]))
        if case["scaling"] == "linear":
            f /= s
        elif case["scaling"] == "ntk":
            # the base is stretched so that the lowest frequency is divided by the factor
            f *= s ** (-2 * j / (r - 2))
        elif case["scaling"] == "yarn":
            turns = case["positions"] / s * f / math.tau
            keep = min(1.0, max(0.0, (turns - 1) / (32 - 1)))
            f, m = f * (keep + (1 - keep) / s), 1 + math.log(s) / 10
        freqs.append(f)
    turn = torch.polar(torch.tensor(m, dtype=torch.float64, device="cuda"),
                       pos.double()[..., None, None] * torch.tensor(freqs, dtype=torch.float64, device="cuda"))
    out, z = x.double(), x[..., :r].double()
    if case["interleaved"]:
        w = torch.view_as_complex(z.reshape(*z.shape[:-1], r // 2, 2).contiguous()) * turn
        out[..., :r] = torch.view_as_real(w).reshape(z.shape)
    else:
        w = torch.complex(z[..., :r // 2].contiguous(), z[..., r // 2:].contiguous()) * turn
        out[..., :r // 2], out[..., r // 2:r] = w.real, w.imag
    return out


def exact(case, seed):
    kind = case["kind"]
    if kind == "rotary":
        x = _rotary_inputs(case, seed)
        return tuple(_exact_turn(case, x[n], x["pos"]) for n in "qk")
    if kind == "copy":
        return None
    if kind == "move":
        x = _move_inputs(case, seed)
        n, s = case["count"], case["drafts"]
        base = x["lens"].long() - s
        took = torch.arange(n, device="cuda").expand(case["batch"], n)
        took = torch.where(x["src"] >= 0, x["src"].long() - base[:, None], took)
        at = took[None, :, :, None, None].expand(case["layers"], -1, -1, case["kv_heads"], case["hd"])
        k, v = (torch.gather(_exact_values(case, x[name]), 2, at) for name in "kv")
        return [y[i] for i in range(case["layers"]) for y in (k, v)]
    D, hq = case["hd"], case["q_heads"]
    G = hq // case["kv_heads"]
    if kind == "prompt":
        x = _prompt_inputs(case, seed)
        y = torch.empty((sum(x["lens"]), hq, D), dtype=torch.float64, device="cuda")
        for b, n in enumerate(x["lens"]):
            own_rows = slice(sum(x["lens"][:b]), sum(x["lens"][:b]) + n)
            hidden = torch.arange(n, device="cuda")[None] > torch.arange(n, device="cuda")[:, None]
            for h in range(hq):
                keys, vals = x["k"][own_rows, h // G].double(), x["v"][own_rows, h // G].double()
                sc = torch.where(hidden, -math.inf, torch.mm(x["q"][own_rows, h].double(), keys.t()) * D ** -0.5)
                y[own_rows, h] = torch.mm(torch.softmax(sc, -1), vals)
        return y
    x = _tree_inputs(case, seed)
    B, S, P = case["batch"], case["seq"], case["prefix"]
    lens = x["lens"].tolist()
    tree = x["tree"] if case["each"] else x["tree"][None].repeat(B, 1, 1)
    y = torch.empty((B, S, hq, D), dtype=torch.float64, device="cuda")
    for h in range(case["kv_heads"]):
        pk, pv = _exact_values(case, x["pk"][0, :, h]), _exact_values(case, x["pv"][0, :, h])
        for b in range(B):
            n = lens[b]
            # the positions in the cache were written as one run that ends at `longest`
            keys = torch.cat((pk, _exact_values(case, x["k"][b, :n, h])))
            vals = torch.cat((pv, _exact_values(case, x["v"][b, :n, h])))
            sees = torch.cat((torch.ones((S, P + n - S), dtype=torch.bool, device="cuda"), tree[b]), -1)
            q = x["q"][b, :, h * G:(h + 1) * G].double().reshape(S * G, D)
            sc = torch.mm(q, keys.t()) * D ** -0.5
            sc = torch.where(sees.repeat_interleave(G, 0), sc, -math.inf)
            y[b, :, h * G:(h + 1) * G] = torch.mm(torch.softmax(sc, -1), vals).reshape(S, G, D)
    return y
