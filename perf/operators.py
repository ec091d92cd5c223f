"""The operators of a decoder's serving step, as cases that can be timed and checked.

A case is a dict of plain values. `kind` selects the operator:
  nbits      y = a W^T + bias with 4-bit weights in blocks along K, each block with a scale (and a zero point)
  cache      keys and values of `seq` new tokens a sequence quantised into the pages of a cache, and the same
             positions read back
  attention  queries over a paged, quantised cache: a prefix that the whole batch shares, then the sequence's own
             tokens, causally

`own` False computes them with elementary torch operations in 32 bits, True through the framework.
Weights and caches are made before the pass, as a serving program holds them.

A cache stands for these values. A group is a head's elements of one token (8 bits) or 32 of them (4 bits),
L is 127 or 7:
  scale = bf16(max |x| / L), code = clamp(round_half_even(x / scale), -L, L), value = code * scale
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
        # one token through a small projection: a launch and little else
        dict(name="nbits_m1_k1024", kind="nbits", m=1, k=1024, n=1024, block=32, zp=False, bias=False, dtype="f16"),
        # one token through a wide projection, as an interactive service answers
        dict(name="nbits_m1_k4096", kind="nbits", m=1, k=4096, n=8192, block=64, zp=True, bias=False, dtype="bf16"),
        # a few tokens, extents that no tile divides, the last block cut short
        dict(name="nbits_m7_odd", kind="nbits", m=7, k=1990, n=1531, block=32, zp=True, bias=True, dtype="f32"),
        # a batch of sequences, one token each, through a large projection
        dict(name="nbits_m64_k8192", kind="nbits", m=64, k=8192, n=8192, block=128, zp=False, bias=False,
             dtype="f16"),
        # a prompt
        dict(name="nbits_m512", kind="nbits", m=512, k=4096, n=4096, block=32, zp=False, bias=True, dtype="bf16"),
        # a decoding step's keys and values
        dict(name="cache_b64_s1", kind="cache", batch=64, seq=1, kv_heads=8, hd=128, bits=8, page=64, longest=4096,
             dtype="f16"),
        # prompts of odd length into 4 bits
        dict(name="cache_b3_s1900", kind="cache", batch=3, seq=1900, kv_heads=8, hd=128, bits=4, page=64,
             longest=2000, dtype="bf16"),
        # one sequence without a shared prefix, fp32
        dict(name="attention_b1", kind="attention", batch=1, seq=1, q_heads=12, kv_heads=12, hd=64, bits=8, page=32,
             prefix=0, longest=700, dtype="f32"),
        # many long sequences that share nothing
        dict(name="attention_b48_own", kind="attention", batch=48, seq=1, q_heads=32, kv_heads=8, hd=128, bits=8,
             page=64, prefix=0, longest=8192, dtype="bf16"),
        # answers to many questions about one document
        dict(name="attention_b32_p8192", kind="attention", batch=32, seq=1, q_heads=32, kv_heads=8, hd=128, bits=8,
             page=64, prefix=8192, longest=512, dtype="f16"),
        # a large batch over a very long prefix in 4 bits
        dict(name="attention_b128_p32768", kind="attention", batch=128, seq=1, q_heads=32, kv_heads=8, hd=128, bits=4,
             page=128, prefix=32768, longest=300, dtype="bf16"),
        # several tokens a sequence (a draft that is verified, a piece of a prompt), an odd prefix
        dict(name="attention_b8_s16", kind="attention", batch=8, seq=16, q_heads=16, kv_heads=4, hd=256, bits=8,
             page=64, prefix=2011, longest=1000, dtype="f16"),
    ]


def _logint(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["nbits", "nbits", "cache", "attention", "attention"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if kind == "nbits":
        m, k, n = _logint(rng, 1, 512), _logint(rng, 256, 8192), _logint(rng, 256, 8192)
        k = k if rng.random() < 0.3 else (k + 63) // 64 * 64
        n = n if rng.random() < 0.3 else (n + 63) // 64 * 64
        while m > 1 and m * k * n > 512 * 4096 * 4096:
            m //= 2
        return dict(kind=kind, m=m, k=k, n=n, block=rng.choice([32, 32, 64, 128, 256]), zp=rng.random() < 0.5,
                    bias=rng.random() < 0.4, dtype=dtype)
    hd, bits, kv_heads = rng.choice([64, 96, 128, 128, 256]), rng.choice([8, 4]), rng.choice([1, 2, 4, 8, 12])
    page = rng.choice([32, 64, 128])
    if kind == "cache":
        seq = _logint(rng, 1, 2000)
        batch = _logint(rng, 1, 64)
        while batch > 1 and batch * seq * kv_heads * hd > 3 * 1900 * 8 * 128:
            batch //= 2
        return dict(kind=kind, batch=batch, seq=seq, kv_heads=kv_heads, hd=hd, bits=bits, page=page,
                    longest=seq + _logint(rng, 1, 2000), dtype=dtype)
    group = rng.choice([1, 2, 4, 4, 8])
    seq = 1 if rng.random() < 0.6 else _logint(rng, 2, 64)
    batch = _logint(rng, 1, 96)
    prefix = 0 if rng.random() < 0.25 else _logint(rng, 16, 16384)
    longest = seq + _logint(rng, 1, 4096)
    # no more than half of the largest listed case's products
    while batch > 1 and batch * seq * kv_heads * group * hd * (prefix + longest) > 64 * 32 * 128 * 32768:
        batch //= 2
    while seq > 1 and batch * seq * kv_heads * group * hd * (prefix + longest) > 64 * 32 * 128 * 32768:
        seq //= 2
    while batch > 1 and batch * longest * kv_heads * hd > 48 * 8192 * 8 * 128:
        batch //= 2
    return dict(kind=kind, batch=batch, seq=seq, q_heads=kv_heads * group, kv_heads=kv_heads, hd=hd, bits=bits,
                page=page, prefix=prefix, longest=longest, dtype=dtype)


# ---------------------------------------------------------------------------
# inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _nbits_inputs(case, seed):
    """Activations, and weights as a quantiser leaves them: codes 0..15 around the zero point, two a byte."""
    g, t = _gen(seed), _T[case["dtype"]]
    n, k, nb = case["n"], case["k"], -(-case["k"] // case["block"])
    codes = (torch.randn((n, nb * case["block"]), generator=g, device="cuda") * 2.7 + 8).round_().clamp_(0, 15)
    codes = codes.to(torch.uint8)
    packed = codes[:, 0::2] | (codes[:, 1::2] << 4)
    scales = ((torch.rand((n, nb), generator=g, device="cuda") + 0.5) * (0.4 / math.sqrt(k))).to(t)
    zp = None
    if case["zp"]:
        zp = torch.randint(5, 12, (n, (nb + 1) // 2 * 2), generator=g, device="cuda").to(torch.uint8)
        zp = zp[:, 0::2] | (zp[:, 1::2] << 4)
    bias = torch.randn(n, generator=g, device="cuda").to(t) if case["bias"] else None
    a = torch.randn((case["m"], k), generator=g, device="cuda").to(t)
    return dict(a=a, b=packed.reshape(n, nb, -1), scales=scales, zp=zp, bias=bias)


def _tokens(shape, g, t):
    """Keys or values [..., heads, hd]: normal, a few channels several times as large."""
    x = torch.randn(shape, generator=g, device="cuda")
    return (x * torch.exp(0.6 * torch.randn(shape[-2:], generator=g, device="cuda"))).to(t)


def _tables(case, g, count):
    """Page tables of `count` sequences and of the prefix, over pages in no order; lengths of the sequences."""
    per = -(-case["longest"] // case["page"])
    pre = -(-case.get("prefix", 0) // case["page"])
    order = torch.randperm(count * per + pre + 3, generator=g, device="cuda").to(torch.int32)
    lens = torch.randint(case["seq"], case["longest"] + 1, (count,), generator=g, device="cuda").to(torch.int32)
    lens[0] = case["longest"]
    return order[:count * per].reshape(count, per).contiguous(), order[count * per:count * per + pre].contiguous(), lens


def _groups(case):
    return 1 if case["bits"] == 8 else case["hd"] // 32


class _PlainCache:
    """Codes and scales of a paged cache, one byte a code whatever the bits."""

    def __init__(self, case, pages):
        self.limit, self.page, self.groups = (127 if case["bits"] == 8 else 7), case["page"], _groups(case)
        shape = (pages, case["page"], case["kv_heads"])
        self.codes = [torch.zeros((*shape, case["hd"]), dtype=torch.int8, device="cuda") for _ in "kv"]
        self.scales = [torch.zeros((*shape, self.groups), dtype=torch.float32, device="cuda") for _ in "kv"]

    def where(self, table, pos):
        """Page and offset of positions [B, S] of the sequences of a table."""
        return torch.gather(table.long(), 1, pos // self.page), pos % self.page

    def write(self, k, v, table, pos):
        page, off = self.where(table, pos)
        for i, x in enumerate((k, v)):
            x = x.float().reshape(*x.shape[:-1], self.groups, -1)
            # a quotient may lie next to a border between two codes
            s = (x.abs().amax(-1, keepdim=True).double() / self.limit).float().bfloat16().float()
            c = (x.double() / torch.where(s > 0, s, 1.0).double()).round().clamp(-self.limit, self.limit)
            self.codes[i][page, off] = c.flatten(-2).to(torch.int8)
            self.scales[i][page, off] = s.squeeze(-1)

    def read(self, i, table, pos):
        page, off = self.where(table, pos)
        c = self.codes[i][page, off].float()
        return (c.reshape(*c.shape[:-1], self.groups, -1) * self.scales[i][page, off].unsqueeze(-1)).flatten(-2)


def _cache_inputs(case, seed):
    g, t = _gen(seed), _T[case["dtype"]]
    table, prefix, lens = _tables(case, g, case["batch"])
    shape = (case["batch"], case["seq"] if case["kind"] == "cache" else case["longest"], case["kv_heads"], case["hd"])
    x = dict(table=table, lens=lens, prefix=prefix, k=_tokens(shape, g, t), v=_tokens(shape, g, t))
    x["pages"] = table.numel() + prefix.numel() + 3
    if case["kind"] == "attention":
        shape = (1, case["prefix"], case["kv_heads"], case["hd"])
        x["pk"], x["pv"] = _tokens(shape, g, t), _tokens(shape, g, t)
        x["q"] = torch.randn((case["batch"], case["seq"], case["q_heads"], case["hd"]), generator=g,
                             device="cuda").to(t)
    return x


def _positions(lens, seq):
    return lens.long()[:, None] - seq + torch.arange(seq, device="cuda")


def prepare(case, seed):
    if case["kind"] == "nbits":
        x = _nbits_inputs(case, seed)
        if own:
            import nnr_amd
            op = nnr_amd.MatMulNBits(x["b"], x["scales"], case["k"], case["block"], zero_points=x["zp"],
                                     bias=x["bias"])
            return dict(case=case, op=op, a=x["a"])
        return dict(case=case, **x)
    x = _cache_inputs(case, seed)
    if own:
        import nnr_amd
        cache = nnr_amd.KVCache(x["pages"], case["kv_heads"], case["hd"], page_size=case["page"], bits=case["bits"])
    else:
        cache = _PlainCache(case, x["pages"])
    if case["kind"] == "cache":
        return dict(case=case, cache=cache, pos=_positions(x["lens"], case["seq"]), **x)
    full = torch.full((case["batch"],), case["longest"], dtype=torch.int32, device="cuda")
    one = torch.full((1,), case["prefix"], dtype=torch.int32, device="cuda")
    if own:
        cache.write(x["k"], x["v"], x["table"], full)
        if case["prefix"]:
            cache.write(x["pk"], x["pv"], x["prefix"][None], one)
    else:
        cache.write(x["k"], x["v"], x["table"], _positions(full, case["longest"]))
        if case["prefix"]:
            cache.write(x["pk"], x["pv"], x["prefix"][None], _positions(one, case["prefix"]))
    return dict(case=case, cache=cache, **{n: x[n] for n in ("q", "table", "lens", "prefix")})


# ---------------------------------------------------------------------------
# one pass

def _plain_nbits(s):
    case, b = s["case"], s["b"]
    codes = torch.stack((b & 15, b >> 4), -1).flatten(-2).float()
    zp = 8.0
    if s["zp"] is not None:
        zp = torch.stack((s["zp"] & 15, s["zp"] >> 4), -1).flatten(-2)[:, :b.shape[1], None].float()
    w = ((codes - zp) * s["scales"].float()[:, :, None]).flatten(-2)[:, :case["k"]]
    y = s["a"].float() @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["a"].dtype)


def _plain_attention(s):
    case, cache, q, lens = s["case"], s["cache"], s["q"], s["lens"].long()
    B, S, H, G, D = case["batch"], case["seq"], case["kv_heads"], case["q_heads"] // case["kv_heads"], case["hd"]
    qs = q.float().reshape(B, S, H, G, D) / math.sqrt(D)
    n = case["longest"]
    pos = torch.arange(n, device="cuda").expand(B, n)
    k, v = (cache.read(i, s["table"], pos).permute(0, 2, 1, 3).contiguous() for i in (0, 1))   # B H n D
    rows = qs.permute(0, 2, 1, 3, 4).reshape(B, H, S * G, D)
    kt = k.transpose(-1, -2).contiguous()
    scores = torch.matmul(rows, kt).reshape(B, H, S, G, n)
    last = lens[:, None] - S + torch.arange(S, device="cuda")
    scores = scores.masked_fill((pos[:, None] > last[:, :, None])[:, None, :, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = case["prefix"]
    if p:
        pos = torch.arange(p, device="cuda")[None]
        pk, pv = (cache.read(i, s["prefix"][None], pos)[0].permute(1, 0, 2).contiguous() for i in (0, 1))   # H p D
        prows = qs.permute(2, 0, 1, 3, 4).reshape(H, B * S * G, D)
        pkt = pk.transpose(-1, -2).contiguous()
        pscores = torch.matmul(prows, pkt)
        ptop = pscores.amax(-1, keepdim=True).reshape(H, B, S, G, 1).transpose(0, 1)
        top = torch.maximum(top, ptop)
        pe = torch.exp(pscores - top.transpose(0, 1).reshape(H, B * S * G, 1))
    e = torch.exp(scores - top)
    total = e.sum(-1, keepdim=True)
    y = torch.matmul(e.reshape(B, H, S * G, n), v).reshape(B, H, S, G, D)
    if p:
        total = total + pe.sum(-1).reshape(H, B, S, G, 1).transpose(0, 1)
        y = y + torch.matmul(pe, pv).reshape(H, B, S, G, D).transpose(0, 1)
    return (y / total).permute(0, 2, 1, 3, 4).reshape(B, S, H * G, D).to(q.dtype)


def run(state):
    case = state["case"]
    if case["kind"] == "nbits":
        return state["op"](state["a"]) if own else _plain_nbits(state)
    cache = state["cache"]
    if case["kind"] == "cache":
        k, v, table = state["k"], state["v"], state["table"]
        if own:
            cache.write(k, v, table, state["lens"])
            return cache.read(case["seq"], table, state["lens"], k.dtype)
        cache.write(k, v, table, state["pos"])
        return tuple(cache.read(i, table, state["pos"]).to(k.dtype) for i in (0, 1))
    if own:
        return cache.attention(state["q"], state["table"], state["lens"], prefix_table=state["prefix"],
                               prefix_len=case["prefix"])
    return _plain_attention(state)


# ---------------------------------------------------------------------------
# what a pass cannot do without

def _token_bytes(case):
    """Codes and scales of one token, keys and values."""
    return 2 * case["kv_heads"] * (case["hd"] * case["bits"] // 8 + 2 * _groups(case))


def work(case):
    e = _SIZE[case["dtype"]]
    if case["kind"] == "nbits":
        m, k, n = case["m"], case["k"], case["n"]
        nb = -(-k // case["block"])
        weights = n * k // 2 + n * nb * e + (n * ((nb + 1) // 2) if case["zp"] else 0) + (n * e if case["bias"] else 0)
        return dict(bytes=(m * k + m * n) * e + weights, flops=2 * m * k * n)
    B, S, D = case["batch"], case["seq"], case["hd"]
    if case["kind"] == "cache":
        # read the new tokens, write them; read them again, write the values
        elems = 2 * B * S * case["kv_heads"] * D
        return dict(bytes=2 * (elems * e + B * S * _token_bytes(case)), flops=6 * elems)
    # lengths are uniform from seq to longest
    keys = B * (case["seq"] + case["longest"]) / 2 + case["prefix"]
    per_row = case["prefix"] + (case["seq"] + case["longest"]) / 2 - (S - 1) / 2
    return dict(bytes=int(2 * B * S * case["q_heads"] * D * e + keys * _token_bytes(case)),
                flops=int(4 * B * S * case["q_heads"] * D * per_row))


# ---------------------------------------------------------------------------
# the definitions in 64 bits

def _exact_values(case, x):
    """What the cache holds for x [..., hd]: code * scale, in 64 bits."""
    limit = 127.0 if case["bits"] == 8 else 7.0
    size = case["hd"] if case["bits"] == 8 else 32
    parts = []
    for at in range(0, case["hd"], size):
        part = x[..., at:at + size].double()
        top = part.abs().max(-1, keepdim=True).values / limit
        scale = _round_bf16(top)
        code = torch.clamp(torch.round(part / torch.where(scale == 0, torch.ones_like(scale), scale)), -limit, limit)
        parts.append(code * scale)
    return torch.cat(parts, -1)


def _round_bf16(x):
    """x > 0 rounded to 8 significant bits, ties to even."""
    m, e = torch.frexp(x)
    return torch.ldexp(torch.round(m * 256.0) / 256.0, e)


def exact(case, seed):
    if case["kind"] == "nbits":
        x = _nbits_inputs(case, seed)
        n, k, block = case["n"], case["k"], case["block"]
        kk = torch.arange(k, device="cuda")
        byte = x["b"].reshape(n, -1)[:, kk // 2].int()
        q = torch.where(kk % 2 == 1, byte // 16, byte % 16).double()
        blk = kk // block
        if case["zp"]:
            byte = x["zp"][:, blk // 2].int()
            q -= torch.where(blk % 2 == 1, byte // 16, byte % 16).double()
        else:
            q -= 8.0
        q *= x["scales"].double()[:, blk]
        y = x["a"].double() @ q.t()
        return y + x["bias"].double() if case["bias"] else y
    x = _cache_inputs(case, seed)
    if case["kind"] == "cache":
        # rounded to the tensors' type once, as any reader of the cache gets them
        return tuple(_exact_values(case, x[n]) for n in "kv")
    B, S, D, H, P = case["batch"], case["seq"], case["hd"], case["kv_heads"], case["prefix"]
    G = case["q_heads"] // H
    lens = x["lens"].tolist()
    y = torch.empty((B, S, case["q_heads"], D), dtype=torch.float64, device="cuda")
    for h in range(H):
        pk = _exact_values(case, x["pk"][0, :, h]) if P else x["q"].new_zeros((0, D), dtype=torch.float64)
        pv = _exact_values(case, x["pv"][0, :, h]) if P else pk
        for b in range(B):
            n = lens[b]
            # the positions in the cache were written as one run that ends at `longest`
            keys = torch.cat((pk, _exact_values(case, x["k"][b, :n, h])))
            vals = torch.cat((pv, _exact_values(case, x["v"][b, :n, h])))
            q = x["q"][b, :, h * G:(h + 1) * G].double().reshape(S * G, D)
            sc = torch.mm(q, keys.t()) * D ** -0.5
            if S > 1:
                own_pos = torch.arange(n, device="cuda")
                query = torch.arange(S, device="cuda").repeat_interleave(G)
                sc[:, P:] = torch.where(own_pos[None] <= (n - S + query)[:, None], sc[:, P:], -math.inf)
            y[b, :, h * G:(h + 1) * G] = torch.mm(torch.softmax(sc, -1), vals).reshape(S, G, D)
    return y
