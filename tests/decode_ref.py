"""Plain forms of the decoder operators in 64 bits, and how far a kernel that
sums in fp32 may be from them."""
import numpy as np
import torch

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}   # half a step, relative
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}   # the same below the normal numbers
U = 2.0 ** -23   # one fp32 operation, also where it cuts instead of rounding


# from here on a value rounds to infinity: half a step past the largest number
OVERFLOW = {t: torch.finfo(t).max * (1 + HALF[t] / (2 - 2 * HALF[t])) for t in HALF}


def close(y, ref, tol, t):
    """Within tol; or the infinity that a reference of that size, give or take tol, rounds to."""
    with np.errstate(invalid="ignore"):
        inf = np.isinf(y) & (np.sign(y) == np.sign(ref)) & (np.abs(ref) + tol >= OVERFLOW[t])
        return (np.abs(y - ref) <= tol) | inf


def unpack(b):
    return np.stack((b & 15, b >> 4), -1).reshape(*b.shape[:-1], -1)


def nbits(a, b, scales, k, block, zp, bias):
    """(y, sum |a w| + |bias|) in float64; a [m][k], b [n][nb][block / 2]."""
    n, nb = b.shape[:2]
    q = unpack(b).reshape(n, nb, block).astype(np.float64)
    z = 8.0 if zp is None else unpack(zp.reshape(n, -1))[:, :nb, None].astype(np.float64)
    w = ((q - z) * scales.astype(np.float64)[:, :, None]).reshape(n, nb * block)[:, :k]
    a = a.astype(np.float64)
    y, mag = a @ w.T, np.abs(a) @ np.abs(w).T
    if bias is not None:
        y, mag = y + bias, mag + np.abs(bias)
    return y, mag


def nbits_tol(y, mag, k, t):
    # a chain of sums: 32 products (three pieces each for fp32), the K / 32
    # scaled block sums, 8 waves, bias, scaling
    n = 3 * 32 + (k + 31) // 32 + 8 + 4
    return n * U * mag + HALF[t] * np.abs(y) + TINY[t]


def quantize(x, bits):
    """What a cache holds for x [..., hd] (a float tensor), in float64: (values, codes, scales)."""
    L = 127.0 if bits == 8 else 7.0
    size = x.shape[-1] if bits == 8 else 32
    v = x.double().reshape(*x.shape[:-1], x.shape[-1] // size, size)
    fin = torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v))
    top = fin.amax(-1, keepdim=True) / L
    m, e = torch.frexp(top)
    s = torch.ldexp(torch.round(m * 256) / 256, e)
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    c = torch.round(v / torch.where(s > 0, s, torch.ones_like(s))).clamp(-L, L)
    c = torch.where(torch.isnan(v) | (s == 0), torch.zeros_like(c), c)
    return (c * s).reshape(x.shape), c.reshape(x.shape), s.squeeze(-1)


def attention(q, keys, vals, scale, visible):
    """One sequence and key/value head, float64. q [S, G, hd], keys / vals
    [n, hd], visible [S] counts of keys seen. Returns (y, tolerance terms)."""
    S, G, hd = q.shape
    floor = 2.0 ** -39 if q.dtype == torch.float32 else 2.0 ** -35
    q = q.double()
    y, tol = torch.zeros(S, G, hd, dtype=torch.float64), torch.zeros(S, G, hd, dtype=torch.float64)
    for s in range(S):
        n = int(visible[s])
        if n == 0:
            continue
        sc = q[s] @ keys[:n].T * scale
        p = torch.softmax(sc, -1)
        y[s], mag = p @ vals[:n], p @ vals[:n].abs()
        size = (q[s].abs() @ keys[:n].abs().T * abs(scale)).amax(-1, keepdim=True)
        # fp16 has no steps below 2^-24. A query's elements are rounded to such
        # a half step of a row scaled to 2^14 and more: 2^-25 / 2^14 of the
        # largest. A weight p times 2^15 (2^11 for fp16 and bf16 tensors; times
        # its value's scale over the unit u, a power of two at most twice the
        # largest scale) is rounded so too: 2^-40 u (2^-36 u) a code, so twice
        # that of the largest value a key.
        low = 2.0 ** -39 * q[s].abs().amax() * keys[:n].abs().sum(-1).amax() * abs(scale)
        tol[s] = mag * (2 * size * (hd + 16) * U + 2 * low + (64 + n / 8) * U) + n * floor * vals[:n].abs().amax()
    return y, tol


def attention_tol(y, mag_tol, weighted, t):
    """mag_tol: attention()'s; weighted: sum p |v|, for the rounding of weights
    to one (fp16, bf16) or two fp16 pieces (fp32)."""
    return mag_tol + (2.0 ** -11 if t != torch.float32 else 2.0 ** -21) * weighted + HALF[t] * y.abs() + TINY[t]


def nbits_graph(dt=np.float32, block=32, K=70, N=24, zp=True, bias=True, shape=(2, 3, 70), scale_dt=None, drop=0, attrs=()):
    """A graph of one MatMulNBits node. drop: bytes missing from the weights."""
    from nnr_amd.graph import Graph
    rng = np.random.default_rng(1)
    nb = -(-K // block)
    g = Graph()
    g.inputs["x"] = (dt, shape)
    b = rng.integers(0, 256, (N, nb, block // 2), dtype=np.uint8)
    ins = ["x", g.init("b", b.reshape(-1)[drop:] if drop else b),
           g.init("s", rng.uniform(0.01, 0.1, (N, nb)).astype(scale_dt or dt)),
           g.init("z", rng.integers(0, 256, (N, (nb + 1) // 2), dtype=np.uint8)) if zp else "", "",
           g.init("c", rng.standard_normal(N).astype(dt)) if bias else ""]
    g.node("MatMulNBits", ins, outputs="y", **{**dict(K=K, N=N, bits=4, block_size=block), **dict(attrs)})
    g.outputs.append("y")
    return g
