"""Attention over a quantized cache where queries, keys and values of one call
are of very different sizes: inputs, and how far a kernel may be from float64.

The bound is by key and by group of elements (32, or a whole head at 8 bits), so
that what is large elsewhere does not hide an error. With p_j the weights and
|v_j| an element's value:
  - the score of key j is a sum of hd products in fp32, (hd + 16) U of sum |q k_j|
    (fp32 queries are two fp16 pieces, 2^-22 more); a query's element keeps half
    a step of fp16 below a row scaled to 2^14: 2^-39 of the row's largest;
  - scores enter an exponential as a difference of two of them, U of each;
  - a weight changes by its score's error, and so do all by their sum: twice
    sum p_j e_j |v_j| and |y| sum p_j e_j;
  - weights are rounded to 11 bits (two pieces of fp16, 22 bits, for fp32), both
    where they meet values and, at 4 bits, where they are summed: 2^-11 (2^-21) of
    sum p |v| and |y|;
  - below that a weight has an fp16 step of its own: a half of it, over the largest
    weight, is 2^-36 (2^-40) of a key's own value at 4 bits, where that is up to
    2^18 of the group's smallest. At 8 bits the value's scale is in the weight,
    and the step is of the row's largest product of the two, 2^-23 for each key
    (no coarser than a step of an fp32 sum);
  - n keys' products are summed in fp32, in parts: (64 + n / 8) U of sum p |v|;
  - the result is rounded once."""
import torch

import decode_ref as R


def attention(q, keys, vals, scale, visible, bits):
    """One sequence and key/value head. q [S, G, hd], keys / vals [n, hd] in float64,
    visible [S]. Returns (y, how far off it may be)."""
    t, (S, G, hd) = q.dtype, q.shape
    size = hd if bits == 8 else 32
    one, floor, two = (2.0 ** -11, 2.0 ** -36, 0.0) if t != torch.float32 else (2.0 ** -21, 2.0 ** -40, 2.0 ** -22)
    q = q.double()
    y, tol = torch.zeros(S, G, hd, dtype=torch.float64), torch.zeros(S, G, hd, dtype=torch.float64)
    for s in range(S):
        n = int(visible[s])
        if n == 0:
            continue
        k, v = keys[:n], vals[:n]
        sc = q[s] @ k.T * scale
        p = torch.softmax(sc, -1)
        e = abs(scale) * (((hd + 16) * R.U + two) * (q[s].abs() @ k.abs().T) +
                          2 * 2.0 ** -39 * q[s].abs().amax(-1, keepdim=True) * k.abs().sum(-1))
        e = e + 4 * R.U * (sc.abs() + sc.amax(-1, keepdim=True).abs()) + 16 * R.U
        y[s] = p @ v
        mag = p @ v.abs()
        top = v.abs().reshape(n, hd // size, size).amax(-1)                       # [n, groups]
        if bits == 4:
            least = torch.where(top > 0, top, torch.full_like(top, float("inf"))).amin(0)
            low = n * floor * torch.minimum(top.amax(0), 2.0 ** 18 * least).expand(G, -1)
        else:
            low = n * 2.0 ** -23 * (p[..., None] * top).amax(1)
        tol[s] = (2 * (p * e.clamp(max=1.0)) @ v.abs() + y[s].abs() * (p * e.clamp(max=1.0)).sum(-1, keepdim=True) + one * (mag + y[s].abs()) +
                  (64 + n / 8) * R.U * mag + low.repeat_interleave(size, -1) + R.HALF[t] * y[s].abs() + R.TINY[t])
    return y, tol


# (sequences' lengths, new tokens, heads, query heads a head, head size, prefix, pages of 32 a sequence)
SHAPES = {
    "one block": ([150], 1, 1, 2, 64, 0, 5),
    "wide": ([150, 40], 1, 1, 4, 128, 0, 5),
    "splits": ([1100, 300], 1, 2, 4, 128, 0, 80),
    "several": ([200, 33, 5], 3, 1, 4, 96, 70, 7),
    "prefix": ([40, 9] + [3] * 38, 1, 1, 4, 128, 500, 2),
    "prompt": ([150, 120], 64, 1, 2, 64, 200, 5),
    "large heads": ([100, 60], 20, 1, 1, 256, 90, 4),
}


def sizes(shape):
    return shape if isinstance(shape, tuple) else SHAPES[shape]


def inputs(pattern, shape, t, seed=0):
    """q [B, S, H G, hd], own k and v [B, longest, H, hd] (a sequence's last tokens are its own) and the
    prefix's [1, P, H, hd]. Every key is 1/4 of the way to a query of ones, so that a token of
    -1s is hardly seen."""
    lens, S, H, G, hd, P, _ = sizes(shape)
    B, n = len(lens), max(lens)
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)
    q, k, v = r(B, S, H * G, hd).abs(), r(B, n, H, hd), r(B, n, H, hd)
    pk, pv = r(1, P, H, hd), r(1, P, H, hd)
    # fp16 has 40 binary orders in all
    far = 20 if t == torch.float16 else 40
    steps = torch.arange(hd // 32).repeat_interleave(32)
    if pattern.startswith("key groups"):
        # queries see the last group alone, that far below the others
        gap = int(pattern.split()[-1])
        f = torch.where(steps == hd // 32 - 1, 2.0 ** (12 - gap), 2.0 ** 12)
        k, pk = k * f, pk * f
        q = torch.where(steps == hd // 32 - 1, q * 2.0 ** (gap - 12) * (hd / 32) ** 0.5, torch.zeros(()))
    elif pattern == "key tokens":
        # one token in fifty far larger, and hardly seen
        k, pk, q = k * 2.0 ** -9, pk * 2.0 ** -9, q * 2.0 ** 9
        for x in (k, pk):
            x[:, 7::50] = -x[:, 7::50].abs() * 2.0 ** (far + 2)
    elif pattern == "value groups":
        f = 2.0 ** (10 - (far * 3 // 4) * steps.double() / max(1, hd // 32 - 1))
        v, pv = v * f, pv * f
    elif pattern == "value tokens":
        # the same for values: what is large is hardly seen, before and behind what is small
        v, pv = v * 2.0 ** -8, pv * 2.0 ** -8
        for x, y in ((k, v), (pk, pv)):
            x[:, 11::45] = -8.0
            y[:, 11::45] *= 2.0 ** (far + 1)
    elif pattern == "seen later":
        # the newest token alone is large: other queries of the call do not see it
        v, pv = v * 2.0 ** -8, pv * 2.0 ** -8
        v[:, -1] *= 2.0 ** (far + 1)
    elif pattern == "rare and large":
        # values so large that small weights count
        k[:, 5::60], pk[:, 5::60] = -1.0, -1.0
        v[:, 5::60] *= 2.0 ** (12 if t == torch.float16 else 30)
        pv[:, 5::60] *= 2.0 ** (12 if t == torch.float16 else 30)
    return q.to(t), k.to(t), v.to(t), pk.to(t), pv.to(t)


PATTERNS = ["key groups 20", "key groups 24", "key tokens", "value groups", "value tokens", "seen later", "rare and large"]
