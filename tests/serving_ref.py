"""Plain forms in 64 bits of the operators around a decoder's cache, and how far
kernels that sum in fp32 may be from them."""
import numpy as np
import torch

from decode_ref import HALF, TINY, U


def attend(q, keys, vals, scale, sees, floor):
    """One sequence and key/value head in float64. q [S, G, hd], keys / vals [n, hd],
    sees bool [S, n]. Returns (y, weighted = sum p |v|, tolerance of scores and sums
    in fp32). A row that sees nothing gives 0. floor: what a weight may be off by in
    parts of the largest, whatever its size (steps of small fp16 numbers)."""
    S, G, hd = q.shape
    n = keys.shape[0]
    if n == 0:
        return tuple(torch.zeros(S, G, hd, dtype=torch.float64) for _ in range(3))
    keys, vals = torch.nan_to_num(keys.double(), 0, 0, 0), torch.nan_to_num(vals.double(), 0, 0, 0)
    q = q.double()
    sc = torch.matmul(q, keys.t()) * scale                                 # [S, G, n]
    sc = sc.masked_fill(~sees[:, None], float("-inf"))
    some = sees.any(-1)[:, None, None]
    top = sc.amax(-1, keepdim=True)
    p = torch.where(some, torch.exp(sc - torch.where(some, top, 0)), 0)
    p = p / torch.where(some, p.sum(-1, keepdim=True), 1)
    y, weighted = torch.matmul(p, vals), torch.matmul(p, vals.abs())
    size = torch.where(sees[:, None], torch.matmul(q.abs(), keys.abs().t()) * abs(scale), 0).amax(-1, keepdim=True)
    # A score sums hd products (size times U each), and twice rounds numbers of its
    # size in powers of two; a weight is off by as much relative to itself, the largest
    # and so all of them by as much again. Sums round once a key at most, their
    # rescaling once a tile; exp2, the reciprocal and the product a few times.
    largest = torch.where(sees[:, :, None], vals.abs(), 0).amax((1, 2))[:, None, None]
    tol = weighted * (2 * size * (hd + 16) * U + (64 + n) * U) + n * floor * largest
    return y, weighted, tol


def rounded(y, weighted, tol, t, weights):
    """tol, and the rounding of weights (`weights` relative) and of the result."""
    return tol + weights * weighted + HALF[t] * y.abs() + TINY[t]


# Prompts: 16-bit weights are rounded to the values' type, as 2^11 p and more in
# fp16, whose steps of small numbers are 2^-24
PROMPT_WEIGHTS = {torch.float32: 0.0, torch.float16: HALF[torch.float16], torch.bfloat16: HALF[torch.bfloat16]}
PROMPT_FLOOR = {torch.float32: 0.0, torch.float16: 2.0 ** -36, torch.bfloat16: 0.0}
# The cache's attention: as its own reference has it (queries of a row with a
# common power of two as well)
CACHE_WEIGHTS = {torch.float32: 2.0 ** -21, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -11}
CACHE_FLOOR = {torch.float32: 2.0 ** -39, torch.float16: 2.0 ** -35, torch.bfloat16: 2.0 ** -35}


def prompt(q, k, v, starts, scale, causal):
    """(y, tolerance) of packed prompts, float64; NaN where no sequence has the token."""
    T, Hq, hd = q.shape
    G = Hq // k.shape[1]
    t = q.dtype
    y, tol = torch.full((T, Hq, hd), float("nan"), dtype=torch.float64), torch.zeros((T, Hq, hd), dtype=torch.float64)
    for s, e in zip(starts[:-1], starts[1:]):
        n = e - s
        sees = torch.ones((n, n), dtype=torch.bool).tril() if causal else torch.ones((n, n), dtype=torch.bool)
        for h in range(k.shape[1]):
            if not n:
                continue
            r, w, tl = attend(q[s:e, h * G:(h + 1) * G], k[s:e, h], v[s:e, h], scale, sees, PROMPT_FLOOR[t])
            y[s:e, h * G:(h + 1) * G], tol[s:e, h * G:(h + 1) * G] = r, rounded(r, w, tl, t, PROMPT_WEIGHTS[t])
    return y, tol


def frequencies(r, base, scaling="none", factor=1.0, original=None):
    """One by one, as the formulas have them: (angles a position, a factor)."""
    out, m = [], 1.0
    for i in range(r // 2):
        f = base ** (-2 * i / r)
        if scaling == "linear":
            f /= factor
        elif scaling == "ntk":
            f = (base * factor ** (r / (r - 2))) ** (-2 * i / r)
        elif scaling == "yarn":
            turns = original * f / (2 * np.pi)
            keep = 0.0 if turns <= 1 else 1.0 if turns >= 32 else (turns - 1) / 31
            f = keep * f + (1 - keep) * f / factor
            m = 0.1 * np.log(factor) + 1
        out.append(f)
    return np.array(out), m


def rotate(x, pos, freqs, m, interleaved, held):
    """(y, tolerance) in float64. x [B, S, H, hd], pos [B, S]"""
    r = 2 * len(freqs)
    y, tol = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64)
    angle = pos.double()[..., None] * torch.from_numpy(freqs)
    c, s = (m * f(angle).unsqueeze(2) for f in (torch.cos, torch.sin))
    at = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    a, b = x[..., at[0]].double(), x[..., at[1]].double()
    turn = (pos >= 0)[..., None, None]
    for i, (p, q) in enumerate(((a * c, -b * s), (b * c, a * s))):
        z = torch.where((pos >= held)[..., None, None], float("nan"), p + q)
        y[..., at[i]] = torch.where(turn, z, (a, b)[i])
        # the table's rounding, the product's and the sum's
        tol[..., at[i]] = torch.where(turn, 3 * 2.0 ** -24 * (p.abs() + q.abs()) + HALF[x.dtype] * (p + q).abs() + TINY[x.dtype], 0)
    return y, tol
