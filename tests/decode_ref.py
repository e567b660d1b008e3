"""Plain 64-bit forms of a decoding step's products and of the next token's choice, on the CPU."""
from __future__ import annotations

import math
from fractions import Fraction

import numpy as np

# type number: values and bytes of a block, where its fp16 fields lie
BLOCKS = {2: (32, 18, (0,)), 3: (32, 20, (0, 2)), 8: (32, 34, (0,)), 12: (256, 144, (0, 2)), 20: (32, 18, (0,)), 23: (256, 136, (0,))}
LEVELS = np.array([-127, -104, -83, -65, -49, -35, -22, -10, 1, 13, 25, 38, 53, 69, 89, 113], dtype=np.float64)


def gguf(wtype: int, n: int, k: int, seed: int = 0, scale: float = 0.01) -> np.ndarray:
    """n rows of random codes and integer scales, with fp16 scales of either sign."""
    rng = np.random.default_rng([seed, wtype, n, k])
    values, size, halves = BLOCKS[wtype]
    raw = rng.integers(0, 256, (n, k // values, size), dtype=np.uint8)
    for at in halves:
        d = (scale * rng.uniform(0.25, 2.0, (n, k // values)) * rng.choice([-1.0, 1.0], (n, k // values))).astype(np.float16)
        raw[:, :, at:at + 2] = d[..., None].view(np.uint8)
    return raw.reshape(n, -1)


def parts(wtype: int, raw: np.ndarray, k: int):
    """(a, b) of each value, which stands for a + b, [n][k] in 64 bits."""
    values, size, _ = BLOCKS[wtype]
    n = raw.shape[0]
    r = raw.reshape(n, k // values, size)
    half = lambda at: r[:, :, at:at + 2].copy().view(np.float16)[:, :, 0].astype(np.float64)  # noqa: E731
    a, b = np.zeros((n, k // values, values)), np.zeros((n, k // values, values))
    d = half(0)
    for i in range(values):
        if wtype == 8:
            a[:, :, i] = d * r[:, :, 2 + i].view(np.int8)
            continue
        s, e = divmod(i, 32)  # sub-block and place in it
        if wtype == 12:
            q = r[:, :, 16 + 32 * (s // 2) + e] >> 4 * (s % 2) & 15
            if s < 4:
                sc, m = r[:, :, 4 + s] & 63, r[:, :, 8 + s] & 63
            else:
                sc = r[:, :, 8 + s] & 15 | r[:, :, s] >> 6 << 4
                m = r[:, :, 8 + s] >> 4 | r[:, :, 4 + s] >> 6 << 4
            a[:, :, i], b[:, :, i] = d * sc * q, -half(2) * m
            continue
        first = {2: 2, 3: 4, 20: 2, 23: 8 + 16 * s}[wtype]
        q = r[:, :, first + e % 16] >> 4 * (e // 16) & 15
        if wtype == 23:
            high = (r[:, :, 2].astype(int) | r[:, :, 3].astype(int) << 8) >> 2 * s & 3
            a[:, :, i] = d * ((r[:, :, 4 + s // 2] >> 4 * (s % 2) & 15) + 16 * high - 32.0) * LEVELS[q]
        elif wtype == 20:
            a[:, :, i] = d * LEVELS[q]
        elif wtype == 2:
            a[:, :, i] = d * (q.astype(np.float64) - 8)
        else:
            a[:, :, i], b[:, :, i] = d * q, half(2)
    return a.reshape(n, k), b.reshape(n, k)


def matvec(wtype: int, x: np.ndarray, raw: np.ndarray):
    """y [m][n] in 64 bits, and how far a kernel may be off: x to 2^-22 of the largest magnitude in its 32, met by each
    part of a weight; sums in fp32 of at most one term each 16 values, each part's, and 24 roundings of a term's own."""
    k = x.shape[1]
    a, b = parts(wtype, raw, k)
    xd = x.astype(np.float64)
    largest = np.repeat(np.abs(xd).reshape(len(x), k // 32, 32).max(axis=2), 32, axis=1)
    size = np.abs(a) + np.abs(b)
    return xd @ (a + b).T, 2.0 ** -22 * (largest @ size.T) + (2 * (k // 16) + 24) * 2.0 ** -24 * (np.abs(xd) @ size.T)


def glu(kind: int, g: np.ndarray, u: np.ndarray) -> np.ndarray:
    if kind == 0:
        return np.where(g > 0, g * u, 0.0)
    if kind == 1:
        return 0.5 * g * (1 + np.tanh(0.7978845608 * g * (1 + 0.044715 * g * g))) * u
    if kind == 2:
        return g / (1 + np.exp(-g)) * u
    if kind == 3:
        return 0.5 * g * (1 + np.vectorize(math.erf)(g * 0.7071067812)) * u
    return g / (1 + np.exp(-1.702 * g)) * u


def glu_bound(g, eg, u, eu):
    """The GLUs' slopes are at most 1.2 (of every kind), their value at most |g u|, computed in fp32 to 2^-20 of that."""
    return 1.2 * (np.abs(u) * eg + np.abs(g) * eu + eg * eu) + 2.0 ** -20 * np.abs(g * u)


# ---- the next token ---------------------------------------------------------------

ONE = 2 ** 45


def kept(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row of logits -> (indices that stay, in index order, their integer weights)."""
    x = np.where(np.isnan(x), -np.inf, np.asarray(x, dtype=np.float64))
    top = x.max()
    if top == -np.inf:
        return [], []
    if not temperature > 0:
        return [int(np.argmax(x))], [ONE]
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        w = np.where(x == top, 1.0, np.where((x > -np.inf) & (top < np.inf), np.exp((x - top) * (1.0 / np.float64(temperature))), 0.0))
    whole = [int(v) for v in np.rint(w * ONE)]
    order = list(np.argsort(-x, kind="stable"))
    if 0 < top_k < len(x):
        order = order[:top_k]
    if top_p < 1:
        goal = max(Fraction(1), Fraction(max(float(np.float32(top_p)), 0.0)) * sum(whole[i] for i in order))
        n, run = 0, 0
        while n < len(order) and run < goal:
            run += whole[order[n]]
            n += 1
        order = order[:n]
    m = min(float(np.float32(min_p)), 1.0) if min_p > 0 else 0.0
    order = sorted(int(i) for i in order if w[i] >= m and whole[i] > 0)
    return order, [whole[i] for i in order]


def fits(token: int, prob: float, stay, weights, u: float) -> bool:
    """Whether a token and its probability are the draw at u. The 64-bit exponentials of two programs may be a unit
    apart each (2^-45), so a border may lie 2^-45 of the row's count away: 2^-27 for the longest row."""
    if not stay:
        return token == -1 and prob == 0
    if token not in stay:
        return False
    at, total = stay.index(token), sum(weights)
    u = min(max(float(np.float32(u)), 0.0), 1.0) if u == u else 0.0
    before, slack = Fraction(sum(weights[:at]), total), Fraction(len(stay), ONE)
    share = Fraction(weights[at], total)
    inside = before - slack <= Fraction(u) < before + share + slack or (u >= 1.0 and at == len(stay) - 1)
    return inside and abs(prob - float(share)) <= 2.0 ** -23 * float(share) + 1e-30
