"""The operators on 4-bit cache pages in numpy, 64 bits: what pages hold, decode attention, the weight that positions receive, eviction."""
from __future__ import annotations

import numpy as np

GROUP, MOST, NOTHING = 32, np.float32(65504.0), np.float32(2.0 ** -80)


def bf16(x):
    """FP32 rounded to BF16, to the nearest, ties to even."""
    u = np.asarray(x, dtype=np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16 << 16).astype(np.uint32).view(np.float32)


def quantise(x):
    """FP32 [..., dim] -> (numbers [..., groups, 32], d, m [..., groups, 1]): each group's numbers and its factors as they are held."""
    g = np.asarray(x, dtype=np.float32).reshape(*x.shape[:-1], -1, GROUP)
    nan = np.isnan(g).any(-1, keepdims=True)
    g = np.clip(np.where(nan, np.float32(0), g), -MOST, MOST)
    lo, reach = g.min(-1, keepdims=True), g.max(-1, keepdims=True) - g.min(-1, keepdims=True)
    m = lo.astype(np.float16).astype(np.float64)
    d = np.where(reach < NOTHING, 0.0, bf16(reach / np.float32(15)).astype(np.float64))
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where(d > 0, np.clip(np.rint((g.astype(np.float64) - m) / d), 0, 15), 0.0)
    return np.where(nan, 0.0, q), np.where(nan, 0.0, d), np.where(nan, np.nan, m)


def held(x):
    """The values that pages hold for x, in 64 bits (the framework gives them rounded to FP32)."""
    q, d, m = quantise(x)
    return (m + d * q).reshape(x.shape)


def attention(q, k, v):
    """q [heads, dim], k and v [positions, kv heads, dim] -> out [heads, dim] and each position's weight, summed over the heads of a key/value head."""
    heads, dim = q.shape
    n, kv, _ = k.shape
    if n == 0:
        return np.zeros((heads, dim)), np.zeros((kv, 0))
    s = np.einsum("hgd,lhd->hgl", q.astype(np.float64).reshape(kv, -1, dim), k) / np.sqrt(dim)
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    return np.einsum("hgl,lhd->hgd", p, v).reshape(heads, dim), p.sum(1)


def kept(w, keep, recent):
    """Places of one head that stay: the newest `recent` ones and, of the others, those of most weight, the earlier of two equal ones."""
    n = len(w)
    if n <= keep:
        return np.arange(n)
    old = np.asarray(w[:n - recent], dtype=np.float64)
    order = sorted(range(n - recent), key=lambda j: (1, 0.0, j) if np.isnan(old[j]) else (0, -old[j], j))
    return np.array(sorted(order[:keep - recent]) + list(range(n - recent, n)))
