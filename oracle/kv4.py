"""Plain 64-bit forms of the 4-bit paged cache and the attention over it (numpy,
loops): what the kernels of rhinoforge_amd/csrc/kv4_* are checked against.
Row-major numbers [blocks, kv_heads, block_size, head_dim], steps and zero points
[blocks, kv_heads, block_size] throughout."""
from __future__ import annotations

import math

import numpy as np

LEAST, MOST = 2.0 ** -20, 4352.0


def axis_of_pairs(sections, mixed):
    """The axis of each rotated pair, by the words of the definition."""
    if not mixed:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    axes = len(sections)
    return [i % axes if i // axes < sections[i % axes] else 0 for i in range(sum(sections))]


def step_of(low, high):
    """(span, the least step of seven bits with 15 of it at least the span)."""
    with np.errstate(over="ignore"):
        span = float(np.float32(high) - np.float32(low))
    if span <= 15 * LEAST or span >= 15 * MOST:
        return span, LEAST if span <= 15 * LEAST else MOST
    unit = max(2.0 ** (math.frexp(span / 15)[1] - 7), LEAST)
    return span, min(math.ceil(span / 15 / unit) * unit, MOST)


def quantize(x):
    """x [..., D] finite -> (numbers, steps, zero points), all float64."""
    flat = x.reshape(-1, x.shape[-1]).astype(np.float64)
    n, s, z = np.zeros_like(flat), np.zeros(len(flat)), np.zeros(len(flat))
    for i, row in enumerate(flat):
        low = min(row.min(), 0.0)
        s[i] = step_of(low, max(row.max(), 0.0))[1]
        z[i] = min(np.rint(-low / s[i]), 15)
        n[i] = np.clip(np.rint(row / s[i]) + z[i], 0, 15)
    return n.reshape(x.shape), s.reshape(x.shape[:-1]), z.reshape(x.shape[:-1])


def values(n, s, z):
    return (n.astype(np.float64) - z.astype(np.float64)[..., None]) * s.astype(np.float64)[..., None]


def append(held, x, slots):
    """held (numbers, steps, zero points), x [T, H, D]; copies with the tokens entered."""
    n, s, z = (a.astype(np.float64).copy() for a in held)
    bs = n.shape[2]
    for t, slot in enumerate(slots):
        if 0 <= slot < n.shape[0] * bs:
            n[slot // bs, :, slot % bs], s[slot // bs, :, slot % bs], z[slot // bs, :, slot % bs] = quantize(x[t])
    return n, s, z


def attention(q, k, v, table, lens, cu, causal=True, window=0, scale=1.0, kmag=None):
    """q [T, H, D], k, v: held values -> out [T, H, D], lse [T, H] and what bounds a
    kernel's error: mass [T, H, D] = sum p |v| / sum p, size [T, H] = max_j sum_d
    |q_d| kmag_jd scale (kmag: |k| where not given).  Block ids outside the cache
    stand for NaN."""
    T, H, D = q.shape
    nb, hk, bs = k.shape[:3]
    g = H // hk
    kmag = np.abs(k) if kmag is None else kmag
    out, mass = np.zeros((T, H, D)), np.zeros((T, H, D))
    lse, size = np.full((T, H), -np.inf), np.zeros((T, H))
    for r, length in enumerate(lens):
        n = cu[r + 1] - cu[r]
        ids = np.asarray(table[r, : -(-length // bs)])
        bad = np.repeat((ids < 0) | (ids >= nb), bs)[:length]
        ids = np.where((ids < 0) | (ids >= nb), 0, ids)
        for h in range(hk):
            kh, vh, mh = (a[ids, h].reshape(-1, D)[:length] for a in (k, v, kmag))
            kh = np.where(bad[:, None], np.nan, kh)
            for i in range(n):
                pos = length - n + i
                lo, hi = 0, length
                if causal:
                    hi = min(length, pos + 1)
                    if window:
                        lo = max(0, pos - window + 1)
                if hi <= lo:
                    continue
                at = (cu[r] + i, slice(h * g, (h + 1) * g))
                x = q[cu[r] + i, h * g:(h + 1) * g].astype(np.float64)  # [g, D]
                s = x @ kh[lo:hi].T * scale
                m = s.max(-1, keepdims=True)
                p = np.exp(s - m)
                l = p.sum(-1, keepdims=True)
                out[at] = p @ vh[lo:hi] / l
                mass[at] = p @ np.abs(vh[lo:hi]) / l
                lse[at] = (m + np.log(l))[:, 0]
                size[at] = (np.abs(x) @ mh[lo:hi].T).max(-1) * scale
    return out, lse, mass, size
