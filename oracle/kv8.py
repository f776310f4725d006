"""Plain 64-bit forms of the attention over an int8 paged cache (numpy, loops):
what the kernels of rhinoforge_amd/csrc/kv8_* are checked against.  Row-major
int8 caches [blocks, kv_heads, block_size, head_dim] throughout."""
from __future__ import annotations

import numpy as np


def norm_rope(x, weight, cos, sin, positions, eps, interleaved):
    """x [T, H, D]; weight [D] or None; cos, sin [R, rot / 2] or None; all float64."""
    y = x.astype(np.float64)
    if weight is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * weight
    if cos is None:
        return y
    half = cos.shape[1]
    out = y.copy()
    for t in range(y.shape[0]):
        row = positions[t] if positions is not None else t
        if not 0 <= row < cos.shape[0]:
            out[t] = np.nan
            continue
        for i in range(half):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
            c, s = cos[row, i], sin[row, i]
            out[t, :, a] = y[t, :, a] * c - y[t, :, b] * s
            out[t, :, b] = y[t, :, b] * c + y[t, :, a] * s
    return out


def plan(table, cached, new, free, start, num_tokens, bs):
    """(table, slots, positions, cu, kv_lens, free_next); the table is a copy."""
    table, nxt = table.copy(), max(int(start), 0)
    slots, pos, cu, lens = [], [], [0], []
    for i in range(len(cached)):
        c, n = max(int(cached[i]), 0), max(int(new[i]), 0)
        for j in range(-(-c // bs), -(-(c + n) // bs)):
            if j < table.shape[1]:
                table[i, j] = free[nxt] if nxt < len(free) else -1
            nxt += 1
        for p in range(c, c + n):
            block = table[i, p // bs] if p // bs < table.shape[1] else -1
            slots.append(block * bs + p % bs if block >= 0 else -1)
            pos.append(p)
        cu.append(cu[-1] + n)
        lens.append(c + n)
    slots, pos = slots[:num_tokens], pos[:num_tokens]
    pad = num_tokens - len(slots)
    return (table, np.array(slots + [-1] * pad, np.int64), np.array(pos + [0] * pad, np.int64),
            np.array(cu, np.int64), np.array(lens, np.int64), nxt)


def append(q, scale, x, slots):
    """x [T, H, D] float64 into q, scale (copies returned).  Also returns the
    quotients (before rounding) of every value written or rounded again."""
    bs = q.shape[2]
    q, scale = q.astype(np.float64), scale.astype(np.float64)
    quot = q.copy()
    t = 0
    while t < len(slots):
        n = 1
        while (t + n < len(slots) and slots[t] >= 0 and slots[t + n] == slots[t] + n
               and slots[t + n] // bs == slots[t] // bs):
            n += 1
        b, o = slots[t] // bs, slots[t] % bs
        if slots[t] >= 0 and b < q.shape[0]:
            new = x[t:t + n].transpose(1, 0, 2)
            amax = np.abs(new).max((1, 2))
            step = np.where(amax < 2.0 ** -100, 0.0, amax / 127)
            if o > 0:
                before = scale[b]
                step = np.maximum(before, step)
                ratio = np.where(step > before, before / np.where(step > 0, step, 1), 1.0)
                quot[b, :, :o] = q[b, :, :o] * ratio[:, None, None]
                q[b, :, :o] = np.rint(quot[b, :, :o])
            scale[b] = step
            safe = np.where(step > 0, step, 1)[:, None, None]
            quot[b, :, o:o + n] = np.where(step[:, None, None] > 0, new / safe, 0.0)
            q[b, :, o:o + n] = np.rint(quot[b, :, o:o + n])
        t += n
    return q, scale, quot


def attention(q, kq, ks, vq, vs, table, lens, cu, causal=True, window=0, scale=1.0):
    """q [T, H, D] -> out [T, H, D], lse [T, H] and what bounds a kernel's error:
    mass [T, H, D] = sum p |v| / sum p, size [T, H] = max_j sum_d |q_d k_jd| scale."""
    T, H, D = q.shape
    hk, bs = kq.shape[1], kq.shape[2]
    g = H // hk
    out, mass = np.zeros((T, H, D)), np.zeros((T, H, D))
    lse, size = np.full((T, H), -np.inf), np.zeros((T, H))
    for r, length in enumerate(lens):
        n = cu[r + 1] - cu[r]
        blocks = table[r, : -(-length // bs)]
        for h in range(hk):
            k = (kq[blocks, h].astype(np.float64) * ks[blocks, h].astype(np.float64)[:, None, None])
            v = (vq[blocks, h].astype(np.float64) * vs[blocks, h].astype(np.float64)[:, None, None])
            k, v = k.reshape(-1, D)[:length], v.reshape(-1, D)[:length]
            for i in range(n):
                pos = length - n + i
                lo, hi = 0, length
                if causal:
                    hi = min(length, pos + 1)
                    if window:
                        lo = max(0, pos - window + 1)
                if hi <= lo:
                    continue
                x = q[cu[r] + i, h * g:(h + 1) * g].astype(np.float64)  # [g, D]
                s = x @ k[lo:hi].T * scale
                m = s.max(-1, keepdims=True)
                p = np.exp(s - m)
                l = p.sum(-1, keepdims=True)
                at = (cu[r] + i, slice(h * g, (h + 1) * g))
                out[at] = p @ v[lo:hi] / l
                mass[at] = p @ np.abs(v[lo:hi]) / l
                lse[at] = (m + np.log(l))[:, 0]
                size[at] = (np.abs(x) @ np.abs(k[lo:hi]).T).max(-1) * scale
    return out, lse, mass, size
