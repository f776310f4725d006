"""Attention over the int8 cache where scales, queries and weights differ by many
powers of two, against 64 bits row by row (MI355X only).

The bound counts only what a row sees.  u is the output type's unit roundoff
(fp16 2^-11, bf16 2^-8), d the head size, n the tokens that the row may see,
x_j = log2(e) s_j, and R the largest |x_j| plus the largest |log2 vs| (and the 8 by
which the kernels' references lag).
  * scores are fp32 sums of d products: |ds| <= (d + 8) 2^-24 size, with
    size = max_j sum |q k_j| scale;
  * a weight p_j vs_j is exp2 of a sum of three fp32 terms of at most R, each
    rounded (and rescaled when a reference rises): 2^-21 (1 + R) of itself, then
    rounded to fp16: 2^-11;
  * sums in fp32: (n + 16) 2^-24 of sum p |v|;
  * the weights are kept between 2^7 and 2^15 for the row's largest, so below fp16's
    normal range each loses at most 2^-25 of a unit, 2^-32 of the row's largest
    p vs: top = max_j p_j vs_j / sum p, n 2^-32 127 top together;
  * one rounding of the output, u |ref|, with the type's smallest step below its
    normal range (bf16: fp32 results below 2^-126 may be 0).
lse: ds + 2^-18 + 2^-22 |lse|.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import rhinoforge_amd as rf

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}
LOG2E = 1.4426950408889634


def _exact(q, kq, ks, vq, vs, table, lens, cu, causal, window, scale):
    """out, lse, and for the bound: sum p|v| / sum p, max p vs / sum p, size, max|x|; fp64."""
    t, hq, d = q.shape
    hk, bs = kq.shape[1:3]
    g = hq // hk
    z = lambda *s: torch.zeros(*s, dtype=torch.float64, device=DEV)  # noqa: E731
    out, mass, top, size, far = z(t, hq, d), z(t, hq, d), z(t, hq), z(t, hq), z(t, hq)
    lse = torch.full((t, hq), -math.inf, dtype=torch.float64, device=DEV)
    for r, length in enumerate(lens):
        rows = slice(cu[r], cu[r + 1])
        n = cu[r + 1] - cu[r]
        if not n or not length:
            continue
        blocks = torch.as_tensor(table[r, : -(-length // bs)], device=DEV).long()
        at = torch.arange(length, device=DEV)
        pos = torch.arange(n, device=DEV)[:, None] + (length - n)
        hidden = torch.zeros(n, length, dtype=torch.bool, device=DEV)
        if causal:
            hidden |= at > pos
            if window:
                hidden |= at <= pos - window
        for h in range(hk):
            k = (kq[blocks, h].double() * ks[blocks, h].double()[:, None, None]).flatten(0, 1)[:length]
            v = (vq[blocks, h].double() * vs[blocks, h].double()[:, None, None]).flatten(0, 1)[:length]
            step = vs[blocks, h].double().repeat_interleave(bs)[:length]
            kt, kabs = k.t().contiguous(), k.abs().t().contiguous()
            for j in range(h * g, (h + 1) * g):
                x = q[rows, j].double()
                s = x @ kt * scale
                far[rows, j] = s.abs().masked_fill(hidden, 0).amax(-1) * LOG2E
                size[rows, j] = (x.abs() @ kabs * scale).masked_fill(hidden, 0).amax(-1)
                s.masked_fill_(hidden, -math.inf)
                m = s.amax(-1, keepdim=True)
                p = torch.exp(s - m.clamp(min=-1e300))
                total = p.sum(-1, keepdim=True)
                lse[rows, j] = (m + total.log()).squeeze(-1)
                p /= total.clamp(min=1e-300)
                out[rows, j], mass[rows, j] = p @ v, p @ v.abs()
                top[rows, j] = (p * step).amax(-1)
    return out, lse, mass, top, size, far


def _check(q, cache, table, lens, news, *, causal=True, window=0, scale=None, hints=True):
    """cache: (kq, ks, vq, vs) on the device."""
    kq, ks, vq, vs = cache
    dt, d = q.dtype, q.size(2)
    scale = d ** -0.5 if scale is None else scale
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    i32 = lambda x: torch.as_tensor(np.asarray(x, np.int32), device=DEV)  # noqa: E731
    kw = dict(max_q_len=max(news), max_kv_len=max(lens)) if hints else {}
    out, lse = rf.kv8_attention(q, rf.KV8Cache.from_quantized(kq, ks, vq, vs), i32(table), i32(lens), i32(cu),
                                causal=causal, window=window, scale=scale, return_lse=True, **kw)
    ref, rlse, mass, top, size, far = _exact(q, kq, ks, vq, vs, table, lens, cu, causal, window, scale)
    some = vs[vs > 0].double().log2().abs()
    reach = far[..., None] + (some.max().item() if some.numel() else 0.0) + 8
    ds = (d + 8) * 2.0 ** -24 * size[..., None]
    n = max(lens)
    tol = (UNIT[dt] * ref.abs() + (2.0 ** -11 + 2 * ds + 2.0 ** -21 * (1 + reach) + (n + 16) * 2.0 ** -24) * mass
           + n * 2.0 ** -32 * 127 * top[..., None] + LEAST[dt])
    err = (out.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} past the bound, worst {(err / tol).max().item():.3g}"
    none = torch.isneginf(rlse)
    assert torch.equal(torch.isneginf(lse), none)
    gap = torch.where(none, 0.0, lse.double() - torch.where(none, 0.0, rlse))
    bound = ds[..., 0] + 2.0 ** -18 + 2.0 ** -22 * torch.where(none, 0.0, rlse).abs()
    assert (gap[~none].abs() <= bound[~none]).all()
    return out


# Both kernels in their forms: tokens, queries, heads, key heads, head size.
SHAPES = [
    (700, 1, 8, 2, 128),       # decode, splits joined in the launch
    (700, 5, 8, 2, 128),       # decode, 32 rows, splits added by a second kernel
    (700, 60, 8, 2, 128),      # decode, whole tiles
    (700, 9, 8, 1, 256),
    (700, 500, 64, 4, 128),    # prefill, two gangs
    (2010, 400, 64, 8, 64),
    (2000, 2000, 64, 4, 128),  # prefill, one gang
    (700, 400, 64, 4, 256),
    (1500, 200, 64, 4, 256),   # prefill, splits
]


def _made(shape, dt, seed, bs=32):
    """Queries, cache and table of one request, with soft scores and ordinary scales."""
    n, new, hq, hk, d = shape
    g = torch.Generator().manual_seed(seed)
    width = -(-n // bs)
    nb = width + 2
    table = torch.randperm(nb, generator=g)[:width].numpy().astype(np.int32)[None]
    kq, vq = (torch.randint(-127, 128, (nb, hk, bs, d), dtype=torch.int8, generator=g) for _ in range(2))
    ks, vs = (torch.rand(nb, hk, generator=g) * 0.01 + 1e-3 for _ in range(2))
    q = torch.randn(new, hq, d, generator=g).to(dt)
    return q, [kq, ks, vq, vs], table


def _on(cache):
    return [t.to(DEV) for t in cache]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("place", ["first", "fourth", "last"])
def test_a_block_of_large_values_without_weight(shape, dt, place):
    """Values 2^33 to 2^40 times the others' in a block whose scores lie 100 nats
    lower: it adds nothing, and takes nothing from the others."""
    print("no weight", shape, dt, place, flush=True)
    small, large = (1e-2, 1e8) if dt == torch.float16 else (1e-6, 1e6)
    q, (kq, ks, vq, vs), table = _made(shape, dt, 1)
    d, width = shape[4], table.shape[1]
    b = int(table[0, {"first": 0, "fourth": 3, "last": width - 1}[place]])
    vs = vs / 0.01 * small
    vs[b] = large
    q[..., 0] = 16.0
    kq[..., 0] = 0
    kq[b] = 0
    kq[b, ..., 0] = -127
    ks[b] = 100.0 / (16 * 127) * d ** 0.5
    if place == "first":   # (the first tokens see that block alone: large outputs)
        dt = torch.bfloat16
        q = q.to(dt)
    _check(q.to(DEV), _on((kq, ks, vq, vs)), table, [shape[0]], [shape[1]])


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("opt", [{}, {"window": 40}, {"causal": False}], ids=["causal", "window", "all"])
def test_blocks_of_large_values_that_other_rows_see(shape, opt):
    """Value scales 1e-6, every seventh block 1e6: rows that do not see the loud
    block of their tile, before it or with it out of their window, keep their bits."""
    print("other rows", shape, opt, flush=True)
    q, (kq, ks, vq, vs), table = _made(shape, torch.bfloat16, 2)
    vs = vs / 0.01 * 1e-6
    vs[table[0, 2::7]] = 1e6
    _check(q.to(DEV), _on((kq, ks, vq, vs)), table, [shape[0]], [shape[1]], **opt)


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("loud", [1.0, 30.0])
def test_value_scales_of_every_size(shape, loud):
    """Value scales from 2^-30 to 2^30 from block to block and head to head."""
    print("every size", shape, loud, flush=True)
    q, (kq, ks, vq, vs), table = _made(shape, torch.bfloat16, 3)
    vs = 2.0 ** (torch.rand(vs.shape, generator=torch.Generator().manual_seed(4)) * 60 - 30)
    _check((q * loud).to(DEV), _on((kq, ks, vq, vs)), table, [shape[0]], [shape[1]])


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_value_scales_of_zero(shape):
    """A scale of 0 makes its block's values 0 whatever the bytes; rows that see
    only such blocks give exact zeros, beside blocks of 1e-6."""
    print("zero", shape, flush=True)
    q, (kq, ks, vq, vs), table = _made(shape, torch.bfloat16, 5)
    vs = vs / 0.01 * 1e-6
    vs[table[0, : table.shape[1] // 2]] = 0.0
    n, new = shape[:2]
    out = _check(q.to(DEV), _on((kq, ks, vq, vs)), table, [n], [new])
    blind = max(table.shape[1] // 2 * 32 - (n - new), 0)
    assert (out[:blind] == 0).all()
    vs[:] = 0.0
    assert (_check(q.to(DEV), _on((kq, ks, vq, vs)), table, [n], [new]) == 0).all()


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("size", [2.0 ** -128, 2.0 ** -107, 2.0 ** 90])
def test_value_scales_at_the_ends_of_fp32(shape, size):
    """2^-128 has no normal fp32 form."""
    print("ends", shape, size, flush=True)
    q, (kq, ks, vq, vs), table = _made(shape, torch.bfloat16, 6)
    vs[:] = size
    vq[vq.abs() < 64] = 127
    _check(q.to(DEV), _on((kq, ks, vq, vs)), table, [shape[0]], [shape[1]])
