"""Attention over the int8 cache where scores are large, far past what softmax needs
(MI355X only): what a row gives has to follow from its scores as fp32 numbers, whatever
their size.

u is the output type's unit roundoff (fp16 2^-11, bf16 2^-8), d the head size, scores
are off by ds = (d + 8) 2^-24 size, size = max_j sum |q k_j| scale.  Weights are rounded
to fp16 (2^-11) from exponents of at most 120 (2^-16 in all).
  * A row that sees one token gives its value: (u + 2^-11 + 2^-16) |v|.
  * So does one whose best score is more than 2 ds + 40 above the others, to n e^-40 of
    the largest value (below the bound's smallest step).
  * Tokens of the same key have the same score in any arithmetic that treats them alike:
    the mean of their values, to (u + 2^-11 + 2^-16) of the mean magnitude and n 2^-32
    127 of the largest value scale.
lse: ds + 2^-18 + 2^-22 |lse|.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import rhinoforge_amd as rf

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}

# queries, heads, kv_heads, head_dim, cached tokens.  Few rows: tiles of 16 and 32.
FEW = [(1, 8, 2, 128, 300), (1, 12, 12, 64, 300), (2, 8, 1, 256, 300), (5, 8, 2, 128, 300), (7, 8, 2, 64, 300),
       (1, 32, 8, 128, 9000), (4, 64, 8, 128, 4000), (4, 8, 1, 256, 4000)]
# Prompts: one gang and two, and their splits.
MANY = [(500, 64, 4, 64, 300), (600, 64, 8, 64, 300), (500, 64, 4, 128, 300), (900, 64, 8, 128, 300),
        (300, 64, 4, 256, 300), (200, 64, 4, 256, 1300)]
BS = 32


def _some(hq):
    """Query heads that are looked at."""
    return sorted({0, 1 % hq, hq // 3, hq // 2, hq - 1})


def _np(t):
    return t.detach().cpu().double().numpy()


def _made(shape, dt, seed, reach, how):
    n, hq, hk, d, cached = shape
    nb = -(-(cached + n) // BS)
    g = torch.Generator().manual_seed(seed)
    kq, vq = (torch.randint(-127, 128, (nb, hk, BS, d), dtype=torch.int8, generator=g) for _ in range(2))
    ks, vs = (torch.rand(nb, hk, generator=g) * 0.01 + 1e-3 for _ in range(2))
    q, scale = torch.randn(n, hq, d, generator=g), d ** -0.5
    if how == "scale":
        scale *= 2.0 ** reach
    elif how == "queries":
        q = q * 2.0 ** reach
    else:                       # what fp16 and an ordinary scale reach
        q = torch.where(q < 0, -1.0, 1.0) * (3e4 + 1e3 * torch.rand(q.shape, generator=g))
        ks = ks * 2e4
    return q.to(dt), (kq, ks, vq, vs), torch.randperm(nb, generator=g).int()[None], scale


def _held(x, scale, table, total, hq):
    """[heads, tokens, d]"""
    x = (_np(x) * _np(scale)[..., None, None])[table[0].numpy()]
    x = np.moveaxis(x, 1, 0).reshape(x.shape[1], -1, x.shape[-1])[:, :total]
    return np.repeat(x, hq // len(x), 0)[_some(hq)]


def _call(q, cache, table, total, scale, cu, **kw):
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    n, hq, _ = q.shape
    hints = dict(max_q_len=n, max_kv_len=total) if cu else {}
    out, lse = rf.kv8_attention(q.to(DEV), rf.KV8Cache.from_quantized(*(t.to(DEV) for t in cache)), table.to(DEV),
                                i32(total), i32(0, n) if cu else None, scale=scale, return_lse=True, **hints, **kw)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    return np.moveaxis(_np(out), 1, 0)[_some(hq)], _np(lse).T[_some(hq)]   # heads first


def _near(out, ref, mass, dt, extra=0.0):
    tol = UNIT[dt] * np.abs(ref) + (2.0 ** -11 + 2.0 ** -16) * mass + extra + 2.0 ** -25
    bad = ~(np.abs(out - ref) <= tol)
    assert not bad.any(), f"{bad.any(-1).mean():.0%} of the rows, e.g. {out[bad][:3]} for {ref[bad][:3]}"


CASES = ([(s, dt, ("scale", r)) for r in (0, 24, 29, 45, 110) for s in FEW for dt in UNIT] +
         [(s, torch.bfloat16, ("queries", r)) for r in (29, 100) for s in FEW] +
         [(s, dt, ("fp16", 0)) for s in FEW + MANY for dt in UNIT] +
         [(s, dt, ("scale", r)) for r in (0, 24, 29, 45, 110) for s in MANY for dt in UNIT] +
         [(s, torch.bfloat16, ("queries", 60)) for s in MANY])


@pytest.mark.parametrize("shape,dt,how", CASES, ids=str)
@pytest.mark.parametrize("window", [1, 0])
def test_one_token_takes_all(shape, dt, how, window):
    """The only one that a row sees, or the one of the best score."""
    print("one token", shape, dt, how, window, flush=True)
    n, hq, hk, d, cached = shape
    q, cache, table, scale = _made(shape, dt, 80, how[1], how[0])
    total = cached + n
    k, values = _held(*cache[:2], table, total, hq), _held(*cache[2:], table, total, hq)
    qn = np.moveaxis(_np(q), 1, 0)[_some(hq)]
    s, size = (np.stack([x @ y.T for x, y in zip(*p)]) * scale for p in ((qn, k), (np.abs(qn), np.abs(k))))
    pos, at = np.arange(n)[:, None] + cached, np.arange(total)
    hidden = (at > pos) | (at <= pos - window) if window else at > pos
    s = np.where(hidden, -np.inf, s)
    ds = (d + 8) * 2.0 ** -24 * np.where(hidden, 0, size).max(-1)
    two = np.partition(s, -2, axis=-1)[..., -2:]
    clear = two[..., 1] - two[..., 0] > 2 * ds + 40
    assert how[0] == "scale" and how[1] < 24 or clear.mean() > 0.9
    want = np.take_along_axis(values, s.argmax(-1)[..., None], 1)
    for cu in (True, False):
        out, lse = _call(q, cache, table, total, scale, cu, window=window)
        assert (np.abs(out) <= np.abs(values).max(1, keepdims=True) * 1.01).all()
        _near(out[clear], want[clear], np.abs(want[clear]), dt)
        x = two[..., 1][clear]
        assert (np.abs(lse[clear] - x) <= ds[clear] + 2.0 ** -18 + 2.0 ** -22 * np.abs(x)).all()


@pytest.mark.parametrize("shape", FEW + MANY, ids=str)
@pytest.mark.parametrize("reach", [0, 20, 26, 30, 90])
@pytest.mark.parametrize("steps", ["alike", "apart"])
def test_tokens_of_one_key_count_alike(shape, reach, steps):
    """Values of all sizes between them, block by block."""
    print("one key", shape, reach, steps, flush=True)
    n, hq, hk, d, cached = shape
    total = cached + n
    nb = -(-total // BS)
    g = torch.Generator().manual_seed(81)
    kq = torch.randint(-127, 128, (1, hk, 1, d), dtype=torch.int8, generator=g).expand(nb, hk, BS, d).contiguous()
    vq = torch.randint(-127, 128, (nb, hk, BS, d), dtype=torch.int8, generator=g)
    ks, vs = torch.full((nb, hk), 0.0078125), torch.rand(nb, hk, generator=g) * 0.01 + 1e-3
    if steps == "apart":   # 2^-20 to the most that fp16 values need
        vs = torch.tensor([2.0 ** -20, 2.0 ** -12, 2.0 ** -6, 500.0])[torch.randint(0, 4, (nb, hk), generator=g)]
    q = torch.randn(n, hq, d, generator=g).bfloat16()
    table = torch.randperm(nb, generator=g).int()[None]
    values = _held(vq, vs, table, total, hq)
    count = np.arange(cached + 1, total + 1)[:, None]
    want, mass = (np.cumsum(x, 1)[:, cached:] / count for x in (values, np.abs(values)))
    for cu in (True, False):
        out, _ = _call(q, (kq, ks, vq, vs), table, total, 2.0 ** reach * d ** -0.5, cu)
        _near(out, want, mass, torch.bfloat16, total * 2.0 ** -32 * 127 * vs.max().item())


@pytest.mark.parametrize("shape", FEW + MANY, ids=str)
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("form", ["no queries", "no keys", "no key scale"])
def test_scores_of_zero_under_the_largest_scales(shape, dt, form):
    """Queries or keys of 0 have scores of 0 whatever the scale: the mean of the values."""
    print("zero", shape, dt, form, flush=True)
    n, hq, hk, d, cached = shape
    total = cached + n
    q, (kq, ks, vq, vs), table, _ = _made(shape, dt, 82, 0, "scale")
    if form == "no queries":
        q[:] = 0
    elif form == "no keys":
        kq[:] = 0
    else:
        ks[:] = 0
    if dt == torch.bfloat16 and form != "no queries":
        q = q * 2.0 ** 100
    values = _held(vq, vs, table, total, hq)
    count = np.arange(cached + 1, total + 1)[:, None]
    want, mass = (np.cumsum(x, 1)[:, cached:] / count for x in (values, np.abs(values)))
    for scale in (1e37, 3e38):
        for cu in (True, False):
            out, lse = _call(q, (kq, ks, vq, vs), table, total, scale, cu)
            _near(out, want, mass, dt, total * 2.0 ** -32 * 127 * vs.max().item())
            assert (np.abs(lse - np.log(count[:, 0])) <= 2.0 ** -18).all()
