"""Attention over the 4-bit cache where scores are large, far past what softmax needs
(MI355X only): what a row gives has to follow from its scores as fp32 numbers, whatever
their size.

u is the output type's unit roundoff (fp16 2^-11, bf16 2^-8), d the head size, scores
are off by ds = (d + 8) 2^-24 size, size = max_j sum_i |q_i| (|n_i - 8| + |z - 8|) s scale.
  * A row that sees one token gives its value: the weight, rounded to fp16, over the
    sum, not rounded: u |v| + (2^-11 + 2^-18) |v|.
  * A row whose best score is more than 2 ds + 40 above the others gives that token's
    value, to the same bound and n e^-40 of the largest one (below the bound's 2^-25).
  * Tokens of the same key have the same score in any arithmetic that treats them
    alike: the mean of their values, (u + 2^-11 + 2^-18) of the mean magnitude, and
    n 2^-32 of the largest value.
lse: ds + 2^-18 + 2^-22 |lse|.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import rhinoforge_amd as rf
from oracle import kv4 as o
from test_gpu_kv4 import DEV, UNIT, _cache, _filled, _np, _rng, _say, _table

pytestmark = pytest.mark.gpu

# queries, heads, kv_heads, head_dim, cached tokens.  Few rows: tiles of 4, 8, 16 and 32.
FEW = [(1, 4, 1, 128, 300), (1, 8, 2, 64, 300), (1, 8, 1, 256, 300), (2, 8, 2, 128, 300), (4, 4, 1, 64, 300),
       (2, 14, 2, 128, 300), (3, 8, 1, 256, 300), (5, 4, 1, 128, 300), (7, 8, 2, 64, 300), (1, 8, 2, 128, 4000)]
# Prompts: one gang and two, and their splits.
MANY = [(500, 64, 4, 64, 300), (600, 64, 8, 64, 300), (500, 64, 4, 128, 300), (900, 64, 8, 128, 300),
        (300, 64, 4, 256, 300), (300, 16, 2, 128, 6000), (300, 32, 2, 256, 6000)]
BS = 32


def _ways(shape):  # (offsets given, the launch's hints)
    n, cached = shape[0], shape[4]
    return (True, dict(max_q_len=n, max_kv_len=cached + n)), (False, {})


def _some(hq):
    """Query heads that are looked at."""
    return sorted({0, 1 % hq, hq // 3, hq // 2, hq - 1})


def _made(shape, dt, seed, reach, how):
    """(q, k, v, table, scale): scores of about 2^reach, by the scale or by the queries."""
    n, hq, hk, d, cached = shape
    nb = -(-(cached + n) // BS) + 2
    g = _rng(seed)
    k, v = _filled(nb, hk, BS, d, seed + 1), _filled(nb, hk, BS, d, seed + 2)
    q = torch.randn(n, hq, d, generator=g)
    table = _table([cached + n], BS, nb, g)
    scale = d ** -0.5
    if how == "scale":
        scale *= 2.0 ** reach
    elif how == "queries":
        q = q * 2.0 ** reach
    else:                       # what fp16 and an ordinary scale reach
        q = torch.where(q < 0, -1.0, 1.0) * (3e4 + 1e3 * torch.rand(q.shape, generator=g))
        k[1][:] = (1 + torch.rand(k[1].shape, generator=g)).half().view(torch.int16).bitwise_and(-16).view(torch.float16) * 1024
    return q.to(dt), k, v, table, scale


def _scores(q, k, table, scale, cached):
    """Exact scores [heads, n, tokens], those not seen -inf, and their error's bound."""
    n, hq, d = q.shape
    hk = k[0].shape[1]
    kn = [_np(t) for t in k]
    kv, mag = o.values(*kn), (np.abs(kn[0] - 8) + np.abs(kn[2] - 8)[..., None]) * kn[1][..., None]
    ids, total = table[0].numpy(), cached + n
    at = lambda x, h: x[ids, h].reshape(-1, x.shape[-1])[:total]  # noqa: E731
    qn, g = _np(q), hq // hk
    s = np.stack([qn[:, h] @ at(kv, h // g).T for h in _some(hq)]) * scale
    size = np.stack([np.abs(qn[:, h]) @ at(mag, h // g).T for h in _some(hq)]) * scale
    hidden = np.arange(total) > np.arange(n)[:, None] + cached
    return np.where(hidden, -np.inf, s), (d + 8) * 2.0 ** -24 * np.where(hidden, 0, size)


def _values(v, table, total, hq):
    """[heads, tokens, d]"""
    x = o.values(*(_np(t) for t in v))[table[0].numpy()]
    x = np.moveaxis(x, 1, 0).reshape(x.shape[1], -1, x.shape[-1])[:, :total]
    return np.repeat(x, hq // len(x), 0)[_some(hq)]


def _call(q, k, v, table, scale, cached, way, **kw):
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    n, hq, _ = q.shape
    cu, hints = way
    out, lse = rf.kv4_attention(q.to(DEV), _cache(k, v), table.to(DEV), i32(cached + n), i32(0, n) if cu else None,
                                scale=scale, return_lse=True, **hints, **kw)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    return np.moveaxis(_np(out), 1, 0)[_some(hq)], _np(lse).T[_some(hq)]   # heads first


def _near(out, ref, mass, dt, extra=0.0):
    tol = UNIT[dt] * np.abs(ref) + (2.0 ** -11 + 2.0 ** -18) * mass + extra + 2.0 ** -25
    bad = ~(np.abs(out - ref) <= tol)
    assert not bad.any(), f"{bad.any(-1).mean():.0%} of the rows, e.g. {out[bad][:3]} for {ref[bad][:3]}"


CASES = ([(s, dt, ("scale", r)) for r in (0, 24, 29, 45, 110) for s in FEW for dt in UNIT] +
         [(s, torch.bfloat16, ("queries", r)) for r in (29, 100) for s in FEW] +
         [(s, dt, ("fp16", 0)) for s in FEW + MANY for dt in UNIT] +
         [(s, dt, ("scale", r)) for r in (0, 24, 29, 45, 110) for s in MANY for dt in UNIT] +
         [(s, torch.bfloat16, ("queries", 60)) for s in MANY])


@pytest.mark.parametrize("shape,dt,how", CASES, ids=str)
def test_rows_that_see_one_token(shape, dt, how):
    _say("one token", shape, dt, how)
    n, hq, hk, d, cached = shape
    q, k, v, table, scale = _made(shape, dt, 70, how[1], how[0])
    s, ds = _scores(q, k, table, scale, cached)
    i = np.arange(n)
    want = _values(v, table, cached + n, hq)[:, cached + i]
    x, ds = s[:, i, cached + i], ds[:, i, cached + i]
    for way in _ways(shape):
        out, lse = _call(q, k, v, table, scale, cached, way, window=1)
        _near(out, want, np.abs(want), dt)
        assert (np.abs(lse - x) <= ds + 2.0 ** -18 + 2.0 ** -22 * np.abs(x)).all()


@pytest.mark.parametrize("shape,dt,how", CASES, ids=str)
def test_the_best_token_takes_all(shape, dt, how):
    _say("best", shape, dt, how)
    n, hq, hk, d, cached = shape
    q, k, v, table, scale = _made(shape, dt, 71, how[1], how[0])
    s, ds = _scores(q, k, table, scale, cached)
    ds = ds.max(-1)
    two = np.partition(s, -2, axis=-1)[..., -2:]
    clear = two[..., 1] - two[..., 0] > 2 * ds + 40
    assert how[0] == "scale" and how[1] < 24 or clear.mean() > 0.9
    values = _values(v, table, cached + n, hq)
    want = np.take_along_axis(values, s.argmax(-1)[..., None], 1)
    for way in _ways(shape):
        out, lse = _call(q, k, v, table, scale, cached, way)
        assert (np.abs(out) <= np.abs(values).max(1, keepdims=True) * 1.01).all()
        _near(out[clear], want[clear], np.abs(want[clear]), dt)
        x = two[..., 1][clear]
        assert (np.abs(lse[clear] - x) <= ds[clear] + 2.0 ** -18 + 2.0 ** -22 * np.abs(x)).all()


KEYS = ([(s, dt, r, a) for s in FEW for dt in UNIT for r in (0, 26, 30, 90) for a in ("alike", "apart")] +
        [(s, torch.bfloat16, r, "apart") for s in MANY for r in (0, 30, 90)])


@pytest.mark.parametrize("shape,dt,reach,steps", KEYS, ids=str)
def test_tokens_of_one_key_count_alike(shape, dt, reach, steps):
    """Values of all sizes between them; those of the largest steps are of the first tokens or the last."""
    _say("one key", shape, dt, reach, steps)
    n, hq, hk, d, cached = shape
    q, k, v, table, scale = _made(shape, dt, 72, reach, "scale")
    for t in k:
        t[:] = t[:1, :, :1].clone()
    if steps == "apart":
        pick = torch.rand(v[1].shape, generator=_rng(73))
        v[1][pick < 0.6] = torch.tensor(2.0 ** -20).half()
        v[1][pick < 0.3] = torch.tensor(2.0 ** -6).half()
        v[1][pick < 0.02] = 512.0
    total = cached + n
    values = _values(v, table, total, hq)
    count = np.arange(cached + 1, total + 1)[:, None]
    want, mass = (np.cumsum(x, 1)[:, cached:] / count for x in (values, np.abs(values)))
    most = np.abs(values).max(1, keepdims=True)
    for way in _ways(shape):
        out, _ = _call(q, k, v, table, scale, cached, way)
        _near(out, want, mass, dt, total * 2.0 ** -32 * most)


@pytest.mark.parametrize("heads", [(4, 1, 128), (8, 1, 128), (16, 1, 64), (20, 1, 128), (8, 1, 256)])
@pytest.mark.parametrize("reach", [0, 30, 60])
@pytest.mark.parametrize("n", [1, 3])
def test_tokens_of_one_key_over_many_workgroups(heads, reach, n):
    """Splits whose values differ by 2^30."""
    _say("one key, splits", heads, reach, n)
    hq, hk, d = heads
    total, bs = 20000 + n, 64
    nb = -(-total // bs)
    k, v = _filled(nb, hk, bs, d, 74), _filled(nb, hk, bs, d, 75)
    for t in k:
        t[:] = t[:1, :, :1].clone()
    v[1][: nb // 3] = torch.tensor(2.0 ** -20).half()
    v[1][nb // 3: nb // 2] = 512.0
    q = torch.randn(n, hq, d, generator=_rng(76)).half()
    table = torch.arange(nb, dtype=torch.int32)[None]
    values = _values(v, table, total, hq)
    out, _ = _call(q, k, v, table, 2.0 ** reach * d ** -0.5, 20000, (False, {}))
    count = np.arange(20001, total + 1)[:, None]
    want, mass = (np.cumsum(x, 1)[:, 20000:] / count for x in (values, np.abs(values)))
    _near(out, want, mass, torch.float16, total * 2.0 ** -32 * np.abs(values).max())


@pytest.mark.parametrize("shape", FEW + MANY, ids=str)
@pytest.mark.parametrize("reach", [0, 32, 100])
def test_scores_far_below_zero(shape, reach):
    """Every score of a row is about -2^reach; a row that sees tokens is not empty."""
    _say("low", shape, reach)
    n, hq, hk, d, cached = shape
    q, k, v, table, scale = _made(shape, torch.bfloat16, 77, reach, "scale")
    q = -q.abs()
    k[2][:] = 0
    k[0][:] = k[0] | 8
    s, ds = _scores(q, k, table, scale, cached)
    m, ds = s.max(-1), ds.max(-1)
    x = m + np.log(np.exp(s - m[..., None]).sum(-1))
    for way in _ways(shape):
        out, lse = _call(q, k, v, table, scale, cached, way)
        assert (np.abs(lse - x) <= ds + 2.0 ** -18 + 2.0 ** -22 * np.abs(x)).all()
        assert (np.abs(out).max(-1) > 0).all()


@pytest.mark.parametrize("shape", FEW + MANY, ids=str)
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("form", ["no queries", "no keys"])
def test_scores_of_zero_under_the_largest_scales(shape, dt, form):
    """Queries or keys of 0 have scores of 0 whatever the scale: the mean of the values."""
    _say("zero", shape, dt, form)
    n, hq, hk, d, cached = shape
    total = cached + n
    q, k, v, table, _ = _made(shape, dt, 78, 0, "scale")
    if form == "no queries":
        q[:] = 0
    else:
        k[0][:], k[2][:] = 8, 8
        q = q * 2.0 ** (100 if dt == torch.bfloat16 else 0)
    values = _values(v, table, total, hq)
    count = np.arange(cached + 1, total + 1)[:, None]
    want, mass = (np.cumsum(x, 1)[:, cached:] / count for x in (values, np.abs(values)))
    for scale in (1e37, 3e38):
        for way in _ways(shape):
            out, lse = _call(q, k, v, table, scale, cached, way)
            _near(out, want, mass, dt, total * 2.0 ** -32 * np.abs(values).max(1, keepdims=True))
            assert (np.abs(lse - np.log(count[:, 0])) <= 2.0 ** -18).all()
