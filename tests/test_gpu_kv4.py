"""The 4-bit paged cache's kernels against oracle/kv4.py in 64 bits (MI355X only).

Append and read-back are exact: the step is a comparison of numbers that fp32 holds,
the rounded quotient is exact where it is a tie, and the held values are fp16
numbers.  Tolerances of the attention follow from the arithmetic.  u is the output
type's unit roundoff (fp16 2^-11, bf16 2^-8), d the head size.
  * Scores are fp32 sums over d products, of the numbers less 8 and of the query's
    sum times the zero point less 8 (or of the values themselves): |ds| <= (d + 8)
    2^-24 size, size = max_j sum_d |q| (|n_j - 8| + |z_j - 8|) s_j scale, which also
    bounds |q k_j| scale.
  * p = 2^x is within 2^-22 (1 + |x|), times the step it is rounded to fp16 (2^-11);
    weights below the fp16 range lose at most n 2^-32 max|v - z| s:
    |o - ref| <= u |ref| + (2^-11 + 2 ds + 2^-18) sum p|v| / sum p + n 2^-32 max|v|.
    lse: ds + 2^-18 + 2^-22 |lse|.
  * norm and rotation: as tests/test_gpu_kv8.py, u |y| + (d / 8 + 16) 2^-23 max|y|.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import rhinoforge_amd as rf
from oracle import kv4 as o
from oracle import kv8 as o8

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _say(*a):
    print(*a, flush=True)


def _rng(seed):
    return torch.Generator().manual_seed(seed)


def _np(t):
    return t.detach().cpu().double().numpy()


# ---- norms and rotation by several axes -----------------------------------------------

MROPE = [
    # tokens, heads, kv_heads, head_dim, sections, mixed, dtype, interleaved, norms, positions
    (1, 32, 8, 128, [24, 20, 20], True, torch.float16, False, "both", torch.int64),
    (17, 28, 4, 128, [16, 24, 24], False, torch.bfloat16, False, "none", torch.int64),
    (3, 8, 1, 256, [48, 40, 40], True, torch.bfloat16, False, "both", torch.int32),
    (5, 12, 12, 64, [16, 16], False, torch.float16, False, "q", torch.int32),
    (6, 12, 12, 64, [16, 16], True, torch.float16, True, "k", torch.int64),
    (9, 3, 2, 40, [4, 2, 2], True, torch.bfloat16, True, "none", torch.int32),
    (4, 3, 1, 80, [10, 10, 10, 10], True, torch.float16, False, "both", torch.int64),
    (4, 3, 1, 80, [0, 40, 0], False, torch.float16, False, "both", torch.int64),
    (2, 5, 2, 512, [86, 85, 85], True, torch.float16, False, "both", torch.int64),
    (2, 5, 2, 512, [1, 2, 3, 250], False, torch.float16, True, "both", torch.int32),
    (7, 2, 1, 96, [24], False, torch.bfloat16, False, "both", torch.int64),
    (1030, 2, 1, 64, [12, 10, 10], True, torch.float16, False, "both", torch.int64),
]


@pytest.mark.parametrize("case", MROPE, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("strided", [False, True])
def test_norm_mrope(case, strided):
    t, hq, hk, d, sections, mixed, dt, inter, norms, post = case
    _say("mrope", case, strided)
    g = _rng(t * 31 + d)
    rows, pairs, axes = 50, sum(sections), len(sections)
    width = (hq + 2 * hk) * d
    f = (torch.randn(t, width, generator=g) * torch.where(torch.rand(t, 1, generator=g) < 0.2, 1e-3, 3.0)).to(dt).to(DEV)
    q = f[:, : hq * d].unflatten(1, (hq, d))
    k = f[:, hq * d: (hq + hk) * d].unflatten(1, (hk, d))
    pos = torch.randint(0, rows, (axes, t), generator=g).to(post)
    p = pos.to(DEV)
    if strided:
        p = torch.stack((p, p), 1)[:, 0] if t % 2 else torch.stack((p, p), -1)[..., 0]
    else:
        q, k = q.contiguous(), k.contiguous()
    qw = torch.randn(d, generator=g).to(dt) if norms in ("both", "q") else None
    kw = torch.randn(d, generator=g).to(dt) if norms in ("both", "k") else None
    ang = torch.rand(rows, pairs, generator=g) * 6.3
    cos, sin = ang.cos(), ang.sin()
    dev = lambda x: None if x is None else x.to(DEV)  # noqa: E731
    got = rf.qk_norm_mrope(q, k, dev(qw), dev(kw), dev(cos), dev(sin), p, sections, mixed=mixed, eps=1e-6,
                           interleaved=inter)
    row = pos.numpy()[o.axis_of_pairs(sections, mixed)].T       # [t, pairs]
    cos, sin = (_np(x)[row, np.arange(pairs)] for x in (cos, sin))
    for x, w, y in ((q, qw, got[0]), (k, kw, got[1])):
        assert y.dtype == dt and y.is_contiguous() and y.shape == x.shape
        ref = o8.norm_rope(_np(x), None if w is None else _np(w), cos, sin, None, 1e-6, inter)
        tol = UNIT[dt] * np.abs(ref) + (d / 8 + 16) * 2.0 ** -23 * np.abs(ref).max(-1, keepdims=True) + 2.0 ** -25
        err = np.abs(_np(y) - ref)
        assert (err <= tol).all(), (err / tol).max()


def test_one_axis_is_the_rotation_by_positions():
    g = _rng(3)
    q, k = (torch.randn(33, n, 128, generator=g).half().to(DEV) for n in (8, 2))
    w = torch.randn(128, generator=g).half().to(DEV)
    cos, sin = rf.rope_table(1e6 ** (-torch.arange(64, device=DEV) / 64), 500)
    pos = torch.randint(0, 500, (33,), generator=g).to(DEV)
    want = rf.qk_norm_rope(q, k, w, w, cos, sin, pos)
    for p, sections, mixed in ((pos[None], [64], False), (pos.expand(3, -1), [24, 20, 20], True),
                               (pos.expand(2, -1), [40, 24], False)):
        got = rf.qk_norm_mrope(q, k, w, w, cos, sin, p, sections, mixed=mixed)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_a_position_of_any_axis_outside_the_table_gives_nan():
    q, k = (torch.ones(5, n, 64, dtype=torch.float16, device=DEV) for n in (2, 1))
    cos = torch.ones(10, 16, device=DEV)  # 32 of 64 dimensions are rotated
    pos = torch.tensor([[0, 1, 2, 3, 9], [0, -1, 2, 3, 9], [0, 1, 2, 10, 9]], device=DEV)
    for y in rf.qk_norm_mrope(q, k, None, None, cos, cos, pos, [6, 5, 5], mixed=True):
        assert torch.isfinite(y[[0, 2, 4]]).all() and torch.isnan(y[[1, 3]]).all()


# ---- append and read ---------------------------------------------------------------------

def _filled(nb, hk, bs, d, seed):
    g = _rng(seed)
    n = torch.randint(0, 16, (nb, hk, bs, d), generator=g).to(torch.uint8)
    s = (torch.randint(0x2000, 0x3c00, (nb, hk, bs), generator=g) & ~15).to(torch.int16).view(torch.float16)
    return n, s, torch.randint(4, 12, (nb, hk, bs), generator=g).to(torch.uint8)


def _cache(k, v):
    return rf.KV4Cache.from_quantized(*(t.to(DEV) for t in (*k, *v)))


APPEND = [
    # kv_heads, head_dim, block_size, dtype, runs of (block, offset, tokens)
    (2, 128, 64, torch.float16, [(3, 5, 1)]),
    (1, 64, 32, torch.bfloat16, [(0, 0, 1), (2, 31, 1), (1, 7, 25)]),
    (8, 128, 64, torch.float16, [(1, 0, 64), (4, 0, 64), (0, 0, 13)]),
    (4, 128, 32, torch.bfloat16, [(5, 30, 2), (6, 0, 32), (7, 0, 9), (2, 15, 3)]),
    (1, 256, 128, torch.float16, [(2, 100, 28), (0, 0, 128), (1, 0, 70)]),
    (3, 256, 32, torch.bfloat16, [(4, 16, 5)]),
    (12, 64, 128, torch.float16, [(4, 33, 60), (5, 1, 127), (0, 127, 1)]),
]


@pytest.mark.parametrize("case", APPEND, ids=lambda c: "-".join(map(str, c[:4])) + "-" + str(len(c[4])))
@pytest.mark.parametrize("form", ["plain", "strided", "scattered"])
def test_append(case, form):
    hk, d, bs, dt, runs = case
    _say("append", case, form)
    g = _rng(d + bs)
    nb = 9
    held_k, held_v = _filled(nb, hk, bs, d, 1), _filled(nb, hk, bs, d, 2)
    slots = np.concatenate([np.arange(b * bs + at, b * bs + at + n) for b, at, n in runs]).astype(np.int32)
    if form == "scattered":
        slots = slots[torch.randperm(len(slots), generator=g).numpy()]
        slots[::5] = -1 - slots[::5] if len(slots) > 1 else slots[::5]
        slots[3:4] = nb * bs
    t = len(slots)
    x = torch.randn(t, 3, hk, d, generator=g) * torch.exp(torch.randn(t, 3, hk, 1, generator=g) * 2)
    x[:, :, 0, : d // 2] = torch.randint(-9, 10, (t, 3, d // 2), generator=g) * 0.5   # ties
    x = x.to(dt)
    k, v = (x[:, 1], x[:, 2]) if form == "strided" else (x[:, 1].contiguous(), x[:, 2].contiguous())
    cache = _cache(held_k, held_v)
    xd = x.to(DEV)
    kd, vd = (xd[:, 1], xd[:, 2]) if form == "strided" else (k.to(DEV), v.to(DEV))
    rf.kv4_append(cache, kd, vd, torch.from_numpy(slots).to(DEV))
    got = cache.to_quantized()
    for side, (held, new) in enumerate(((held_k, k), (held_v, v))):
        want = o.append([_np(h) for h in held], _np(new), slots)
        for a, b, what in zip(got[3 * side: 3 * side + 3], want, ("numbers", "steps", "zero points")):
            assert np.array_equal(_np(a), b), (what, side)


def test_append_of_extreme_rows():
    """Zeros, one value, spans at the ends of what steps reach, denormals, ties, in both types."""
    d, bs = 64, 32
    for dt in (torch.float16, torch.bfloat16):
        big = 65504.0 if dt == torch.float16 else 3e38
        rows = [torch.zeros(d), torch.full((d,), 3.5), torch.full((d,), -1e-4), torch.full((d,), 2.0 ** -24),
                torch.linspace(-big, big, d), torch.linspace(0, 65280, d), torch.linspace(-32768, 32000, d),
                torch.linspace(-2.0 ** -20, 2.0 ** -20, d), torch.linspace(-15 * 2.0 ** -15, 0, d),
                torch.arange(d) * 0.25 - 4, torch.arange(d).float(), -torch.arange(d).float() / 2,
                torch.cat((torch.full((1,), 15.0), torch.full((1,), -2.0 ** -20), torch.zeros(d - 2))),
                torch.cat((torch.full((1,), 7.5), torch.full((1,), -7.5), torch.linspace(-7.5, 7.5, d - 2)))]
        x = torch.stack(rows).to(dt)[:, None]
        cache = rf.KV4Cache(1, 1, d, bs, device=DEV)
        slots = torch.arange(len(rows), dtype=torch.int32, device=DEV)
        cache.append(x.to(DEV), x.flip(0).to(DEV), slots)
        got = [_np(t)[0, 0, : len(rows)] for t in cache.to_quantized()]
        for side, y in ((0, x), (3, x.flip(0))):
            for i, row in enumerate(_np(y)[:, 0]):
                if not (np.isfinite(_np(x)[i, 0]).all() and np.isfinite(_np(x.flip(0))[i, 0]).all()):
                    assert np.isnan(got[1][i])   # (linspace's own overflow, at the end of bf16)
                    continue
                n, s, z = o.quantize(row)
                assert s == got[side + 1][i] and z == got[side + 2][i], (dt, side, i, s, got[side + 1][i])
                assert np.array_equal(n, got[side][i]), (dt, side, i)


def test_append_of_infinities_and_nan():
    d, bs, hk = 128, 32, 2
    for dt in (torch.float16, torch.bfloat16):
        x = torch.randn(2, 9, hk, d, generator=_rng(4)).to(dt)
        x[0, 1, 0, 5], x[1, 3, 1, 127], x[0, 5, 1, 0], x[1, 5, 1, 1] = (float(s) for s in ("inf", "nan", "-inf", "nan"))
        cache = rf.KV4Cache(2, hk, d, bs, device=DEV)
        slots = torch.arange(20, 29, dtype=torch.int32, device=DEV)
        cache.append(x[0].to(DEV), x[1].to(DEV), slots)
        bad = torch.zeros(9, hk, dtype=torch.bool)
        bad[1, 0] = bad[3, 1] = bad[5, 1] = True
        for side, y in enumerate(cache.read(slots, torch.float32)):
            assert torch.equal(torch.isnan(y).all(-1).cpu(), bad) and torch.equal(torch.isnan(y).any(-1).cpu(), bad)
            ref = o.values(*o.quantize(_np(torch.where(bad[..., None], 0, x[side]))))
            assert np.array_equal(_np(y)[~bad.numpy()], ref[~bad.numpy()])
        q = cache.to_quantized()
        assert torch.isfinite(q[4]).all() and torch.isnan(q[1]).sum() == 3


@pytest.mark.parametrize("hk,d,bs", [(2, 64, 32), (8, 128, 64), (1, 256, 128), (3, 128, 128)])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
def test_read(hk, d, bs, dt):
    _say("read", hk, d, bs, dt)
    k, v = _filled(6, hk, bs, d, 5), _filled(6, hk, bs, d, 6)
    cache = _cache(k, v)
    for n in (1, 31, 700, 5000):
        slots = torch.randint(-3, 6 * bs + 3, (n,), generator=_rng(n), dtype=torch.int32)
        got = cache.read(slots.to(DEV), dt)
        inside = ((slots >= 0) & (slots < 6 * bs)).numpy()
        at = slots.clamp(0, 6 * bs - 1).numpy()
        for side, y in ((k, got[0]), (v, got[1])):
            ref = o.values(*(_np(t) for t in side))[at // bs, :, at % bs] * inside[:, None, None]
            assert y.dtype == dt and y.shape == (n, hk, d)
            assert torch.equal(y.cpu(), torch.from_numpy(ref).to(dt))
    assert cache.read(slots[:0].to(DEV), dt)[0].shape == (0, hk, d)


# ---- attention ---------------------------------------------------------------------------

def _table(lens, bs, nb, g, width=None):
    counts = [-(-n // bs) for n in lens]
    w = width or max(1, max(counts))
    ids = torch.randperm(nb, generator=g).to(torch.int32)
    table, at = torch.full((len(lens), w), -1, dtype=torch.int32), 0
    for r, c in enumerate(counts):
        table[r, :c] = ids[at:at + c]
        at += c
    return table


def _check(q, k, v, table, lens, news, *, cu=True, scale=None, lse=True, uniform=False, **kw):
    """The kernel's output and lse against the oracle; returns them."""
    cache = _cache(k, v)
    kn, vn = [_np(t) for t in k], [_np(t) for t in v]
    kv, vv = o.values(*kn), o.values(*vn)
    mag = (np.abs(kn[0] - 8) + np.abs(kn[2] - 8)[..., None]) * kn[1][..., None]
    d = q.size(-1)
    offsets = np.concatenate(([0], np.cumsum(news)))
    scale = d ** -0.5 if scale is None else scale
    ref, rlse, mass, size = o.attention(_np(q), kv, vv, table.numpy(), lens, offsets, scale=scale, kmag=mag,
                                        causal=kw.get("causal", True), window=kw.get("window", 0))
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)  # noqa: E731
    got, glse = rf.kv4_attention(q.to(DEV), cache, table.to(DEV), i32(lens), i32(offsets) if cu else None,
                                 scale=scale, return_lse=True, **kw)
    ds = (d + 8) * 2.0 ** -24 * size
    most = np.nanmax(np.abs(vv)) + 15 * np.nanmax(vn[1])
    tol = (UNIT[q.dtype] * np.abs(ref) + (2.0 ** -11 + 2 * ds[..., None] + 2.0 ** -18) * mass
           + max(lens) * 2.0 ** -32 * most + 2.0 ** -25)
    out = _np(got)
    nan = np.isnan(ref)
    assert np.array_equal(np.isnan(out), nan), "NaN where it should not be, or the other way round"
    err = np.where(nan, 0, np.abs(out - np.where(nan, 0, ref)))
    assert (err <= np.where(nan, 1, tol)).all(), (err / tol)[~nan].max()
    l = _np(glse)
    seen = np.isfinite(rlse)
    assert np.array_equal(np.isneginf(l), np.isneginf(rlse))
    off = np.abs(l[seen] - rlse[seen])
    assert (off <= ds[seen] + 2.0 ** -18 + 2.0 ** -22 * np.abs(rlse[seen])).all(), off.max()
    return got, glse


ATTEND = [
    # heads, kv_heads, head_dim, block_size, dtype, [(cached, new)], options
    (8, 2, 128, 64, torch.float16, [(0, 1)], {}),
    (32, 8, 128, 64, torch.float16, [(776, 1)], {}),
    (4, 4, 64, 32, torch.bfloat16, [(31, 1), (32, 1), (33, 1), (0, 1), (500, 1)], {}),
    (8, 1, 256, 128, torch.bfloat16, [(300, 1), (127, 1)], {}),
    (28, 4, 128, 64, torch.float16, [(100, 5), (0, 3), (63, 1), (64, 2)], {}),
    (16, 2, 64, 64, torch.float16, [(1000, 4)], dict(window=100)),
    (8, 1, 256, 32, torch.bfloat16, [(90, 50), (0, 50)], dict(causal=False)),
    (8, 2, 128, 32, torch.bfloat16, [(0, 200)], {}),
    (4, 1, 128, 64, torch.float16, [(70, 333), (0, 1), (5, 150)], dict(window=64)),
    (12, 12, 64, 128, torch.float16, [(0, 300)], {}),
    (8, 1, 256, 64, torch.float16, [(3, 260)], {}),
    (2, 1, 256, 64, torch.bfloat16, [(200, 130)], dict(window=33)),
    (4, 2, 64, 32, torch.bfloat16, [(10, 140), (0, 129)], dict(causal=False)),
    (1, 1, 128, 64, torch.float16, [(2000, 9)], {}),
    (40, 2, 128, 32, torch.float16, [(64, 1), (1, 1)], {}),
    (20, 1, 64, 32, torch.bfloat16, [(40, 2), (0, 0), (7, 1)], {}),
]


@pytest.mark.parametrize("case", ATTEND, ids=lambda c: "-".join(map(str, c[:5])) + "-" + str(c[5])[:40])
@pytest.mark.parametrize("known", [False, True])
def test_attention(case, known):
    hq, hk, d, bs, dt, batch, kw = case
    _say("attention", case, known)
    g = _rng(hq * d + len(batch))
    lens, news = [a + n for a, n in batch], [n for _, n in batch]
    nb = sum(-(-n // bs) for n in lens) + 3
    k, v = _filled(nb, hk, bs, d, 7), _filled(nb, hk, bs, d, 8)
    q = torch.randn(sum(news), hq, d, generator=g).to(dt)
    hints = dict(max_q_len=max(news), max_kv_len=max(lens)) if known else {}
    _check(q, k, v, _table(lens, bs, nb, g), lens, news, **hints, **kw)


def test_attention_of_equal_queries_without_offsets():
    g = _rng(20)
    k, v = _filled(12, 2, 32, 64, 9), _filled(12, 2, 32, 64, 10)
    q = torch.randn(9, 6, 64, generator=g).half()
    _check(q, k, v, _table([100, 3, 64], 32, 12, g), [100, 3, 64], [3, 3, 3], cu=False)


@pytest.mark.parametrize("n,hq", [(1, 8), (40, 8), (200, 4)])
def test_queries_that_see_nothing_give_zeros(n, hq):
    """More queries than cached tokens: the first ones are before the sequence."""
    _say("nothing seen", n, hq)
    g = _rng(21)
    k, v = _filled(6, 2, 32, 128, 11), _filled(6, 2, 32, 128, 12)
    q = torch.randn(2 * n, hq, 128, generator=g).half()
    lens = [max(n // 2, 0), 0]
    got, lse = _check(q, k, v, _table([max(x, 1) for x in lens], 32, 6, g, 4), lens, [n, n])
    assert (got[n:] == 0).all() and torch.isneginf(lse[n:]).all()


@pytest.mark.parametrize("n", [1, 6, 150])
def test_tokens_behind_the_batch_give_zeros(n):
    g = _rng(22)
    k, v = _filled(9, 1, 32, 64, 13), _filled(9, 1, 32, 64, 14)
    q = torch.randn(n + 7, 4, 64, generator=g).half().to(DEV)
    table = _table([n + 50], 32, 9, g).to(DEV)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    cache = _cache(k, v)
    out, lse = rf.kv4_attention(q, cache, table, i32(n + 50), i32(0, n), return_lse=True)
    assert (out[n:] == 0).all() and torch.isneginf(lse[n:]).all()
    want = rf.kv4_attention(q[:n], cache, table, i32(n + 50), i32(0, n))
    assert torch.equal(out[:n], want) or (out[:n].float() - want.float()).abs().max() < 1e-2


@pytest.mark.parametrize("n", [1, 4, 160])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_tokens_that_stand_for_nan(n, d):
    """NaN to the queries that see them, no difference to the others."""
    _say("nan", n, d)
    g = _rng(23)
    k, v = _filled(20, 2, 32, d, 15), _filled(20, 2, 32, d, 16)
    cached = 300
    table = _table([cached + n], 32, 20, g)
    for at, head in ((cached + n - 1, 0), (10, 1)):
        k[1][table[0, at // 32].long(), head, at % 32] = float("nan")
    q = torch.randn(n, 4, d, generator=g).half()
    # a window that does not reach token 10, and the last query alone sees the last token
    _check(q, k, v, table, [cached + n], [n], window=100)
    _check(q, k, v, table, [cached + n], [n])


@pytest.mark.parametrize("n", [1, 4, 160])
def test_block_ids_outside_the_cache_give_nan(n):
    g = _rng(24)
    k, v = _filled(12, 2, 32, 128, 17), _filled(12, 2, 32, 128, 18)
    table = _table([200 + n] if n < 100 else [n + 60], 32, 12, g)
    for bad in (-1, 12, 2 ** 31 - 1):
        table[0, 1] = bad
        q = torch.randn(n, 4, 128, generator=g).half()
        lens = [200 + n] if n < 100 else [n + 60]
        _check(q, k, v, table, lens, [n])
        _check(q, k, v, table, lens, [n], window=40)


@pytest.mark.parametrize("n", [1, 7, 140])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("form", ["values", "keys", "both"])
def test_steps_far_apart(n, dt, form):
    """Tokens whose steps differ by 2^30, loud ones seen and unseen, with and without weight."""
    _say("steps", n, dt, form)
    g = _rng(25)
    k, v = _filled(16, 2, 32, 128, 19), _filled(16, 2, 32, 128, 20)
    lens = [300 + n]
    table = _table(lens, 32, 16, g)
    pick = torch.rand(16, 2, 32, generator=g)
    small, large = torch.tensor(2.0 ** -20).half(), torch.tensor(1024.0).half()
    if form in ("values", "both"):
        v[1][pick < 0.5] = small
        v[1][pick < 0.02] = large
    if form in ("keys", "both"):
        k[1][pick > 0.6] = small
        k[1][pick > 0.99] = torch.tensor(8.0).half()
    q = torch.randn(n, 4, 128, generator=g).to(dt)
    _check(q, k, v, table, lens, [n])
    _check(q, k, v, table, lens, [n], window=50)


@pytest.mark.parametrize("n", [1, 140])
@pytest.mark.parametrize("scale", [1e-44, 1e-38, 1e-20, 30.0])
def test_scales_at_the_ends(n, scale):
    g = _rng(26)
    k, v = _filled(10, 1, 32, 128, 21), _filled(10, 1, 32, 128, 22)
    q = torch.randn(n, 4, 128, generator=g).half()
    _check(q, k, v, _table([150 + n], 32, 10, g), [150 + n], [n], scale=scale)


@pytest.mark.parametrize("n", [1, 140])
@pytest.mark.parametrize("size", [1e-37, 1e-20, 1e20, 1e30])
def test_bf16_queries_past_the_range_of_fp16(n, size):
    g = _rng(27)
    k, v = _filled(10, 1, 32, 128, 23), _filled(10, 1, 32, 128, 24)
    q = (torch.randn(n, 4, 128, generator=g).bfloat16().double() * size).bfloat16()
    _check(q, k, v, _table([150 + n], 32, 10, g), [150 + n], [n], scale=1.0 / size)


@pytest.mark.parametrize("lens", [[20000], [9000, 1, 4000, 700], [130] * 40])
@pytest.mark.parametrize("n", [1, 3])
def test_long_and_ragged_batches(lens, n):
    """Tokens split over workgroups; the order of arrival does not show."""
    _say("long", lens[:4], n)
    g = _rng(28)
    bs, hk, d = 64, 1, 64
    nb = sum(-(-x // bs) for x in lens) + 1
    k, v = _filled(nb, hk, bs, d, 25), _filled(nb, hk, bs, d, 26)
    table = _table(lens, bs, nb, g)
    q = torch.randn(n * len(lens), 4, d, generator=g).half()
    got, lse = _check(q, k, v, table, [max(x, n) for x in lens] if n <= min(lens) else lens, [n] * len(lens),
                      max_q_len=n, max_kv_len=max(lens))
    for _ in range(3):
        again, l2 = _check(q, k, v, table, lens, [n] * len(lens), max_q_len=n, max_kv_len=max(lens))
        assert torch.equal(again, got) and torch.equal(l2, lse)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_read_of_mixed_lists(d):
    """Runs of all lengths from every place, single tokens and what is outside, in lists of odd lengths."""
    bs, hk, nb = 64, 5, 40
    k, v = _filled(nb, hk, bs, d, 30), _filled(nb, hk, bs, d, 31)
    cache = _cache(k, v)
    refs = [o.values(*(_np(t) for t in side)) for side in (k, v)]
    for n in (17, 49, 1650, 2003):
        r, slots = np.random.default_rng(n), []
        while len(slots) < n:
            at = int(r.integers(-5, nb * bs))
            slots += range(at, at + int(r.choice([1, 1, 1, 2, 7, 8, 9, 31, 70])))
            if r.random() < 0.3:
                slots += [int(r.integers(0, nb * bs))] * 2 + r.integers(0, nb * bs, int(r.integers(0, 40))).tolist()
        slots = np.array(slots[:n], np.int32)
        got = cache.read(torch.from_numpy(slots).to(DEV), torch.float32)
        inside = (slots >= 0) & (slots < nb * bs)
        at = np.clip(slots, 0, nb * bs - 1)
        for ref, y in zip(refs, got):
            assert np.array_equal(_np(y), ref[at // bs, :, at % bs] * inside[:, None, None]), n
