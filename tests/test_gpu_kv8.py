"""The int8 paged cache's kernels against oracle/kv8.py in 64 bits (MI355X only).

Tolerances follow from the arithmetic.  u is the output type's unit roundoff
(fp16 2^-11, bf16 2^-8), d the head size.
  * norm and rotation: fp32 sums of d squares and four more operations per
    value, each within 2^-23 of the row's largest value, then one rounding:
    u |y| + (d / 8 + 16) 2^-23 max|y| (the sum is a tree of d / 8 terms a lane).
  * append: x / step and its rounding are exact except where the quotient lies
    within 2^-15 of a tie (step has two fp32 roundings: 127 * 2^-23 < 2^-15); there the
    neighbouring integer is right too.
  * attention: scores are fp32 sums of d products: |ds| <= (d + 8) 2^-24 size with
    size = max_j sum |q k_j| scale; p = 2^x is within 2^-22 (1 + |x|) and rounded to
    fp16 (2^-11), weights below the fp16 range lose at most n 2^-32 max|v|:
    |o - ref| <= u |ref| + (2^-11 + 2 ds + 2^-18) sum p|v| / sum p + n 2^-32 max|v|.
    lse: ds + 2^-18 + 2^-22 |lse|.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import rhinoforge_amd as rf
from oracle import kv8 as o

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _say(*a):
    print(*a, flush=True)


def _rng(seed):
    return torch.Generator().manual_seed(seed)


def _np(t):
    return t.detach().cpu().double().numpy()


# ---- norms and rotation ----------------------------------------------------------

ROPE = [
    # tokens, heads, kv_heads, head_dim, rot, dtype, interleaved, norms, positions
    (1, 32, 8, 128, 128, torch.float16, False, "both", "int64"),
    (3, 16, 8, 128, 64, torch.bfloat16, False, "both", "int32"),
    (17, 8, 1, 256, 256, torch.bfloat16, False, "none", "none"),
    (5, 28, 4, 128, 128, torch.float16, True, "q", "int64"),
    (2, 12, 12, 64, 32, torch.float16, True, "both", "int32"),
    (4, 3, 1, 80, 80, torch.float16, False, "k", "int32"),
    (6, 1, 1, 96, 48, torch.bfloat16, False, "both", "int64"),
    (2, 2, 1, 8, 0, torch.float16, False, "both", "none"),
    (2, 5, 2, 512, 512, torch.float16, False, "both", "int64"),
    (1030, 2, 1, 64, 64, torch.float16, False, "both", "int64"),
    (9, 3, 2, 40, 16, torch.bfloat16, True, "none", "int32"),
]


@pytest.mark.parametrize("case", ROPE, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("strided", [False, True])
def test_norm_rope(case, strided):
    t, hq, hk, d, rot, dt, inter, norms, posk = case
    _say("rope", case, strided)
    g = _rng(t * 31 + d)
    rows = max(t, 50)
    width = (hq + 2 * hk) * d
    fused = (torch.randn(t, width, generator=g) * torch.where(torch.rand(t, 1, generator=g) < 0.2, 1e-3, 3.0)).to(dt)
    fused[0, :d] = 0  # a head of zeros: the norm's eps
    f = fused.to(DEV)
    q = f[:, : hq * d].unflatten(1, (hq, d))
    k = f[:, hq * d: (hq + hk) * d].unflatten(1, (hk, d))
    if not strided:
        q, k = q.contiguous(), k.contiguous()
    qw = torch.randn(d, generator=g).to(dt) if norms in ("both", "q") else None
    kw = torch.randn(d, generator=g).to(dt) if norms in ("both", "k") else None
    cos = sin = pos = None
    if rot:
        ang = torch.rand(rows, rot // 2, generator=g) * 6.3
        cos, sin = ang.cos(), ang.sin()
        if posk != "none":
            pos = torch.randint(0, rows, (t,), generator=g).to(getattr(torch, posk))
    dev = lambda x: None if x is None else x.to(DEV)  # noqa: E731
    got = rf.qk_norm_rope(q, k, dev(qw), dev(kw), dev(cos), dev(sin), dev(pos), eps=1e-6, interleaved=inter)
    for x, w, y in ((q, qw, got[0]), (k, kw, got[1])):
        assert y.dtype == dt and y.is_contiguous() and y.shape == x.shape
        ref = o.norm_rope(_np(x), None if w is None else _np(w), None if cos is None else _np(cos),
                          None if sin is None else _np(sin), None if pos is None else pos.tolist(), 1e-6, inter)
        tol = UNIT[dt] * np.abs(ref) + (d / 8 + 16) * 2.0 ** -23 * np.abs(ref).max(-1, keepdims=True) + 2.0 ** -25
        err = np.abs(_np(y) - ref)
        assert (err <= tol).all(), (err / tol).max()


def test_norm_rope_positions_outside_the_table_give_nan():
    q = torch.ones(4, 2, 64, dtype=torch.float16, device=DEV)
    k = torch.ones(4, 1, 64, dtype=torch.float16, device=DEV)
    cos = torch.ones(10, 16, device=DEV)  # 32 of 64 dimensions are rotated
    pos = torch.tensor([0, -1, 10, 9], device=DEV)
    yq, yk = rf.qk_norm_rope(q, k, None, None, cos, cos, pos)
    for y in (yq, yk):
        assert torch.isfinite(y[[0, 3]]).all() and torch.isnan(y[[1, 2]]).all()


# ---- block tables ----------------------------------------------------------------

def _plan_case(b, new, cached, bs, seed, width=None, free=None, pad=0, start=3):
    r = np.random.default_rng(seed)
    c = r.integers(0, cached + 1, b).astype(np.int32)
    n = r.integers(0, new + 1, b).astype(np.int32)
    if seed % 3 == 1 and b > 1:
        c[r.integers(b)] = -5
        n[r.integers(b)] = -2
    c0, n0 = np.maximum(c, 0), np.maximum(n, 0)
    need = int((-(-(c0 + n0) // bs) - -(-c0 // bs)).sum())
    w = width or max(1, int((-(-(c0 + n0) // bs)).max()))
    have = -(-c0 // bs)
    ids = r.permutation(int(have.sum()) + need + 50).astype(np.int32)
    table = np.full((b, w), -1, np.int32)
    at = 0
    for i in range(b):
        m = min(int(have[i]), w)
        table[i, :m] = ids[at:at + m]
        at += m
    fl = ids[at:at + (need + 10 if free is None else free) + start]
    return table, c, n, fl, start, int(n0.sum()) + pad


@pytest.mark.parametrize("b,new,cached,bs,kw", [
    (1, 1, 0, 32, {}), (1, 1, 31, 32, {}), (1, 300, 100, 64, {}), (7, 1, 500, 64, {}),
    (64, 40, 300, 128, {"pad": 9}), (300, 3, 100, 32, {}), (5, 100, 50, 32, {"free": 4}),
    (6, 100, 50, 32, {"width": 2}), (4, 50, 60, 64, {"free": 0, "start": 0}), (8192, 2, 70, 32, {}),
    (257, 700, 300, 32, {"pad": 1000}), (2, 0, 40, 32, {}), (2, 0, 0, 32, {"pad": 3}),
])
@pytest.mark.parametrize("strided", [False, True])
def test_plan(b, new, cached, bs, kw, strided):
    _say("plan", b, new, cached, bs, kw)
    for seed in range(3):
        table, c, n, free, start, total = _plan_case(b, new, cached, bs, seed + b, **kw)
        ref = o.plan(table, c, n, free, start, total, bs)
        td = torch.from_numpy(table).to(DEV)
        if strided:
            wide = torch.full((b, table.shape[1] + 3), -7, dtype=torch.int32, device=DEV)
            wide[:, : table.shape[1]] = td
            td = wide[:, : table.shape[1]]
        dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(DEV)  # noqa: E731
        p = rf.kv8_plan(td, dev(c), dev(n), dev(free), torch.tensor([start], dtype=torch.int32, device=DEV),
                        total, bs)
        for name, got, want in (("table", td, ref[0]), ("slots", p.slots, ref[1]),
                                ("positions", p.positions, ref[2]), ("cu", p.cu_new, ref[3]),
                                ("lens", p.kv_lens, ref[4]), ("free_next", p.free_next, [ref[5]])):
            assert np.array_equal(got.cpu().numpy(), np.asarray(want)), name
        if strided:
            assert (wide[:, table.shape[1]:] == -7).all()


# ---- append and read ---------------------------------------------------------------

def _filled(nb, hk, bs, d, seed, loud=1.0):
    g = _rng(seed)
    kq = torch.randint(-127, 128, (nb, hk, bs, d), dtype=torch.int8, generator=g)
    vq = torch.randint(-127, 128, (nb, hk, bs, d), dtype=torch.int8, generator=g)
    ks = torch.rand(nb, hk, generator=g) * 0.02 * loud + 1e-3
    vs = torch.rand(nb, hk, generator=g) * 0.02 * loud + 1e-3
    return kq, ks, vq, vs


APPEND = [
    # kv_heads, head_dim, block_size, dtype, runs of (block, offset, tokens)
    (2, 128, 64, torch.float16, [(3, 5, 1)]),
    (1, 64, 32, torch.bfloat16, [(0, 0, 1), (2, 31, 1), (1, 7, 25)]),
    (8, 128, 64, torch.float16, [(1, 0, 64), (4, 0, 64), (0, 0, 13)]),
    (4, 128, 32, torch.bfloat16, [(5, 30, 2), (6, 0, 32), (7, 0, 9), (2, 15, 3)]),
    (1, 256, 128, torch.float16, [(2, 100, 28), (0, 0, 128), (1, 0, 70)]),
    (3, 256, 32, torch.bfloat16, [(4, 16, 5)]),
    (2, 64, 128, torch.float16, [(4, 33, 60), (5, 1, 127), (0, 127, 1)]),
    (2, 128, 64, torch.float16, [(b, (7 * b) % 64, 1) for b in range(9)]),
]


@pytest.mark.parametrize("case", range(len(APPEND)))
@pytest.mark.parametrize("size", [0.05, 1.0, 8.0])
@pytest.mark.parametrize("many", [False, True])
def test_append_and_read(case, size, many):
    """`many`: the same after a long stretch of skipped tokens (the launch for prompts)."""
    hk, d, bs, dt, runs = APPEND[case]
    _say("append", APPEND[case], size, many)
    nb = 10
    kq, ks, vq, vs = _filled(nb, hk, bs, d, case)
    cache = rf.KV8Cache.from_quantized(*(t.to(DEV) for t in (kq, ks, vq, vs)))
    slots = [b * bs + off + i for b, off, n in runs for i in range(n)]
    if many:
        slots = [-1] * 4099 + slots
    t = len(slots)
    g = _rng(100 + case)
    fused = (torch.randn(t, 3 * hk * d, generator=g) * size).to(dt)
    f = fused.to(DEV)
    k, v = (f[:, i * hk * d:(i + 1) * hk * d].unflatten(1, (hk, d)) for i in (0, 2))
    if case % 2:
        k = k.contiguous()
    sd = torch.tensor(slots, dtype=torch.int32, device=DEV)
    rf.kv8_append(cache, k, v, sd)
    gk, gks, gv, gvs = cache.to_quantized()
    for name, x, q0, s0, got, gscale in (("k", k, kq, ks, gk, gks), ("v", v, vq, vs, gv, gvs)):
        q, scale, quot = o.append(q0.numpy(), s0.numpy(), _np(x), slots)
        assert np.abs(_np(gscale) / scale - 1).max() <= 2.0 ** -22, name
        diff = _np(got) - q
        tie = np.abs(np.abs(quot - np.floor(quot)) - 0.5) < 2.0 ** -15
        assert ((diff == 0) | (tie & (np.abs(diff) == 1))).all(), name
    used = [s for s in slots if s >= 0]
    ask = torch.tensor([used[0], -1, nb * bs, used[-1], 0], dtype=torch.int32, device=DEV)
    for rdt in (torch.float16, torch.bfloat16, torch.float32):
        rk, rv = rf.kv8_read(cache, ask, rdt)
        for r, q, s in ((rk, gk, gks), (rv, gv, gvs)):
            want = torch.zeros(5, hk, d, device=DEV)
            for i, sl in enumerate(ask.tolist()):
                if 0 <= sl < nb * bs:
                    want[i] = q[sl // bs, :, sl % bs].float() * s[sl // bs][:, None]
            assert r.dtype == rdt and torch.equal(r, want.to(rdt))


def test_append_piece_by_piece_holds_the_largest_magnitude():
    """Single tokens into one block: each step's values are within half a step
    of what was appended, plus half a step per earlier rounding."""
    hk, d, bs = 2, 64, 32
    cache = rf.KV8Cache(2, hk, d, bs)
    g = _rng(9)
    x = torch.randn(bs, hk, d, generator=g).half() * torch.linspace(0.1, 3, bs).half()[:, None, None]
    raised = 0
    for i in range(bs):
        xi = x[i:i + 1].to(DEV)
        rf.kv8_append(cache, xi, -xi, torch.tensor([bs + i], dtype=torch.int32, device=DEV))
    rk, rv = rf.kv8_read(cache, torch.arange(bs, 2 * bs, dtype=torch.int32, device=DEV), torch.float32)
    step = cache.k_scale[1].cpu()
    amax = x.float().abs().amax((0, 2))
    assert torch.allclose(step, amax / 127, rtol=1e-6)
    run = x.float().abs().amax(2).cummax(0).values  # [bs, hk]: scale history times 127
    for h in range(hk):
        for i in range(bs):
            raised = int((run[i + 1:, h] > run[i:-1, h]).sum()) if i < bs - 1 else 0
            bound = 0.5 * (1 + raised) * step[h].item() * 1.001
            assert (rk[i, h].cpu() - x[i, h].float()).abs().max() <= bound
            assert (rv[i, h].cpu() + x[i, h].float()).abs().max() <= bound


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_append_of_values_that_are_not_finite(bad):
    hk, d, bs = 2, 64, 32
    cache = rf.KV8Cache(3, hk, d, bs)
    x = torch.ones(4, hk, d, dtype=torch.float16)
    x[2, 1, 5] = bad
    xd = x.to(DEV)
    slots = torch.tensor([32, 33, 34, 64], dtype=torch.int32, device=DEV)
    rf.kv8_append(cache, xd, torch.ones_like(xd), slots)
    rk, rv = rf.kv8_read(cache, slots)
    assert torch.isfinite(rv).all() and torch.isfinite(rk[:, 0]).all() and torch.isfinite(rk[3]).all()
    assert torch.isnan(rk[:3, 1]).all()
    # later tokens of that block do not make it finite again; a fresh block is
    rf.kv8_append(cache, xd[:1], xd[:1], torch.tensor([35], dtype=torch.int32, device=DEV))
    assert torch.isnan(rf.kv8_read(cache, slots)[0][:3, 1]).all()
    rf.kv8_append(cache, xd[:1], xd[:1], torch.tensor([32], dtype=torch.int32, device=DEV))
    assert torch.isfinite(rf.kv8_read(cache, slots[:1])[0]).all()


def test_append_of_zeros_and_of_tiny_values():
    cache = rf.KV8Cache(2, 1, 64, 32)
    cache.k_scale.fill_(float("nan"))  # a free block's old scale does not count
    cache.v_scale.fill_(float("nan"))
    x = torch.zeros(3, 1, 64, dtype=torch.bfloat16, device=DEV)
    x[2] = 2.0 ** -120
    slots = torch.tensor([0, 1, 32], dtype=torch.int32, device=DEV)
    rf.kv8_append(cache, x, x, slots)
    assert (cache.k_scale == 0).all() and (rf.kv8_read(cache, slots)[0] == 0).all()


def test_append_skips_slots_outside_the_cache():
    kq, ks, vq, vs = (t.to(DEV) for t in _filled(2, 1, 32, 64, 1))
    cache = rf.KV8Cache.from_quantized(kq, ks, vq, vs)
    x = torch.ones(5, 1, 64, dtype=torch.float16, device=DEV)
    rf.kv8_append(cache, x, x, torch.tensor([-1, 64, 2 ** 31 - 1, -2 ** 31, 65], dtype=torch.int32, device=DEV))
    for a, b in zip(cache.to_quantized(), (kq, ks, vq, vs)):
        assert torch.equal(a, b)


# ---- attention -----------------------------------------------------------------------

def _batch(lens, news, bs, seed, extra=2):
    r = np.random.default_rng(seed)
    counts = [-(-n // bs) for n in lens]
    nb = sum(counts) + 3
    ids = r.permutation(nb).astype(np.int32)
    width = max(1, max(counts)) + extra
    table = np.full((len(lens), width), -1, np.int32)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = ids[at:at + c]
        at += c
    cu = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    return table, cu, nb, ids[at:]


def _check_attention(q, cache_np, table, lens, cu, got, lse, dt, **kw):
    kq, ks, vq, vs = cache_np
    ref, rlse, mass, size = o.attention(_np(q), kq, ks, vq, vs, table, lens, cu, **kw)
    d = q.shape[2]
    ds = (d + 8) * 2.0 ** -24 * size[..., None]
    vmax = np.abs(vq).max() * np.abs(vs[np.isfinite(vs)]).max()
    tol = (UNIT[dt] * np.abs(ref) + (2.0 ** -11 + 2 * ds + 2.0 ** -18) * mass
           + max(lens) * 2.0 ** -32 * vmax + 2.0 ** -25)
    err = np.abs(_np(got) - ref)
    assert np.isfinite(_np(got)).all()
    assert (err <= tol).all(), f"worst {(err / tol).max():.2f} of the bound"
    if lse is not None:
        gl = _np(lse)
        none = np.isneginf(rlse)
        assert np.array_equal(np.isneginf(gl), none)
        bound = (ds[..., 0] + 2.0 ** -18 + 2.0 ** -22 * np.abs(np.where(none, 0, rlse)))[~none]
        assert (np.abs(gl - rlse)[~none] <= bound).all()


# lens (kv), news (queries), heads, kv_heads, head_dim, bs, dtype, options
ATTEND = [
    ([1], [1], 1, 1, 64, 32, torch.float16, {}),
    ([31], [1], 4, 1, 128, 32, torch.bfloat16, {}),
    ([32, 33, 0, 1, 64], [1, 1, 1, 1, 1], 8, 2, 128, 32, torch.float16, {}),
    ([777], [1], 32, 8, 128, 64, torch.float16, {}),
    ([4097, 5, 1030], [1, 1, 1], 28, 4, 128, 64, torch.bfloat16, {}),
    ([600, 129], [1, 1], 8, 1, 256, 128, torch.float16, {}),
    ([600, 129], [1, 1], 8, 1, 256, 32, torch.bfloat16, {"window": 100}),
    ([200, 63], [1, 1], 12, 12, 64, 64, torch.float16, {"window": 1}),
    ([500, 40, 3], [5, 7, 3], 16, 8, 128, 64, torch.float16, {}),
    ([500, 40], [9, 2], 8, 1, 256, 64, torch.float16, {"window": 33}),
    ([260, 100], [4, 8], 28, 4, 128, 32, torch.bfloat16, {"causal": False}),
    ([90, 10, 7], [6, 10, 9], 4, 2, 64, 32, torch.float16, {}),            # more queries than tokens
    ([130, 64, 257], [130, 1, 100], 8, 2, 128, 64, torch.float16, {}),     # prompts: 128-row tiles
    ([200, 33], [70, 33], 28, 4, 128, 64, torch.bfloat16, {"window": 40}),
    ([300], [300], 2, 2, 64, 32, torch.float16, {}),
    ([300, 170], [150, 170], 4, 1, 256, 128, torch.bfloat16, {}),
    ([96, 18], [50, 18], 8, 1, 256, 32, torch.bfloat16, {"causal": False}),
    ([700, 0, 5], [40, 20, 30], 16, 4, 128, 64, torch.float16, {}),        # nothing to see
    ([1200], [129], 4, 2, 128, 64, torch.float16, {"window": 300}),
    ([2500], [33], 8, 2, 64, 64, torch.bfloat16, {}),
    ([2500], [33], 16, 2, 256, 64, torch.float16, {}),
]


@pytest.mark.parametrize("case", range(len(ATTEND)))
@pytest.mark.parametrize("form", ["plain", "hints", "strided"])
def test_attention(case, form):
    lens, news, hq, hk, d, bs, dt, opt = ATTEND[case]
    _say("attend", ATTEND[case], form)
    table, cu, nb, spare = _batch(lens, news, bs, case)
    g = _rng(case)
    kq, ks, vq, vs = _filled(nb, hk, bs, d, 50 + case)
    # blocks that no request owns hold a scale of NaN: nothing of them may be read
    for b in spare:
        ks[b], vs[b] = float("nan"), float("nan")
    cache = rf.KV8Cache.from_quantized(*(t.to(DEV) for t in (kq, ks, vq, vs)))
    total = int(cu[-1])
    wide = (torch.randn(total, hq + 3, d + 8, generator=g) * 2).to(dt).to(DEV)
    q = wide[:, 1:1 + hq, :d]
    td = torch.from_numpy(table).to(DEV)
    kw = dict(scale=d ** -0.5, **opt)
    hints = {}
    if form == "hints":
        hints = {"max_q_len": max(news), "max_kv_len": max(lens)}
    if form == "strided":
        big = torch.full((len(lens), table.shape[1] + 5), 2 ** 30, dtype=torch.int32, device=DEV)
        big[:, : table.shape[1]] = td
        td = big[:, : table.shape[1]]
    else:
        q = q.contiguous()
    out, lse = rf.kv8_attention(q, cache, td, torch.tensor(lens, dtype=torch.int32, device=DEV),
                                torch.from_numpy(cu).to(DEV), return_lse=True, **kw, **hints)
    torch.cuda.synchronize()
    _check_attention(q, (kq.numpy(), ks.numpy(), vq.numpy(), vs.numpy()), table, lens, cu, out, lse, dt, **kw)
    again = rf.kv8_attention(q, cache, td, torch.tensor(lens, dtype=torch.int32, device=DEV),
                             torch.from_numpy(cu).to(DEV), **kw, **hints)
    assert torch.equal(again, out)  # the same bits, with and without the lse


@pytest.mark.parametrize("n", [1, 3, 40])
def test_attention_of_equal_numbers_of_queries_without_offsets(n):
    lens, hq, hk, d, bs = [100, 0, 64], 8, 2, 64, 32
    table, cu, nb, _ = _batch(lens, [n] * 3, bs, n)
    kq, ks, vq, vs = _filled(nb, hk, bs, d, n)
    cache = rf.KV8Cache.from_quantized(*(t.to(DEV) for t in (kq, ks, vq, vs)))
    q = torch.randn(3 * n, hq, d, generator=_rng(n)).half().to(DEV)
    args = (q, cache, torch.from_numpy(table).to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV))
    a = rf.kv8_attention(*args)
    _check_attention(q, (kq.numpy(), ks.numpy(), vq.numpy(), vs.numpy()), table, lens, cu, a, None,
                     torch.float16, scale=d ** -0.5)
    b = rf.kv8_attention(*args, torch.from_numpy(cu).to(DEV), max_q_len=n)
    assert torch.equal(a, b)


def test_attention_scales_far_apart_and_peaked_scores():
    """Value scales from 1e-6 to 1e3 from block to block (the weight of each
    block's values differs by as much), and queries 30 times larger."""
    d, bs, hq, hk = 128, 32, 8, 2
    for seed, loud in ((0, 1.0), (1, 30.0)):
        for n in (1, 60):
            lens, news = [700], [n]
            table, cu, nb, _ = _batch(lens, news, bs, seed)
            kq, ks, vq, vs = _filled(nb, hk, bs, d, seed)
            vs = 10.0 ** (torch.rand(nb, hk, generator=_rng(seed)) * 9 - 6)
            vs[int(table[0, 3])] = 0.0     # a block of zeros
            vq[int(table[0, 3])] = 0
            ks[int(table[0, 5])] = 0.0
            kq[int(table[0, 5])] = 0
            cache = rf.KV8Cache.from_quantized(*(t.to(DEV) for t in (kq, ks, vq, vs)))
            q = (torch.randn(n, hq, d, generator=_rng(seed)) * loud).half().to(DEV)
            out, lse = rf.kv8_attention(q, cache, torch.from_numpy(table).to(DEV),
                                        torch.tensor(lens, dtype=torch.int32, device=DEV),
                                        torch.from_numpy(cu).to(DEV), return_lse=True)
            fin = [t.numpy() for t in (kq, ks, vq, vs)]
            ok = torch.isfinite(out)
            ref = o.attention(_np(q), *fin, table, lens, cu, scale=d ** -0.5)
            big = np.abs(ref[0]) > 6e4    # past fp16's range
            assert np.array_equal(~ok.cpu().numpy() & ~big, np.zeros_like(big))
            out = torch.where(torch.from_numpy(big).to(DEV), torch.zeros_like(out), out)
            d_s = (d + 8) * 2.0 ** -24 * ref[3][..., None]
            tol = (2.0 ** -11 * np.abs(ref[0]) + (2.0 ** -11 + 2 * d_s + 2.0 ** -18) * ref[2]
                   + 700 * 2.0 ** -32 * 127 * float(vs.max()) + 2.0 ** -25)
            assert (np.abs(_np(out) - np.where(big, 0, ref[0])) <= tol).all()


@pytest.mark.parametrize("size", [1e-20, 1e20, 1e30])
def test_attention_bf16_queries_past_the_range_of_fp16(size):
    d, bs, lens = 64, 32, [90]
    table, cu, nb, _ = _batch(lens, [1], bs, 0)
    kq, ks, vq, vs = _filled(nb, 1, bs, d, 3)
    cache = rf.KV8Cache.from_quantized(*(t.to(DEV) for t in (kq, ks, vq, vs)))
    q = (torch.randn(1, 2, d, generator=_rng(1)) * size).bfloat16().to(DEV)
    scale = 1.0 / size
    out = rf.kv8_attention(q, cache, torch.from_numpy(table).to(DEV),
                           torch.tensor(lens, dtype=torch.int32, device=DEV), scale=scale)
    _check_attention(q, (kq.numpy(), ks.numpy(), vq.numpy(), vs.numpy()), table, lens, cu, out, None,
                     torch.bfloat16, scale=scale)


@pytest.mark.parametrize("n", [1, 50])
def test_attention_nan_stays_where_it_is_seen(n):
    """A block of NaN counts only for queries that see its tokens; a block id
    outside the cache gives NaN for its request alone; NaN queries for their own."""
    d, bs, hq, hk = 64, 32, 4, 2
    lens, news = [200, 200, 70], [n, n, n]
    table, cu, nb, spare = _batch(lens, news, bs, 4)
    kq, ks, vq, vs = _filled(nb, hk, bs, d, 4)
    ks[int(table[0, 0]), 1] = float("nan")   # request 0, key head 1: block of tokens 0..31
    vs[int(table[2, 2]), 0] = float("inf")   # request 2, value head 0: tokens 64..69
    cache = rf.KV8Cache.from_quantized(*(t.to(DEV) for t in (kq, ks, vq, vs)))
    q = torch.randn(3 * n, hq, d, generator=_rng(4)).half()
    qd = q.to(DEV)
    args = (torch.from_numpy(table).to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV),
            torch.from_numpy(cu).to(DEV))
    out = rf.kv8_attention(qd, cache, *args)
    nan = torch.isnan(out).cpu()
    want = torch.zeros_like(nan)
    want[:n, 2:] = True                       # request 0, the two heads on key head 1
    for i in range(n):
        if 70 - n + i >= 64:
            want[2 * n + i, :2] = True
    assert torch.equal(nan, want)
    out = rf.kv8_attention(qd, cache, *args, window=100)  # request 0's block 0 is out of sight
    assert torch.isfinite(out[:n]).all()
    table2 = table.copy()
    table2[1, 1] = nb + 5
    out = rf.kv8_attention(qd, cache, torch.from_numpy(table2).to(DEV), *args[1:])
    assert torch.isnan(out[n:2 * n]).all() and not torch.isnan(out[:n, :2]).any()
    q[0, 0, 3] = float("nan")
    out = rf.kv8_attention(q.to(DEV), cache, *args)
    assert torch.isnan(out[0, 0]).all() and not torch.isnan(out[0, 1]).any()


def test_attention_tokens_past_the_batch_and_lengths_past_the_table():
    d, bs = 64, 32
    lens, news = [50, 20], [3, 2]
    table, cu, nb, _ = _batch(lens, news, bs, 7, extra=0)
    kq, ks, vq, vs = _filled(nb, 1, bs, d, 7)
    cache = rf.KV8Cache.from_quantized(*(t.to(DEV) for t in (kq, ks, vq, vs)))
    for pad, hint in ((4, 3), (300, 0)):
        q = torch.randn(5 + pad, 2, d, generator=_rng(7)).half().to(DEV)
        out, lse = rf.kv8_attention(q, cache, torch.from_numpy(table).to(DEV),
                                    torch.tensor(lens, dtype=torch.int32, device=DEV),
                                    torch.from_numpy(cu).to(DEV), max_q_len=hint, return_lse=True)
        assert (out[5:] == 0).all() and torch.isneginf(lse[5:]).all()
        _check_attention(q[:5], (kq.numpy(), ks.numpy(), vq.numpy(), vs.numpy()), table, lens, cu, out[:5],
                         lse[:5], torch.float16, scale=d ** -0.5)
    # a length past the table counts as the table's width
    long = torch.tensor([10 ** 9, 20], dtype=torch.int32, device=DEV)
    full = torch.tensor([64, 20], dtype=torch.int32, device=DEV)
    a = rf.kv8_attention(q[:5], cache, torch.from_numpy(table).to(DEV), long, torch.from_numpy(cu).to(DEV))
    b = rf.kv8_attention(q[:5], cache, torch.from_numpy(table).to(DEV), full, torch.from_numpy(cu).to(DEV))
    assert torch.equal(a, b)


def test_no_tokens_at_all():
    cache = rf.KV8Cache(2, 1, 64, 32)
    e = torch.empty(0, 1, 64, dtype=torch.float16, device=DEV)
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    one = torch.zeros(1, dtype=torch.int32, device=DEV)
    rf.kv8_append(cache, e, e, none)
    assert rf.kv8_read(cache, none)[0].shape == (0, 1, 64)
    assert rf.kv8_attention(e, cache, one[:, None], one).shape == (0, 1, 64)
    assert rf.qk_norm_rope(e, e, None, None, None, None)[0].shape == (0, 1, 64)


def test_a_cache_past_32_bits_of_offsets():
    """Blocks whose bytes lie past 2^32: append, read and attention reach them."""
    hk, d, bs = 8, 256, 128
    nb = 2 ** 32 // (hk * d * bs) + 40
    cache = rf.KV8Cache(nb, hk, d, bs)
    assert cache.k.numel() > 2 ** 32
    blocks = [nb - 1, nb - 7, 3]
    n = 300
    g = _rng(1)
    k, v = (torch.randn(n, hk, d, generator=g).half() for _ in range(2))
    slots = torch.tensor([blocks[i // bs] * bs + i % bs for i in range(n)], dtype=torch.int32, device=DEV)
    rf.kv8_append(cache, k.to(DEV), v.to(DEV), slots)
    rk, rv = rf.kv8_read(cache, slots, torch.float32)
    for r, x in ((rk, k), (rv, v)):
        assert (r.cpu() - x.float()).abs().max() <= 0.51 * x.float().abs().max() / 127
    q = torch.randn(1, 2 * hk, d, generator=g).half().to(DEV)
    table = torch.tensor([blocks], dtype=torch.int32, device=DEV)
    for rows in (1, 40):
        qq = q.expand(rows, -1, -1)
        out = rf.kv8_attention(qq, cache, table, torch.tensor([n], dtype=torch.int32, device=DEV), causal=False)
        s = (q[0].view(hk, 2, d).double().cpu() @ rk.double().cpu().permute(1, 2, 0)) * d ** -0.5
        ref = (torch.softmax(s, -1) @ rv.double().cpu().transpose(0, 1)).reshape(2 * hk, d)
        assert (out[-1].double().cpu() - ref).abs().max() <= 2e-3


# ---- streams and graphs ----------------------------------------------------------------

def _step(cache, qkv, wq, wk, cos, sin, table, cached, new, free, start, hq, hk, d):
    """One decode step's attention side on the current stream."""
    p = rf.kv8_plan(table, cached, new, free, start, qkv.size(0), cache.block_size)
    q = qkv[:, : hq * d].unflatten(1, (hq, d))
    k = qkv[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d))
    v = qkv[:, (hq + hk) * d:].unflatten(1, (hk, d))
    q, k = rf.qk_norm_rope(q, k, wq, wk, cos, sin, p.positions)
    rf.kv8_append(cache, k, v, p.slots)
    return rf.kv8_attention(q, cache, table, p.kv_lens, p.cu_new, max_q_len=1)


def _step_state(seed):
    b, hq, hk, d, bs = 5, 8, 2, 128, 32
    lens = [70, 0, 31, 1300, 32]
    table, _, nb, spare = _batch(lens, [1] * b, bs, seed, extra=3)
    kq, ks, vq, vs = (t.to(DEV) for t in _filled(nb + 10, hk, bs, d, seed))
    g = _rng(seed)
    cos, sin = rf.rope_table(1e4 ** (-torch.arange(0, d, 2) / d).to(DEV), 2000)
    return dict(
        cache=rf.KV8Cache.from_quantized(kq, ks, vq, vs),
        qkv=torch.randn(b, (hq + 2 * hk) * d, generator=g).half().to(DEV),
        wq=torch.rand(d, generator=g).half().to(DEV), wk=torch.rand(d, generator=g).half().to(DEV),
        cos=cos, sin=sin, table=torch.from_numpy(table).to(DEV),
        cached=torch.tensor(lens, dtype=torch.int32, device=DEV),
        new=torch.ones(b, dtype=torch.int32, device=DEV),
        free=torch.arange(nb, nb + 10, dtype=torch.int32, device=DEV),
        start=torch.zeros(1, dtype=torch.int32, device=DEV), hq=hq, hk=hk, d=d)


def test_a_step_on_another_stream_is_the_same():
    a, b = _step_state(1), _step_state(1)
    ref = _step(**a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _step(**b)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(ref, got)
    for x, y in zip(a["cache"].tensors(), b["cache"].tensors()):
        assert torch.equal(x, y)


def test_a_captured_step_replays_with_new_inputs():
    """The whole step in one graph: replayed with other inputs and lengths, with
    eager work in between, each replay equals the eager step."""
    s = _step_state(2)
    warm = _step_state(2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(**warm)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(**s)
    for rep in range(3):
        e = _step_state(20 + rep)
        for name in ("qkv", "wq", "wk", "table", "cached", "free", "start", "new"):
            if name == "table":
                s[name].fill_(-1)
                s[name][:, : e[name].size(1)] = e[name]
            else:
                s[name].copy_(e[name])
        for x, y in zip(s["cache"].tensors(), e["cache"].tensors()):
            x.copy_(y)
        graph.replay()
        ref = _step(**e)
        torch.cuda.synchronize()
        assert torch.equal(out, ref), rep
        for x, y in zip(s["cache"].tensors(), e["cache"].tensors()):
            assert torch.equal(x, y)


# ---- refusals on device tensors -------------------------------------------------------

def test_refusals_on_the_device():
    cache = rf.KV8Cache(2, 2, 64, 32)
    q = torch.zeros(1, 4, 64, dtype=torch.float16, device=DEV)
    lens = torch.ones(1, dtype=torch.int32, device=DEV)
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="HIP device"):
        rf.kv8_attention(q, cache, table.cpu(), lens)
    with pytest.raises(RuntimeError, match="HIP device"):
        rf.kv8_append(cache, q[:, :2].cpu(), q[:, :2], lens)
    with pytest.raises(RuntimeError, match="HIP device"):
        rf.kv8_plan(table, lens.cpu(), lens, lens, lens, 1, 32)
    with pytest.raises(RuntimeError, match="int32"):
        rf.kv8_attention(q, cache, table.long(), lens)


# ---- attention of many requests of unequal lengths -------------------------------

@pytest.mark.parametrize("b", [2, 48, 63, 64, 65, 130, 511, 700, 2500])
@pytest.mark.parametrize("new", [1, 3, 20])
@pytest.mark.parametrize("hints", [False, True])
def test_attention_of_many_requests(b, new, hints):
    """Most requests short or empty, a few long: shares of all sizes, and every
    way of finding them (up to 64 requests at once, several a lane, searched for)."""
    _say("many", b, new, hints)
    d, bs, hq, hk = (64, 32, 4, 2) if b != 130 else (256, 64, 8, 1)
    r = np.random.default_rng(b * 7 + new)
    lens = r.integers(0, 60, b)
    long = r.integers(0, b, 2)
    lens[long] = r.integers(1500, 3001, 2)
    lens = [int(x) for x in lens]
    news = [new] * b if new == 1 else [int(x) for x in r.integers(0, new + 1, b)]
    opt = {"window": 777} if new == 3 else {}
    table, cu, nb, spare = _batch(lens, news, bs, b + new)
    kq, ks, vq, vs = _filled(nb, hk, bs, d, b)
    for i in spare:
        ks[i], vs[i] = float("nan"), float("nan")
    cache = rf.KV8Cache.from_quantized(*(t.to(DEV) for t in (kq, ks, vq, vs)))
    q = torch.randn(int(cu[-1]), hq, d, generator=_rng(b)).half()
    args = (q.to(DEV), cache, torch.from_numpy(table).to(DEV),
            torch.tensor(lens, dtype=torch.int32, device=DEV))
    args += () if new == 1 else (torch.from_numpy(cu).to(DEV),)
    kw = {**opt, **({"max_kv_len": max(lens)} if hints else {}),
          **({"max_q_len": max(news)} if hints and new > 1 else {})}
    out, lse = rf.kv8_attention(*args, return_lse=True, **kw)
    for _ in range(3):
        assert torch.equal(rf.kv8_attention(*args, **kw), out)
    _check_attention(q, (kq.numpy(), ks.numpy(), vq.numpy(), vs.numpy()), table, lens, cu, out, lse,
                     torch.float16, scale=d ** -0.5, **opt)


def test_attention_offsets_out_of_order_leave_the_next_call_right():
    """Offsets that go back ask for more tiles than the batch has: what such a call
    returns is not said, but it ends, and the calls after it are right."""
    d, bs, hq, hk, b = 64, 32, 4, 2, 40
    lens, news = [2000] * b, [9] * b
    table, cu, nb, _ = _batch(lens, news, bs, 3)
    kq, ks, vq, vs = _filled(nb, hk, bs, d, 3)
    cache = rf.KV8Cache.from_quantized(*(t.to(DEV) for t in (kq, ks, vq, vs)))
    q = torch.randn(int(cu[-1]), hq, d, generator=_rng(3)).half()
    args = (q.to(DEV), cache, torch.from_numpy(table).to(DEV),
            torch.tensor(lens, dtype=torch.int32, device=DEV))
    good = torch.from_numpy(cu).to(DEV)
    want = rf.kv8_attention(*args, good, max_q_len=9)
    bad = good.clone()
    bad[1:b:2] = 360
    for hint in (9, 0):
        rf.kv8_attention(*args, bad, max_q_len=hint)
        assert torch.equal(rf.kv8_attention(*args, good, max_q_len=9), want)
    _check_attention(q, (kq.numpy(), ks.numpy(), vq.numpy(), vs.numpy()), table, lens, cu, want, None,
                     torch.float16, scale=d ** -0.5)


@pytest.mark.parametrize("run", [1, 2, 7, 8, 9, 16])
@pytest.mark.parametrize("tokens", [15, 16, 17, 63, 65, 640, 2100])
@pytest.mark.parametrize("d,hk,bs", [(64, 12, 32), (128, 8, 64), (256, 1, 128)])
def test_append_of_many_short_runs(run, tokens, d, hk, bs):
    """Runs of `run` tokens, each in its own block behind `seen` held ones, some
    skipped: together, cut by chunk ends, at the ends of blocks."""
    _say("runs", run, tokens, d, bs)
    dt = torch.float16
    r = np.random.default_rng(run * 1000 + tokens)
    count = -(-tokens // run)
    kq, ks, vq, vs = _filled(count, hk, bs, d, tokens + run)
    cache = rf.KV8Cache.from_quantized(*(t.to(DEV) for t in (kq, ks, vq, vs)))
    seen = r.choice([0, 1, 5, bs - run], count)
    blocks = r.permutation(count)
    slots = [int(b) * bs + int(s) + j for b, s in zip(blocks, seen) for j in range(run)][:tokens]
    for i in range(count):
        if r.random() < 0.1:
            slots[i * run:(i + 1) * run] = [int(r.choice([-1, count * bs, 2 ** 31 - 200]))] * len(slots[i * run:(i + 1) * run])
    k, v = (torch.randn(tokens, hk, d, generator=_rng(s)).to(dt) * 2.0 ** -(s % 3) for s in (tokens, run + 5))
    rf.kv8_append(cache, k.to(DEV), v.to(DEV), torch.tensor(slots, dtype=torch.int32, device=DEV))
    gk, gks, gv, gvs = cache.to_quantized()
    for name, x, q0, s0, got, gscale in (("k", k, kq, ks, gk, gks), ("v", v, vq, vs, gv, gvs)):
        q, scale, quot = o.append(q0.numpy(), s0.numpy(), _np(x), slots)
        assert np.abs(_np(gscale) / scale - 1).max() <= 2.0 ** -22, name
        diff = _np(got) - q
        tie = np.abs(np.abs(quot - np.floor(quot)) - 0.5) < 2.0 ** -15
        assert ((diff == 0) | (tie & (np.abs(diff) == 1))).all(), name


@pytest.mark.parametrize("d,hk,bs", [(64, 3, 32), (128, 2, 64), (256, 1, 128)])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
def test_read_of_whole_groups_and_of_others(d, hk, bs, dt):
    """32 slots in a row are read together where they are a group of a block."""
    nb = 9
    kq, ks, vq, vs = _filled(nb, hk, bs, d, d)
    cache = rf.KV8Cache.from_quantized(*(t.to(DEV) for t in (kq, ks, vq, vs)))
    r = np.random.default_rng(d)
    group = lambda g: list(range(32 * g, 32 * g + 32))  # noqa: E731
    last = nb * bs // 32 - 1
    slots = group(last) + group(0) + group(3)[1:] + [5] + group(2)[::-1] + list(range(40, 72))
    slots += [nb * bs + i for i in range(32)] + [-1] * 32 + [int(x) for x in r.integers(0, nb * bs, 32)]
    slots += group(4)[:31] + [-1] + group(1)
    for n in (len(slots), len(slots) - 1, 33, 32, 31):
        rk, rv = rf.kv8_read(cache, torch.tensor(slots[:n], dtype=torch.int32, device=DEV), dt)
        for got, q, s in ((rk, kq, ks), (rv, vq, vs)):
            want = torch.zeros(n, hk, d)
            for i, sl in enumerate(slots[:n]):
                if 0 <= sl < nb * bs:
                    want[i] = q[sl // bs, :, sl % bs].float() * s[sl // bs][:, None]
            assert torch.equal(got.cpu(), want.to(dt))


# ---- prompts that fill the chip, or nearly: one gang of wavefronts a tile, or two,
# ---- with and without splits

PROMPTS = [
    ([499], [499], 64, 4, 128, torch.float16, {}),
    ([501], [501], 64, 4, 128, torch.bfloat16, {"causal": False}),
    ([1799], [500], 64, 4, 128, torch.bfloat16, {"window": 300}),
    ([1490, 203], [200, 100], 64, 4, 128, torch.float16, {}),
    ([2497, 40, 170], [180, 30, 90], 64, 4, 128, torch.float16, {}),
    ([2010], [400], 64, 8, 64, torch.bfloat16, {}),
    ([6001], [250], 64, 8, 64, torch.float16, {}),
    ([3170], [500], 32, 8, 128, torch.bfloat16, {}),
    ([600], [600], 64, 2, 64, torch.float16, {}),
    ([3000], [300], 64, 2, 64, torch.float16, {"window": 2000}),
    ([300, 64, 0], [300, 0, 200], 64, 4, 128, torch.float16, {}),   # rows that see nothing
    # fewer rows, many splits: joined by the last workgroup or added by a second kernel
    ([5000], [5], 16, 8, 128, torch.float16, {}),
    ([1000], [20], 16, 8, 128, torch.bfloat16, {}),
    ([5000], [60], 16, 8, 128, torch.float16, {}),
    ([5003], [9], 8, 1, 256, torch.float16, {}),
    ([3000], [40], 8, 1, 256, torch.bfloat16, {}),
    ([700], [700], 8, 1, 256, torch.float16, {}),
]


@pytest.mark.parametrize("case", range(len(PROMPTS)))
def test_attention_of_prompts(case):
    lens, news, hq, hk, d, dt, opt = PROMPTS[case]
    _say("prompt", PROMPTS[case])
    bs = 64
    table, cu, nb, spare = _batch(lens, news, bs, case)
    kq, ks, vq, vs = _filled(nb, hk, bs, d, 70 + case)
    vs = vs * 2.0 ** torch.randint(-6, 3, vs.shape, generator=_rng(case))
    for b in spare:
        ks[b], vs[b] = float("nan"), float("nan")
    cache = rf.KV8Cache.from_quantized(*(t.to(DEV) for t in (kq, ks, vq, vs)))
    q = (torch.randn(int(cu[-1]), hq, d, generator=_rng(case)) * 2).to(dt)
    args = (q.to(DEV), cache, torch.from_numpy(table).to(DEV),
            torch.tensor(lens, dtype=torch.int32, device=DEV), torch.from_numpy(cu).to(DEV))
    out, lse = rf.kv8_attention(*args, max_q_len=max(news), max_kv_len=max(lens), return_lse=True, **opt)
    assert torch.equal(rf.kv8_attention(*args, max_q_len=max(news), max_kv_len=max(lens), **opt), out)
    _check_attention(q, (kq.numpy(), ks.numpy(), vq.numpy(), vs.numpy()), table, lens, cu, out, lse, dt,
                     scale=d ** -0.5, **opt)
    # a block that is not finite reaches the queries that see it, and no others
    if lens[0] > 320 and opt.get("causal", True) and not opt:
        bad = ks.clone()
        bad[int(table[0, (lens[0] - 1) // bs]), 0] = float("inf")
        cache.k_scale.copy_(bad)
        nan = torch.isnan(rf.kv8_attention(*args, max_q_len=max(news), max_kv_len=max(lens))).cpu()
        first = (lens[0] - 1) // bs * bs - (lens[0] - news[0])   # the first query that sees it
        want = torch.zeros_like(nan)
        want[max(first, 0):news[0], :hq // hk] = True
        assert torch.equal(nan, want)
