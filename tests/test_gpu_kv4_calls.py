"""Calls of the 4-bit paged cache as a serving loop makes them (MI355X only): captured
steps, several streams and threads, batches of many requests, all launch forms,
layouts that the kernels do not read in place, caches past 4 GiB, and the whole
attention side of a layer.  Values are held to the tolerances of test_gpu_kv4.py, or
to equality where two calls do the same arithmetic."""
from __future__ import annotations

import threading

import numpy as np
import pytest
import torch

import rhinoforge_amd as rf
from oracle import kv4 as o
from test_gpu_kv4 import DEV, UNIT, _cache, _check, _filled, _np, _rng, _say, _table

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ---- batches and launch forms ------------------------------------------------------------

@pytest.mark.parametrize("b", [2, 61, 62, 63, 64, 65, 127, 200, 510, 511, 512, 513, 700])
@pytest.mark.parametrize("hq", [1, 8])
def test_batches_of_many_requests(b, hq):
    """One query a request, some with none or several, tokens behind the last one."""
    _say("requests", b, hq)
    g = _rng(b)
    lens = torch.randint(0, 80, (b,), generator=g).tolist()
    news = torch.where(torch.rand(b, generator=g) < 0.8, 1, torch.randint(0, 12, (b,), generator=g)).tolist()
    nb = sum(-(-n // 32) for n in lens) + 1
    k, v = _filled(nb, 1, 32, 64, 40), _filled(nb, 1, 32, 64, 41)
    q = torch.randn(sum(news), hq, 64, generator=g).half()
    table = _table(lens, 32, nb, g)
    got, lse = _check(q, k, v, table, lens, news, max_q_len=max(news))
    behind = torch.cat((q, q[:1].expand(9, hq, 64)))
    cu = np.concatenate(([0], np.cumsum(news)))
    out, lse2 = rf.kv4_attention(behind.to(DEV), _cache(k, v), table.to(DEV), _i32(lens), _i32(cu),
                                 max_q_len=max(news), return_lse=True)
    assert torch.equal(out[:-9], got) and torch.equal(lse2[:-9], lse)
    assert (out[-9:] == 0).all() and torch.isneginf(lse2[-9:]).all()


@pytest.mark.parametrize("b,most", [(3, 300), (63, 60), (100, 120), (511, 40), (530, 40)])
@pytest.mark.parametrize("d,hk", [(64, 2), (128, 1), (256, 1)])
def test_prompts_of_many_requests(b, most, d, hk):
    """Prompts of unequal lengths, some without tokens, some behind cached ones."""
    _say("prompts", b, most, d)
    g = _rng(b + d)
    news = torch.randint(0, most, (b,), generator=g).tolist()
    lens = [n + int(c) for n, c in zip(news, torch.randint(0, 50, (b,), generator=g))]
    nb = sum(-(-n // 64) for n in lens) + 1
    k, v = _filled(nb, hk, 64, d, 50), _filled(nb, hk, 64, d, 51)
    q = torch.randn(sum(news), 8, d, generator=g).half()
    _check(q, k, v, _table(lens, 64, nb, g), lens, news, max_q_len=max(news), max_kv_len=max(lens))


@pytest.mark.parametrize("heads", [(8, 2, 64), (8, 2, 128), (4, 1, 256), (64, 16, 128)])
@pytest.mark.parametrize("n", [1, 2, 4, 8, 40])
@pytest.mark.parametrize("context", [100, 2500, 17000])
def test_launch_forms(heads, n, context):
    """4, 8, 16, 32 and 160 rows a key head, one workgroup a tile to 64 of them."""
    _say("forms", heads, n, context)
    hq, hk, d = heads
    if context > 10000 and hk > 2:
        context //= 4
    g = _rng(context + n)
    nb = -(-(context + n) // 64) + 1
    k, v = _filled(nb, hk, 64, d, 42), _filled(nb, hk, 64, d, 43)
    q = torch.randn(n, hq, d, generator=g).bfloat16()
    first = _check(q, k, v, _table([context + n], 64, nb, g), [context + n], [n])
    again = _check(q, k, v, _table([context + n], 64, nb, _rng(context + n + 1)), [context + n], [n], cu=False)
    assert first[0].shape == again[0].shape


@pytest.mark.parametrize("lens", [[5000] * 3, [1, 0, 12000, 3], [700, 2900] * 12])
@pytest.mark.parametrize("n", [1, 5])
@pytest.mark.parametrize("window", [0, 333])
def test_ragged_contexts(lens, n, window):
    _say("ragged", lens[:4], n, window)
    g = _rng(len(lens))
    lens = [x + n for x in lens]
    nb = sum(-(-x // 128) for x in lens) + 1
    k, v = _filled(nb, 2, 128, 64, 44), _filled(nb, 2, 128, 64, 45)
    q = torch.randn(n * len(lens), 6, 64, generator=g).half()
    _check(q, k, v, _table(lens, 128, nb, g), lens, [n] * len(lens), window=window)


def test_offsets_that_are_not_in_order_stay_inside():
    """They name no batch; rows that no request claims are not written."""
    k, v = _filled(30, 2, 32, 128, 46), _filled(30, 2, 32, 128, 47)
    q = torch.randn(12, 4, 128, generator=_rng(1)).half().to(DEV)
    cache, table = _cache(k, v), torch.arange(30, dtype=torch.int32, device=DEV).view(3, 10)
    for cu in ([0, 9, 2, 12], [5, 4, 3, 2], [-7, 100, -100, 2 ** 31 - 1]):
        for lens in ([300, 10, 90], [2 ** 31 - 1, -5, 0]):
            out = rf.kv4_attention(q, cache, table, _i32(lens), _i32(cu))
            assert out.shape == q.shape
    torch.cuda.synchronize()


# ---- layouts -------------------------------------------------------------------------------

FORMS = ["odd stride", "unit stride elsewhere", "off by one value", "broadcast"]


def _laid_out(x, form):
    t, h, d = x.shape
    if form == "broadcast":
        return x[:1].expand(t, h, d)
    if form == "odd stride":
        y = torch.zeros(t, h, d + 3, dtype=x.dtype, device=DEV)[..., 1:d + 1]
    elif form == "unit stride elsewhere":
        y = torch.zeros(t, d, h, dtype=x.dtype, device=DEV).transpose(1, 2)
    else:
        y = torch.zeros(t * h * d + 1, dtype=x.dtype, device=DEV)[1:].view(t, h, d)
    return y.copy_(x)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("n", [1, 3, 70])
def test_layouts(form, n):
    _say("layouts", form, n)
    g = _rng(n)
    hq, hk, d, cached = 6, 2, 64, 100
    x = [torch.randn(n, h, d, generator=g).half().to(DEV) for h in (hq, hk, hk)]
    if form == "broadcast":
        x = [t[:1].expand_as(t).contiguous() for t in x]
    y = [_laid_out(t, form) for t in x]
    held = _cache(_filled(9, hk, 32, d, 48), _filled(9, hk, 32, d, 49)), _cache(_filled(9, hk, 32, d, 48), _filled(9, hk, 32, d, 49))
    table = torch.full((1, 11), -1, dtype=torch.int32, device=DEV)[:, 1:10].copy_(torch.randperm(9, generator=g))
    at = torch.arange(cached, cached + n, device=DEV)
    slots = (table[0, at // 32].long() * 32 + at % 32).int()
    wide = torch.zeros(n + 1, dtype=torch.int32, device=DEV)[1:].copy_(slots)
    lens, cu = _i32([0, cached + n])[1:], _i32([9, 0, n])[1:]
    outs = []
    for cache, (q, k, v), s in ((held[0], x, slots), (held[1], y, wide)):
        cache.append(k, v, s)
        outs.append(cache.attention(q, table, lens, cu, return_lse=True) + cache.read(s))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    a = rf.qk_norm_mrope(x[0], x[1], None, None, *(cs := torch.rand(2, 20, 32, device=DEV)),
                         at[None].expand(3, -1) % 20, [12, 10, 10], mixed=True)
    b = rf.qk_norm_mrope(y[0], y[1], None, None, *cs, (at % 20).view(1, n).expand(3, n), [12, 10, 10], mixed=True)
    assert all(torch.equal(p, r) for p, r in zip(a, b))


def test_a_cache_past_4_gib():
    """The same tokens in the last blocks of a large cache and in a small one."""
    hk, d, bs = 8, 256, 128
    large, small = rf.KV4Cache(36000, hk, d, bs), rf.KV4Cache(12, hk, d, bs)
    assert large.k.numel() > 2 ** 32
    g = _rng(7)
    ids = torch.randperm(12, generator=g)
    n = 12 * bs - 7
    k, v = (torch.randn(n, hk, d, generator=g).half().to(DEV) for _ in range(2))
    at = torch.arange(n)
    outs = []
    for cache, base in ((small, 0), (large, 36000 - 12)):
        blocks = ids + base
        slots = (blocks[at // bs] * bs + at % bs).int().to(DEV)
        cache.append(k, v, slots)
        table = blocks.int()[None].to(DEV)
        res = list(cache.read(slots)) + list(cache.read(slots[::3].contiguous()))
        for rows in (1, 9, 200):
            q = torch.randn(rows, 2 * hk, d, generator=_rng(rows)).half().to(DEV)
            res += cache.attention(q, table, _i32([n]), return_lse=True)
        outs.append(res)
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    assert not large.k[:36000 - 12].any() and not large.v[:36000 - 12].any()


# ---- streams, threads, captured steps ------------------------------------------------------

BATCHES = {
    "one long": ([15000], 1), "drafted tokens": ([9000], 4), "ragged": ([900, 30, 4000, 2500], 1),
    "many": ([100, 300] * 40, 1), "prompts": ([0, 500, 40], 150), "several rows": ([60, 2000], 9),
}


def _state(name, seed):
    lens, n = BATCHES[name]
    hk, hq, d, bs = 2, 8, 128, 64
    g = _rng(seed)
    nb = sum(-(-(x + n) // bs) for x in lens) + 1
    lens = [max(x - int(r), 0) + n for x, r in zip(lens, torch.randint(0, 60, (len(lens),), generator=g))]
    width = max(-(-(x + n) // bs) for x in BATCHES[name][0])
    table = _table(lens, bs, nb, g, width)
    t = n * len(lens)
    at = torch.cat([torch.arange(x - n, x) for x in lens])
    rows = torch.arange(len(lens)).repeat_interleave(n)
    q, k, v = (torch.randn(t, h, d, generator=g).half().to(DEV) for h in (hq, hk, hk))
    return dict(cache=_cache(_filled(nb, hk, bs, d, seed), _filled(nb, hk, bs, d, seed + 1)), q=q, k=k, v=v,
                table=table.to(DEV), lens=_i32(lens), cu=_i32(range(0, t + 1, n)), most=n,
                slots=(table[rows, at // bs] * bs + at % bs).int().to(DEV))


def _step(s):
    s["cache"].append(s["k"], s["v"], s["slots"])
    return s["cache"].attention(s["q"], s["table"], s["lens"], s["cu"], max_q_len=s["most"],
                                return_lse=True) + s["cache"].read(s["slots"])


@pytest.mark.parametrize("name", sorted(BATCHES))
def test_a_captured_step_replays_with_new_inputs(name):
    _say("graph", name)
    s = _state(name, 60)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(s)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(s)
    for rep in range(4):
        e = _state(name, 70 + rep)
        for key, x in s.items():
            if torch.is_tensor(x):
                x.copy_(e[key])
        for x, y in zip(s["cache"].tensors(), e["cache"].tensors()):
            x.copy_(y)
        graph.replay()
        ref = _step(e)
        torch.cuda.synchronize()
        for a, b in zip(out, ref):
            assert torch.equal(a, b), rep


def test_two_captured_steps_share_a_stream_and_its_scratch():
    """Graphs of two batches, replayed by turns on one stream, then on two, joined by events."""
    states = [_state("one long", 80), _state("ragged", 81)]
    want = [[x.clone() for x in _step(s)] for s in states]
    graphs, outs = [], []
    for s in states:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(_step(s))
    for _ in range(4):
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for out, ref in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(out, ref))
            for x in out:
                x.zero_()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(4):
        with torch.cuda.stream(a):
            graphs[0].replay()
        b.wait_stream(a)
        with torch.cuda.stream(b):
            graphs[1].replay()
        a.wait_stream(b)
    torch.cuda.synchronize()
    for out, ref in zip(outs, want):
        assert all(torch.equal(x, y) for x, y in zip(out, ref))


@pytest.mark.parametrize("threads", [False, True])
def test_calls_on_two_streams_at_once(threads):
    names = ["one long", "ragged"]
    states = [_state(n, 90) for n in names]
    want = [[x.clone() for x in _step(s)] for s in states]
    streams = [torch.cuda.Stream() for _ in names]
    torch.cuda.synchronize()
    got = [[], []]

    def run(i, turns):
        with torch.cuda.stream(streams[i]):
            for _ in range(turns):
                got[i].append(_step(states[i]))

    if threads:
        workers = [threading.Thread(target=run, args=(i, 20)) for i in range(2)]
        for w in workers:
            w.start()
        for w in workers:
            w.join()
    else:
        for _ in range(20):
            run(0, 1)
            run(1, 1)
    torch.cuda.synchronize()
    for outs, ref in zip(got, want):
        assert len(outs) == 20
        assert all(torch.equal(x, y) for out in outs for x, y in zip(out, ref))


# ---- together --------------------------------------------------------------------------------

@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", [(8, 2, 128), (6, 6, 64), (4, 1, 256)])
def test_the_attention_side_of_a_layer(heads, dt):
    """Prompts with pictures, then single tokens: rotation by three axes, plan, append,
    attention and read, each step's output against the oracle's from the same inputs."""
    _say("layer", heads, dt)
    hq, hk, d = heads
    bs, g = 32, _rng(d)
    lens = [37, 130, 1]
    sections = {64: [12, 10, 10], 128: [24, 20, 20], 256: [48, 40, 40]}[d]
    cos, sin = rf.rope_table(1e4 ** (-torch.arange(d // 2, device=DEV) / (d / 2)), 400)
    wq, wk = (torch.randn(d, generator=g).to(dt).to(DEV) for _ in range(2))
    cache = rf.KV4Cache(12, hk, d, bs)
    table = torch.full((3, 6), -1, dtype=torch.int32, device=DEV)
    cached, start = torch.zeros(3, dtype=torch.int32, device=DEV), _i32([0])
    free = torch.randperm(12, generator=g).int().to(DEV)
    held = [[] for _ in lens]          # each request's keys and values, as held
    total = [0] * len(lens)
    for news in (lens, [1, 1, 1], [3, 0, 2]):
        t = sum(news)
        q, k, v = (torch.randn(t, h, d, generator=g).to(dt).to(DEV) for h in (hq, hk, hk))
        plan = rf.kv8_plan(table, cached, _i32(news), free, start, t, bs)
        at = plan.positions.long()
        positions = torch.stack((at, at // 7, at % 7))
        q, k = rf.qk_norm_mrope(q, k, wq, wk, cos, sin, positions, sections, mixed=True)
        cache.append(k, v, plan.slots)
        out, lse = cache.attention(q, table, plan.kv_lens, plan.cu_new, max_q_len=max(news), return_lse=True)
        back = cache.read(plan.slots, torch.float32)
        offsets = np.concatenate(([0], np.cumsum(news)))
        kq, vq = o.quantize(_np(k)), o.quantize(_np(v))
        kr, vr = o.values(*kq), o.values(*vq)
        assert np.array_equal(_np(back[0]), kr) and np.array_equal(_np(back[1]), vr)
        mag = (np.abs(kq[0] - 8.0) + np.abs(kq[2] - 8.0)[..., None]) * kq[1][..., None]
        for r in range(len(lens)):
            part = slice(offsets[r], offsets[r + 1])
            held[r].append((kr[part], vr[part], mag[part], vq[1][part]))
            total[r] += news[r]
            if news[r] == 0:
                continue
            keys, vals, mags, steps = (np.concatenate(x) for x in zip(*held[r]))
            x = _np(q)[part].reshape(news[r], hk, hq // hk, d)
            s = np.einsum("qhgd,jhd->qhgj", x, keys) * d ** -0.5
            size = np.einsum("qhgd,jhd->qhgj", np.abs(x), mags).max(-1) * d ** -0.5
            seen = np.arange(total[r])[None] <= total[r] - news[r] + np.arange(news[r])[:, None]
            s = np.where(seen[:, None, None], s, -np.inf)
            p = np.exp(s - s.max(-1, keepdims=True))
            ref = np.einsum("qhgj,jhd->qhgd", p, vals) / p.sum(-1)[..., None]
            mass = np.einsum("qhgj,jhd->qhgd", p, np.abs(vals)) / p.sum(-1)[..., None]
            ds = (d + 8) * 2.0 ** -24 * size
            tol = (UNIT[dt] * np.abs(ref) + (2.0 ** -11 + 2 * ds[..., None] + 2.0 ** -18) * mass
                   + total[r] * 2.0 ** -32 * (np.abs(vals).max() + 15 * steps.max()) + 2.0 ** -25)
            err = np.abs(_np(out)[part].reshape(ref.shape) - ref)
            assert (err <= tol).all(), (err / tol).max()
        assert plan.kv_lens.tolist() == total
        cached.copy_(plan.kv_lens)
        start.copy_(plan.free_next)
