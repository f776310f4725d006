"""What the attention side of a decoder is timed on: the work between the q/k/v
projections and the o projection of one layer, over a paged cache held in int8
with one fp32 scale for each block of tokens and head.

A case is one call of one of these operators:

* ``rope``    norms of the query and key heads and the position rotation, one pass;
* ``plan``    block tables, slots and positions of a batch from its lengths;
* ``append``  new keys and values quantized into the blocks of the cache, and the
  touched blocks read back as the values they stand for (what a program does that
  hands a prefix on, and here the way to see the updated state);
* ``attend``  attention of the batch's queries over the cache: single tokens,
  a few drafted tokens, ragged prompts behind a cached context.

Head layouts (query heads, key/value heads, head size) are those of the decoders
that ``bench.py`` and ``perf/cases.py`` take their projections from.
"""
from __future__ import annotations

import math

import torch

own = False

LAYOUTS = {
    "16/8/128": (16, 8, 128),   # 0.6B: 2048 and 1024 wide
    "32/8/128": (32, 8, 128),   # 4B, 8B
    "64/8/128": (64, 8, 128),   # 32B: 8192 and 1024 wide
    "28/4/128": (28, 4, 128),   # 7B: 3584 and 512 wide, seven query heads to one
    "8/1/256": (8, 1, 256),     # Gemma decoder: one shared head of 256
    "12/12/64": (12, 12, 64),   # a head for each query head, size 64
}


def _rope(t, heads, dtype="float16", **kw):
    return {"kind": "rope", "t": t, "heads": heads, "dtype": dtype, "norm": True, "rot": 1.0,
            "interleaved": False, **kw}


def _plan(b, new, cached, bs):
    """b requests of up to `new` new tokens (1: one each) behind up to `cached` cached ones."""
    return {"kind": "plan", "b": b, "new": new, "cached": cached, "bs": bs}


def _append(b, new, cached, heads, dtype="float16", bs=64):
    return {"kind": "append", "b": b, "new": new, "cached": cached, "heads": heads, "dtype": dtype,
            "bs": bs}


def _attend(b, new, cached, heads, dtype="float16", bs=64, causal=True, window=0, lse=False,
            ragged=True):
    return {"kind": "attend", "b": b, "new": new, "cached": cached, "heads": heads, "dtype": dtype,
            "bs": bs, "causal": causal, "window": window, "lse": lse, "ragged": ragged}


def listed():
    return [
        # One decode step of 16 sequences: launch latency.
        {"name": "rope_decode_16", **_rope(16, "32/8/128")},
        # A prompt of an odd length through the widest layer: memory rate.
        {"name": "rope_prefill_4001", **_rope(4001, "64/8/128", "bfloat16")},
        # The bookkeeping of a decode step of 64 sequences.
        {"name": "plan_decode_64", **_plan(64, 1, 8000, 64)},
        # The same for 200 prompts of up to 700 tokens, admitted at once.
        {"name": "plan_prefill_200", **_plan(200, 700, 300, 32)},
        # One new token for each of 48 sequences, in the middle of their blocks.
        {"name": "append_decode_48", **_append(48, 1, 500, "64/8/128")},
        # Three prompts of up to 4000 tokens, the first blocks partly filled.
        {"name": "append_prefill_3", **_append(3, 4000, 500, "32/8/128", "bfloat16")},
        # Single-stream decode behind a short context: latency.
        {"name": "attend_decode_1", **_attend(1, 1, 777, "32/8/128", ragged=False)},
        # Single-stream decode behind a very long context, an odd length.
        {"name": "attend_decode_long", **_attend(1, 1, 130999, "32/8/128", ragged=False)},
        # 48 sequences of up to 9000 tokens each decode one token: serving.
        {"name": "attend_decode_48", **_attend(48, 1, 9000, "64/8/128")},
        # A block of 50 queries that see each other and a prefix (no causal
        # order), one shared head of 256, four at a time.
        {"name": "attend_block_50", **_attend(4, 50, 968, "8/1/256", "bfloat16", 32, causal=False,
                                               ragged=False)},
        # Chunks of five prompts of up to 1500 tokens behind cached ones, a
        # window of 2000 tokens, seven query heads to a key head.
        {"name": "attend_chunks_5", **_attend(5, 1500, 6000, "28/4/128", "bfloat16", 64, window=2000,
                                               lse=True)},
        # A prompt of an odd length through the widest layer: the largest.
        {"name": "attend_prefill_7999", **_attend(1, 7999, 0, "64/8/128", ragged=False)},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "plan", "append", "attend", "attend", "attend"])
    heads = rng.choice(sorted(LAYOUTS))
    dtype = rng.choice(["float16", "bfloat16"])
    bs = rng.choice([32, 64, 64, 128])
    if kind == "rope":
        return _rope(_log_int(rng, 1, 8192), heads, dtype, norm=rng.random() < 0.75,
                     rot=rng.choice([1.0, 1.0, 0.5]), interleaved=rng.random() < 0.25)
    if kind == "plan":
        new = 1 if rng.random() < 0.4 else _log_int(rng, 2, 4096)
        return _plan(_log_int(rng, 1, 1024 if new < 256 else 100), new, _log_int(rng, 1, 32000), bs)
    if kind == "append":
        new = 1 if rng.random() < 0.4 else _log_int(rng, 2, 8000)
        return _append(_log_int(rng, 1, max(1, min(256, 16000 // new))), new, _log_int(rng, 1, 2000), heads, dtype, bs)
    form = rng.choice(["decode", "decode", "drafted", "prompt", "prompt"])
    window = rng.choice([0, 0, 0, _log_int(rng, 16, 4096)])
    lse = rng.random() < 0.3
    if form == "prompt":
        new, cached = _log_int(rng, 16, 3800), rng.choice([0, _log_int(rng, 1, 4000)])
        b = rng.randint(1, max(1, min(4, 30_000_000 // (new * (cached + new)))))
        causal = rng.random() < 0.85
        return _attend(b, new, cached, heads, dtype, bs, causal, window if causal else 0, lse,
                       rng.random() < 0.5)
    new = 1 if form == "decode" else rng.randint(2, 9)
    cached = _log_int(rng, 1, 60000)
    b = _log_int(rng, 1, max(1, min(64, 250000 // cached)))
    return _attend(b, new, cached, heads, dtype, bs, True, window, lse, rng.random() < 0.8)


# ---- inputs --------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _head_values(g, *shape):
    """What projections give: N(0, 1) with a few loud channels in each head."""
    x = torch.randn(*shape, generator=g, device="cuda")
    loud = torch.randperm(shape[-1], generator=g, device="cuda")[: max(1, shape[-1] // 64)]
    x[..., loud] *= 6.0
    return x


def _quantize_blocks(x):
    """x [blocks, heads, tokens, D] -> int8 values and one fp32 scale for each block and head."""
    scale = x.abs().amax((2, 3)) * (1.0 / 127.0)
    return torch.round(x / scale[:, :, None, None]).clamp_(-127, 127).to(torch.int8), scale


def _table(g, counts, width, blocks):
    """Block tables [b, width] of counts[i] blocks each, in no order of the cache; -1 past them."""
    ids = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    first = torch.cumsum(counts, 0) - counts
    j = torch.arange(width, device="cuda")[None, :]
    at = first[:, None] + j
    return torch.where(j < counts[:, None], ids[at.clamp(max=blocks - 1)], -1).to(torch.int32).contiguous()


def _lens(c):
    """(cached, new) lengths of the batch: request 0 has the case's, a ragged batch's
    others fall evenly between nothing cached (one new token) and those."""
    part = [(0.3819660113 * i) % 1.0 if i and c.get("ragged", True) else 1.0 for i in range(c["b"])]
    return [int(c["cached"] * f) for f in part], [max(1, int(c["new"] * (1.5 * f % 1.0 if f < 1 else f))) for f in part]


def _lengths(c):
    return [torch.tensor(n, device="cuda", dtype=torch.int32) for n in _lens(c)]


def _state_rope(c, seed):
    g = _gen(seed)
    hq, hk, d = LAYOUTS[c["heads"]]
    dt = getattr(torch, c["dtype"])
    t, rot, table = c["t"], int(d * c["rot"]), 16384
    freq = 1e6 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    angle = torch.arange(table, device="cuda", dtype=torch.float64)[:, None] * freq
    # one run of positions for each of a few requests, as a ragged batch has
    positions = (torch.arange(t, device="cuda") + torch.randint(0, table - t, (1,), generator=g, device="cuda")
                 if t > 64 else torch.randint(0, table, (t,), generator=g, device="cuda"))
    weight = [(1.0 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dt) if c["norm"] else None
              for _ in range(2)]
    return {"case": c, "q": _head_values(g, t, hq, d).to(dt), "k": _head_values(g, t, hk, d).to(dt),
            "q_weight": weight[0], "k_weight": weight[1], "cos": angle.cos().float(),
            "sin": angle.sin().float(), "positions": positions, "eps": 1e-6}


def _state_plan(c, seed):
    g = _gen(seed)
    cached, new = _lengths(c)
    total, bs = int(new.sum()), c["bs"]
    have, want = (cached + bs - 1) // bs, (cached + new + bs - 1) // bs
    width, used, need = int(want.max()), int(have.sum()), int((want - have).sum())
    blocks = used + need + 1000
    ids = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    j = torch.arange(width, device="cuda")[None, :]
    at = (torch.cumsum(have, 0) - have)[:, None] + j
    table = torch.where(j < have[:, None], ids[at.clamp(max=blocks - 1)], -1).to(torch.int32).contiguous()
    return {"case": c, "table": table, "cached": cached, "new": new, "free": ids[used:].contiguous(),
            "start": torch.full((1,), 7, device="cuda", dtype=torch.int32), "total": total}


def _cache_state(g, k, v):
    """The quantized cache: what the plain form reads, or the framework's own."""
    kq, ks = _quantize_blocks(k)
    vq, vs = _quantize_blocks(v)
    if own:
        import rhinoforge_amd as rf
        return {"cache": rf.KV8Cache.from_quantized(kq, ks, vq, vs)}
    return {"kq": kq, "ks": ks, "vq": vq, "vs": vs}


def _state_append(c, seed):
    g = _gen(seed)
    _, hk, d = LAYOUTS[c["heads"]]
    dt, bs = getattr(torch, c["dtype"]), c["bs"]
    cached, new = _lengths(c)
    # Only the block that each request's new tokens begin in is in hand.
    cached = cached % bs
    counts = (cached + new + bs - 1) // bs
    blocks, total = int(counts.sum()) + 5, int(new.sum())
    table = _table(g, counts, int(counts.max()), blocks)

    def slots(lo, n):  # slots of positions lo[i] .. lo[i] + n[i] - 1 of every request
        req = torch.repeat_interleave(torch.arange(len(n), device="cuda"), n.long())
        pos = torch.arange(len(req), device="cuda") - (torch.cumsum(n, 0) - n)[req] + lo[req]
        return (table[req, pos // bs] * bs + pos % bs).to(torch.int32)

    old = [torch.randn(blocks, hk, bs, d, generator=g, device="cuda") for _ in range(2)]
    return {"case": c, **_cache_state(g, *old), "k": _head_values(g, total, hk, d).to(dt),
            "v": _head_values(g, total, hk, d).to(dt), "slots": slots(cached, new),
            "read": slots(torch.zeros_like(cached), cached + new)}


def _state_attend(c, seed):
    g = _gen(seed)
    hq, hk, d = LAYOUTS[c["heads"]]
    dt, bs = getattr(torch, c["dtype"]), c["bs"]
    cached, new = _lengths(c)
    lens = cached + new
    counts = (lens + bs - 1) // bs
    width, blocks, total = int(counts.max()), int(counts.sum()) + 3, int(new.sum())
    cu = torch.zeros(c["b"] + 1, device="cuda", dtype=torch.int32)
    cu[1:] = torch.cumsum(new, 0)
    q = _head_values(g, total, hq, d).to(dt)
    state = _cache_state(g, _head_values(g, blocks, hk, bs, d),
                         torch.randn(blocks, hk, bs, d, generator=g, device="cuda"))
    return {"case": c, **state, "q": q, "table": _table(g, counts, width, blocks), "lens": lens, "cu": cu,
            "scale": d ** -0.5, "max_q": c["new"], "max_kv": c["cached"] + c["new"]}


_STATE = {"rope": _state_rope, "plan": _state_plan, "append": _state_append, "attend": _state_attend}


def prepare(case, seed):
    return _STATE[case["kind"]](case, seed)


# ---- the framework's calls -------------------------------------------------------

def _own_rope(s):
    import rhinoforge_amd as rf
    return rf.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["cos"], s["sin"],
                           s["positions"], eps=s["eps"], interleaved=s["case"]["interleaved"])


def _own_plan(s):
    import rhinoforge_amd as rf
    p = rf.kv8_plan(s["table"], s["cached"], s["new"], s["free"], s["start"], s["total"], s["case"]["bs"])
    return {"table": s["table"], "slots": p.slots, "positions": p.positions, "cu": p.cu_new,
            "lens": p.kv_lens, "free_next": p.free_next}


def _own_append(s):
    import rhinoforge_amd as rf
    rf.kv8_append(s["cache"], s["k"], s["v"], s["slots"])
    return rf.kv8_read(s["cache"], s["read"], s["k"].dtype)


def _own_attend(s):
    import rhinoforge_amd as rf
    c = s["case"]
    return rf.kv8_attention(s["q"], s["cache"], s["table"], s["lens"], s["cu"], max_q_len=s["max_q"],
                            max_kv_len=s["max_kv"], causal=c["causal"], window=c["window"],
                            scale=s["scale"], return_lse=c["lse"])


# ---- the plain forms -------------------------------------------------------------

def _rotated(x, cos, sin, interleaved):
    """x [T, H, D] with its first 2 * cos.size(-1) positions of each head rotated."""
    half = cos.size(-1)
    part, rest = x[..., : 2 * half], x[..., 2 * half:]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :half], part[..., half:])
    a, b = a * cos - b * sin, b * cos + a * sin
    part = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((part, rest), -1)


def _plain_rope(s):
    c = s["case"]
    cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]

    def heads(x, w):
        y = x.float()
        if w is not None:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + s["eps"]) * w.float()
        return _rotated(y, cos, sin, c["interleaved"]).to(x.dtype)

    return heads(s["q"], s["q_weight"]), heads(s["k"], s["k_weight"])


def _plain_plan(s):
    bs, table, cached, new = s["case"]["bs"], s["table"], s["cached"], s["new"]
    lens = cached + new
    have, want = (cached + bs - 1) // bs, (lens + bs - 1) // bs
    need = want - have
    ends = torch.cumsum(need, 0)
    first = s["start"] + ends - need
    j = torch.arange(table.size(1), device="cuda")[None, :]
    at = first[:, None] + j - have[:, None]
    fresh = (j >= have[:, None]) & (j < want[:, None])
    there = at < s["free"].numel()
    ids = torch.where(there, s["free"][at.clamp(0, s["free"].numel() - 1).long()], -1)
    table.copy_(torch.where(fresh, ids, table))
    cu = torch.zeros(new.numel() + 1, device="cuda", dtype=torch.int32)
    cu[1:] = torch.cumsum(new, 0)
    t = torch.arange(s["total"], device="cuda")
    req = torch.searchsorted(cu[1:].long(), t, right=True)
    pos = (t - cu[req] + cached[req]).to(torch.int32)
    block = table[req, (pos // bs).long()]
    slots = torch.where(block < 0, -1, block * bs + pos % bs)
    return {"table": table, "slots": slots, "positions": pos, "cu": cu, "lens": lens,
            "free_next": s["start"] + ends[-1].to(torch.int32)}


def _plain_append_one(x, slots, q, scale):
    """New tokens x [T, H, D] into q [blocks, H, tokens, D] int8 and scale [blocks, H]."""
    bs, heads = q.size(2), q.size(1)
    block, off = (slots // bs).long(), (slots % bs).long()
    x = x.float()
    touched, at = torch.unique(block, return_inverse=True)
    index = at[:, None].expand(-1, heads)
    amax = torch.zeros(touched.numel(), heads, device="cuda").scatter_reduce(
        0, index, x.abs().amax(-1), "amax")
    begin = torch.full((touched.numel(),), bs, device="cuda").scatter_reduce(0, at, off, "amin")
    fresh = torch.where(amax < 2.0 ** -100, 0.0, amax * (1.0 / 127.0))
    before = torch.where((begin > 0)[:, None], scale[touched], 0.0)
    after = torch.maximum(before, fresh)
    ratio = torch.where(after > before, before / after, 1.0)[:, :, None, None]
    kept = torch.arange(bs, device="cuda")[None, :] < begin[:, None]
    old = q[touched]
    q[touched] = torch.where(kept[:, None, :, None], torch.round(old.float() * ratio).to(torch.int8), old)
    scale[touched] = after
    step = after[at][:, :, None]
    q[block, :, off] = torch.where(step > 0, torch.round(x / step).clamp(-127, 127), 0.0).to(torch.int8)


def _plain_append(s):
    _plain_append_one(s["k"], s["slots"], s["kq"], s["ks"])
    _plain_append_one(s["v"], s["slots"], s["vq"], s["vs"])
    bs, dt = s["case"]["bs"], s["k"].dtype
    block, off = (s["read"] // bs).long(), (s["read"] % bs).long()
    return ((s["kq"][block, :, off].float() * s["ks"][block][:, :, None]).to(dt),
            (s["vq"][block, :, off].float() * s["vs"][block][:, :, None]).to(dt))


def _plain_attend(s):
    c = s["case"]
    q, table, lens, cu = s["q"], s["table"].long().clamp(min=0), s["lens"].long(), s["cu"].long()
    hk, bs, d = s["kq"].size(1), s["kq"].size(2), s["kq"].size(3)
    b, width, most, total, hq = table.size(0), table.size(1), s["max_q"], q.size(0), q.size(1)
    group, length = hq // hk, width * bs

    def gathered(x, scale):  # [b, hk, length, d] fp32
        y = x[table].float() * scale[table][..., None, None]
        return y.permute(0, 2, 1, 3, 4).reshape(b, hk, length, d)

    t = torch.arange(total, device="cuda")
    req = torch.searchsorted(cu[1:], t, right=True)
    i = t - cu[req]
    rows = torch.zeros(b, most, hq, d, device="cuda")
    rows[req, i] = q.float()
    rows = rows.reshape(b, most, hk, group, d).permute(0, 2, 3, 1, 4).reshape(b, hk, group * most, d)
    scores = (rows @ gathered(s["kq"], s["ks"]).transpose(-1, -2)).mul_(s["scale"])
    at = torch.arange(length, device="cuda")
    seen = (at < lens[:, None])[:, None, :].expand(b, most, length)
    pos = (lens - (cu[1:] - cu[:-1]))[:, None] + torch.arange(most, device="cuda")
    if c["causal"]:
        seen = seen & (at <= pos[:, :, None])
    if c["window"]:
        seen = seen & (at > pos[:, :, None] - c["window"])
    scores = scores.view(b, hk, group, most, length)
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(top.clamp(min=-3e38)).exp_()
    norm = p.sum(-1, keepdim=True)
    out = p.view(b, hk, group * most, length) @ gathered(s["vq"], s["vs"])
    out = out.view(b, hk, group, most, d) / norm.clamp(min=1e-37)
    out = out.permute(0, 3, 1, 2, 4).reshape(b, most, hq, d)[req, i].to(q.dtype)
    if not c["lse"]:
        return out
    lse = (top + norm.log()).squeeze(-1).permute(0, 3, 1, 2).reshape(b, most, hq)[req, i]
    return out, lse


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"rope": _own_rope, "plan": _own_plan, "append": _own_append, "attend": _own_attend}[kind](state)
    return {"rope": _plain_rope, "plan": _plain_plan, "append": _plain_append, "attend": _plain_attend}[kind](state)


# ---- what a pass cannot do without -----------------------------------------------

def work(case):
    c = case
    if c["kind"] == "rope":
        hq, hk, d = LAYOUTS[c["heads"]]
        n = c["t"] * (hq + hk) * d
        return {"bytes": 2 * 2 * n + c["t"] * (8 + 4 * d * c["rot"]), "flops": (8 if c["norm"] else 3) * n}
    cached, new = _lens(c)
    if c["kind"] == "plan":
        fresh = sum(-(-(a + n) // c["bs"]) - -(-a // c["bs"]) for a, n in zip(cached, new))
        touched = sum((a + n - 1) // c["bs"] - a // c["bs"] + 1 for a, n in zip(cached, new))
        # lengths in, offsets and lengths out; each touched block's entry read, each
        # token's slot and position written; each new block taken and entered.
        return {"bytes": 16 * c["b"] + 8 * sum(new) + 4 * touched + 8 * fresh, "flops": 4 * sum(new)}
    hq, hk, d = LAYOUTS[c["heads"]]
    if c["kind"] == "append":
        back = sum(a % c["bs"] for a in cached) + sum(new)
        # new tokens in, their bytes out; the touched blocks' bytes in, values out
        return {"bytes": 2 * hk * d * (3 * sum(new) + 3 * back), "flops": 2 * hk * d * (3 * sum(new) + back)}
    pairs = tokens = 0.0
    for a, n in zip(cached, new):
        if not c["causal"]:
            pairs, tokens = pairs + n * (a + n), tokens + a + n
            continue
        w = c["window"] or a + n
        # query i of n sees min(a + i + 1, w) tokens
        full = max(0.0, min(n, a + n - w))
        ramp = n - full
        pairs += full * w + ramp * (a + n - full) - ramp * (ramp - 1) / 2
        tokens += min(a + n, w + n - 1)
    return {"bytes": 2 * hk * d * tokens + 4 * hq * d * sum(new), "flops": 4 * hq * d * pairs}


# ---- the definitions in 64 bits --------------------------------------------------

def _exact_rope(s):
    """Pair (x, y) at angle a turns to (x cos a - y sin a, x sin a + y cos a)."""
    c = s["case"]
    outs = []
    for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
        y = x.double()
        if w is not None:
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / y.size(-1) + s["eps"]) * w.double()
        half = s["cos"].size(1)
        turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"]].unsqueeze(1)
        n = torch.arange(half, device="cuda")
        first, second = (2 * n, 2 * n + 1) if c["interleaved"] else (n, n + half)
        z = torch.complex(y[..., first], y[..., second]) * turn
        out = y.clone()
        out[..., first], out[..., second] = z.real, z.imag
        outs.append(out)
    return tuple(outs)


def _exact_append(s):
    """Block by block: the scale is the largest magnitude held, over 127."""
    bs = s["case"]["bs"]
    slots = s["slots"].tolist()
    runs, begin = [], 0
    for n in range(1, len(slots) + 1):
        if n == len(slots) or slots[n] // bs != slots[begin] // bs:
            runs.append((begin, n))
            begin = n
    if len(runs) > 4000:
        return None
    outs = []
    for x, q, scale in ((s["k"], s["kq"].clone(), s["ks"].double()), (s["v"], s["vq"].clone(), s["vs"].double())):
        q = q.double()
        for lo, hi in runs:
            block, off = slots[lo] // bs, slots[lo] % bs
            new = x[lo:hi].double().transpose(0, 1)
            step = new.abs().amax((1, 2)) / 127
            if off:
                step = torch.maximum(step, scale[block])
                q[block, :, :off] = torch.round(q[block, :, :off] * (scale[block] / step)[:, None, None])
            scale[block] = step
            q[block, :, off: off + hi - lo] = torch.round(new / step[:, None, None])
        at = s["read"].long()
        outs.append(q[at // bs, :, at % bs] * scale[at // bs][:, :, None])
    return tuple(outs)


def _exact_attend(s):
    """Request by request and head by head, each over the tokens that its queries see."""
    c = s["case"]
    hk, bs = s["kq"].size(1), s["kq"].size(2)
    group = s["q"].size(1) // hk
    out = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    lse = torch.full(s["q"].shape[:2], -math.inf, device="cuda", dtype=torch.float64)
    cu = s["cu"].tolist()
    for r, length in enumerate(s["lens"].tolist()):
        n = cu[r + 1] - cu[r]
        if not n or not length:
            continue
        blocks = s["table"][r, : (length + bs - 1) // bs].long()
        place = torch.arange(length, device="cuda")
        mine = torch.arange(n, device="cuda")[:, None] + (length - n)
        for h in range(hk):
            k = (s["kq"][blocks, h].double() * s["ks"][blocks, h].double()[:, None, None]).flatten(0, 1)[:length]
            v = (s["vq"][blocks, h].double() * s["vs"][blocks, h].double()[:, None, None]).flatten(0, 1)[:length]
            hidden = torch.zeros(n, length, device="cuda", dtype=torch.bool)
            if c["causal"]:
                hidden |= place > mine
            if c["window"]:
                hidden |= place <= mine - c["window"]
            for j in range(h * group, (h + 1) * group):
                logits = s["q"][cu[r]:cu[r + 1], j].double() @ k.t().contiguous() * s["scale"]
                logits[hidden] = -math.inf
                some = torch.logsumexp(logits, -1)
                lse[cu[r]:cu[r + 1], j] = some
                out[cu[r]:cu[r + 1], j] = torch.exp(logits - some[:, None]).nan_to_num(0.0) @ v
    return (out, lse) if c["lse"] else out


def exact(case, seed):
    if case["kind"] == "plan":
        return None
    state = _STATE[case["kind"]](case, seed)
    return {"rope": _exact_rope, "append": _exact_append, "attend": _exact_attend}[case["kind"]](state)
