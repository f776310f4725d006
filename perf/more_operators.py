"""What the attention side of a vision-language decoder over a 4-bit paged cache is
timed on.

A case is one call of one of these operators:

* ``rope``    norms of the query and key heads and the rotation by positions of
              several axes (time, height, width), one pass;
* ``append``  new keys and values quantized to 4 bits into the blocks of the cache,
              and the touched blocks read back as the values they stand for (what a
              program does that hands a prefix on, and here the way to see the
              updated state);
* ``read``    cached tokens as the values they stand for;
* ``attend``  attention of a ragged batch's queries over the cache: single tokens,
              a few drafted tokens, prompts behind a cached context.

In the cache every token has, for each key/value head and for keys and values
apart, ``head_dim`` whole numbers n of 0..15, a step s and a zero point z of 0..15:
it holds the values ``(n - z) * s``.  Steps are fp16 numbers of seven significant
bits (the last four of the mantissa are 0), so all of these values are fp16 numbers.

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
TABLE = 16384                   # positions of the rotation's tables


def _rope(t, heads, dtype="float16", **kw):
    """axes: 3 (time, height, width) or 2 (height, width); mixed: the axes' pairs in turn."""
    return {"kind": "rope", "t": t, "heads": heads, "dtype": dtype, "axes": 3, "mixed": True, "norm": True,
            "rot": 1.0, "interleaved": False, **kw}


def _append(b, new, cached, heads, dtype="float16", bs=64):
    """b requests of up to `new` new tokens (1: one each) behind up to `cached` cached ones."""
    return {"kind": "append", "b": b, "new": new, "cached": cached, "heads": heads, "dtype": dtype, "bs": bs}


def _read(n, heads, dtype="float16", bs=64, scattered=False):
    return {"kind": "read", "n": n, "heads": heads, "dtype": dtype, "bs": bs, "scattered": scattered}


def _attend(b, new, cached, heads, dtype="float16", bs=64, causal=True, window=0, lse=False, ragged=True):
    return {"kind": "attend", "b": b, "new": new, "cached": cached, "heads": heads, "dtype": dtype,
            "bs": bs, "causal": causal, "window": window, "lse": lse, "ragged": ragged}


def listed():
    return [
        # One decode step of 16 sequences: launch latency.
        {"name": "rope_decode_16", **_rope(16, "32/8/128")},
        # Two images and their text, an odd number of tokens, through the widest layer.
        {"name": "rope_images_5003", **_rope(5003, "64/8/128", "bfloat16")},
        # The same through a layer without norms, whose axes are runs of pairs.
        {"name": "rope_images_2301", **_rope(2301, "28/4/128", "bfloat16", mixed=False, norm=False)},
        # One new token for each of 48 sequences, in the middle of their blocks.
        {"name": "append_decode_48", **_append(48, 1, 500, "64/8/128")},
        # Three prompts of up to 4000 tokens, the first blocks partly filled.
        {"name": "append_prefill_3", **_append(3, 4000, 500, "32/8/128", "bfloat16")},
        # A prefix of an odd length, handed to another sequence.
        {"name": "read_prefix_9001", **_read(9001, "32/8/128")},
        # A few hundred tokens from anywhere in the cache.
        {"name": "read_tokens_333", **_read(333, "28/4/128", "float32", scattered=True)},
        # Single-stream decode behind a short context: latency.
        {"name": "attend_decode_1", **_attend(1, 1, 777, "32/8/128", ragged=False)},
        # Single-stream decode behind a very long context, an odd length.
        {"name": "attend_decode_long", **_attend(1, 1, 130999, "32/8/128", ragged=False)},
        # 48 sequences of up to 9000 tokens each decode one token: serving.
        {"name": "attend_decode_48", **_attend(48, 1, 9000, "64/8/128")},
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
    kind = rng.choice(["rope", "append", "read", "attend", "attend", "attend"])
    heads = rng.choice(sorted(LAYOUTS))
    dtype = rng.choice(["float16", "bfloat16"])
    bs = rng.choice([32, 64, 64, 128])
    if kind == "rope":
        return _rope(_log_int(rng, 1, 8192), heads, dtype, axes=rng.choice([2, 3, 3]), mixed=rng.random() < 0.5,
                     norm=rng.random() < 0.75, rot=rng.choice([1.0, 1.0, 0.5]), interleaved=rng.random() < 0.25)
    if kind == "append":
        new = 1 if rng.random() < 0.4 else _log_int(rng, 2, 8000)
        return _append(_log_int(rng, 1, max(1, min(256, 16000 // new))), new, _log_int(rng, 1, 2000), heads, dtype, bs)
    if kind == "read":
        return _read(_log_int(rng, 1, 20000), heads, rng.choice(["float16", "bfloat16", "float32"]), bs,
                     rng.random() < 0.5)
    form = rng.choice(["decode", "decode", "drafted", "prompt", "prompt"])
    window = rng.choice([0, 0, 0, _log_int(rng, 16, 4096)])
    lse = rng.random() < 0.3
    if form == "prompt":
        new, cached = _log_int(rng, 16, 3800), rng.choice([0, _log_int(rng, 1, 4000)])
        b = rng.randint(1, max(1, min(4, 30_000_000 // (new * (cached + new)))))
        causal = rng.random() < 0.85
        return _attend(b, new, cached, heads, dtype, bs, causal, window if causal else 0, lse, rng.random() < 0.5)
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
    x[..., loud] *= 3.0
    return x


def _step_and_zero(x):
    """The step of each row of x [..., D] fp32, the least of seven bits with 15 steps
    to the row's span (0 is in the span), and the number that stands for 0."""
    low = x.amin(-1).clamp(max=0.0)
    span = x.amax(-1).clamp(min=0.0) - low
    least = (span * (1.0 / 15.0)).clamp(2.0 ** -20, 4352.0)
    power = (least.view(torch.int32) & 0x7f800000).view(torch.float32)   # of 2, at or below
    ulp = (power * 2.0 ** -6).clamp(min=2.0 ** -20)
    step = torch.floor(least / ulp) * ulp
    step = torch.where(15.0 * step < span, step + ulp, step).clamp(max=4352.0)
    return step, torch.round(-low / step).clamp(max=15.0)


def _quantize(x):
    """x [..., D] -> whole numbers (uint8), steps (fp16) and zero points (uint8) [...]."""
    step, zero = _step_and_zero(x)
    n = (torch.round(x / step[..., None]) + zero[..., None]).clamp_(0.0, 15.0)
    return n.to(torch.uint8), step.half(), zero.to(torch.uint8)


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


def _sections(c):
    """Pairs of each axis."""
    pairs = int(LAYOUTS[c["heads"]][2] * c["rot"]) // 2
    if c["axes"] == 2:
        return [pairs // 2, pairs - pairs // 2]
    side = 5 * pairs // 16 if c["mixed"] else 3 * pairs // 8
    return [pairs - 2 * side, side, side]


def _grid_positions(g, t, axes):
    """Positions [axes, t] of text, images and text again: a text token counts on along
    every axis, an image's patches have one time and their row and column."""
    start = int(torch.randint(0, TABLE // 2 - t // 2, (1,), generator=g, device="cuda"))
    runs, at, left = [], start, t
    while left > 0:
        words = min(left, 1 + left // 20)
        run = torch.arange(words, device="cuda") + at
        runs.append(run.expand(3, -1))
        at, left = at + words, left - words
        side = math.isqrt(max(0, left // 2))
        if side > 1:
            i = torch.arange(side * side, device="cuda")
            runs.append(torch.stack((torch.full_like(i, at), at + i // side, at + i % side)))
            at, left = at + side, left - side * side
    return torch.cat(runs, 1)[3 - axes:].contiguous()


def _state_rope(c, seed):
    g = _gen(seed)
    hq, hk, d = LAYOUTS[c["heads"]]
    dt, t, rot = getattr(torch, c["dtype"]), c["t"], int(d * c["rot"])
    freq = 1e6 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    angle = torch.arange(TABLE, device="cuda", dtype=torch.float64)[:, None] * freq
    positions = (_grid_positions(g, t, c["axes"]) if t > 64
                 else torch.randint(0, TABLE, (c["axes"], t), generator=g, device="cuda"))
    weight = [(1.0 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dt) if c["norm"] else None
              for _ in range(2)]
    return {"case": c, "q": _head_values(g, t, hq, d).to(dt), "k": _head_values(g, t, hk, d).to(dt),
            "q_weight": weight[0], "k_weight": weight[1], "cos": angle.cos().float(),
            "sin": angle.sin().float(), "positions": positions, "sections": _sections(c), "eps": 1e-6}


def _cache_state(k, v):
    """The quantized cache [blocks, heads, tokens, D]: what the plain form reads, or the framework's own."""
    k, v = _quantize(k), _quantize(v)
    if own:
        import rhinoforge_amd as rf
        return {"cache": rf.KV4Cache.from_quantized(*k, *v)}
    return {"k4": k, "v4": v}


def _slots(table, bs, lo, n):
    """Slots of positions lo[i] .. lo[i] + n[i] - 1 of every request."""
    req = torch.repeat_interleave(torch.arange(len(n), device="cuda"), n.long())
    pos = torch.arange(len(req), device="cuda") - (torch.cumsum(n, 0) - n)[req] + lo[req]
    return (table[req, pos // bs] * bs + pos % bs).to(torch.int32)


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
    old = [torch.randn(blocks, hk, bs, d, generator=g, device="cuda") for _ in range(2)]
    return {"case": c, **_cache_state(*old), "k": _head_values(g, total, hk, d).to(dt),
            "v": _head_values(g, total, hk, d).to(dt), "slots": _slots(table, bs, cached, new),
            "read": _slots(table, bs, torch.zeros_like(cached), cached + new)}


def _state_read(c, seed):
    g = _gen(seed)
    _, hk, d = LAYOUTS[c["heads"]]
    n, bs = c["n"], c["bs"]
    blocks = (n + bs - 1) // bs + 7
    held = [_head_values(g, blocks, hk, bs, d) for _ in range(2)]
    if c["scattered"]:
        slots = torch.randint(0, blocks * bs, (n,), generator=g, device="cuda", dtype=torch.int32)
    else:
        ids = torch.randperm(blocks, generator=g, device="cuda")
        i = torch.arange(n, device="cuda")
        slots = (ids[i // bs] * bs + i % bs).to(torch.int32)
    return {"case": c, **_cache_state(*held), "read": slots}


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
    state = _cache_state(_head_values(g, blocks, hk, bs, d),
                         torch.randn(blocks, hk, bs, d, generator=g, device="cuda"))
    return {"case": c, **state, "q": q, "table": _table(g, counts, width, blocks), "lens": lens, "cu": cu,
            "scale": d ** -0.5, "max_q": c["new"], "max_kv": c["cached"] + c["new"]}


_STATE = {"rope": _state_rope, "append": _state_append, "read": _state_read, "attend": _state_attend}


def prepare(case, seed):
    return _STATE[case["kind"]](case, seed)


# ---- the framework's calls -------------------------------------------------------

def _own_rope(s):
    import rhinoforge_amd as rf
    c = s["case"]
    return rf.qk_norm_mrope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["cos"], s["sin"], s["positions"],
                            s["sections"], mixed=c["mixed"], eps=s["eps"], interleaved=c["interleaved"])


def _own_append(s):
    import rhinoforge_amd as rf
    rf.kv4_append(s["cache"], s["k"], s["v"], s["slots"])
    return rf.kv4_read(s["cache"], s["read"], s["k"].dtype)


def _own_read(s):
    import rhinoforge_amd as rf
    return rf.kv4_read(s["cache"], s["read"], getattr(torch, s["case"]["dtype"]))


def _own_attend(s):
    import rhinoforge_amd as rf
    c = s["case"]
    return rf.kv4_attention(s["q"], s["cache"], s["table"], s["lens"], s["cu"], max_q_len=s["max_q"],
                            max_kv_len=s["max_kv"], causal=c["causal"], window=c["window"],
                            scale=s["scale"], return_lse=c["lse"])


# ---- the plain forms -------------------------------------------------------------

def _axis_of_pair(c, sections):
    """Which axis' position turns each pair: runs of pairs, or the axes in turn while
    an axis has pairs left and the first one after that."""
    axes = len(sections)
    if not c["mixed"]:
        return torch.repeat_interleave(torch.arange(axes), torch.tensor(sections)).cuda()
    i = torch.arange(sum(sections), device="cuda")
    upto = torch.tensor(sections, device="cuda") * axes
    return torch.where(i < upto[i % axes], i % axes, 0)


def _rotated(x, cos, sin, interleaved):
    """x [T, H, D] with its first 2 * cos.size(-1) dimensions of each head rotated."""
    half = cos.size(-1)
    part, rest = x[..., : 2 * half], x[..., 2 * half:]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :half], part[..., half:])
    a, b = a * cos - b * sin, b * cos + a * sin
    part = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((part, rest), -1)


def _plain_rope(s):
    c = s["case"]
    row = s["positions"][_axis_of_pair(c, s["sections"])].t()        # [tokens, pairs]
    pair = torch.arange(row.size(1), device="cuda")
    cos, sin = s["cos"][row, pair][:, None], s["sin"][row, pair][:, None]

    def heads(x, w):
        y = x.float()
        if w is not None:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + s["eps"]) * w.float()
        return _rotated(y, cos, sin, c["interleaved"]).to(x.dtype)

    return heads(s["q"], s["q_weight"]), heads(s["k"], s["k_weight"])


def _values(side, block, off):
    """fp32 values [n, heads, D] of tokens off[i] of blocks block[i]."""
    n, step, zero = side
    return (n[block, :, off].float() - zero[block, :, off].float()[..., None]) * step[block, :, off].float()[..., None]


def _plain_read(s, dtype=None):
    bs, dtype = s["case"]["bs"], dtype or getattr(torch, s["case"]["dtype"])
    block, off = (s["read"] // bs).long(), (s["read"] % bs).long()
    return _values(s["k4"], block, off).to(dtype), _values(s["v4"], block, off).to(dtype)


def _plain_append(s):
    bs = s["case"]["bs"]
    block, off = (s["slots"] // bs).long(), (s["slots"] % bs).long()
    for x, side in ((s["k"], s["k4"]), (s["v"], s["v4"])):
        for held, new in zip(side, _quantize(x.float())):
            held[block, :, off] = new
    return _plain_read(s, s["k"].dtype)


def _plain_attend(s):
    c = s["case"]
    q, table, lens, cu = s["q"], s["table"].long().clamp(min=0), s["lens"].long(), s["cu"].long()
    _, hk, bs, d = s["k4"][0].shape
    b, width, most, total, hq = table.size(0), table.size(1), s["max_q"], q.size(0), q.size(1)
    group, length = hq // hk, width * bs

    def gathered(side):  # [b, hk, length, d] fp32
        n, step, zero = (x[table] for x in side)
        y = (n.float() - zero.float()[..., None]) * step.float()[..., None]
        return y.permute(0, 2, 1, 3, 4).reshape(b, hk, length, d)

    t = torch.arange(total, device="cuda")
    req = torch.searchsorted(cu[1:], t, right=True)
    i = t - cu[req]
    rows = torch.zeros(b, most, hq, d, device="cuda")
    rows[req, i] = q.float()
    rows = rows.reshape(b, most, hk, group, d).permute(0, 2, 3, 1, 4).reshape(b, hk, group * most, d)
    scores = (rows @ gathered(s["k4"]).transpose(-1, -2)).mul_(s["scale"])
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
    out = p.view(b, hk, group * most, length) @ gathered(s["v4"])
    out = out.view(b, hk, group, most, d) / norm.clamp(min=1e-37)
    out = out.permute(0, 3, 1, 2, 4).reshape(b, most, hq, d)[req, i].to(q.dtype)
    if not c["lse"]:
        return out
    lse = (top + norm.log()).squeeze(-1).permute(0, 3, 1, 2).reshape(b, most, hq)[req, i]
    return out, lse


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"rope": _own_rope, "append": _own_append, "read": _own_read, "attend": _own_attend}[kind](state)
    return {"rope": _plain_rope, "append": _plain_append, "read": _plain_read, "attend": _plain_attend}[kind](state)


# ---- what a pass cannot do without -----------------------------------------------

def work(case):
    c = case
    hq, hk, d = LAYOUTS[c["heads"]]
    held = 2 * hk * (d // 2 + 2)  # a token's keys and values: numbers, and 11 + 4 bits of step and zero point
    if c["kind"] == "rope":
        n = c["t"] * (hq + hk) * d
        return {"bytes": 2 * 2 * n + c["t"] * (8 * c["axes"] + 4 * d * c["rot"]), "flops": (8 if c["norm"] else 3) * n}
    if c["kind"] == "read":
        size = 4 if c["dtype"] == "float32" else 2
        return {"bytes": c["n"] * (4 + held + 2 * hk * d * size), "flops": 4 * c["n"] * hk * d}
    cached, new = _lens(c)
    if c["kind"] == "append":
        back = sum(a % c["bs"] for a in cached) + sum(new)
        # new tokens in, their numbers out; the touched blocks' numbers in, values out
        return {"bytes": sum(new) * (4 * hk * d + held) + back * (held + 4 * hk * d),
                "flops": 2 * hk * d * (5 * sum(new) + 2 * back)}
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
    return {"bytes": held * tokens + 4 * hq * d * sum(new), "flops": 4 * hq * d * pairs}


# ---- the definitions in 64 bits --------------------------------------------------

def _exact_rope(s):
    """Pair (x, y) at angle a turns to (x cos a - y sin a, x sin a + y cos a)."""
    c = s["case"]
    half = s["cos"].size(1)
    axis, ends = [], [sum(s["sections"][: n + 1]) for n in range(c["axes"])]
    for n in range(half):
        if c["mixed"]:
            a = n % c["axes"]
            axis.append(a if n // c["axes"] < s["sections"][a] else 0)
        else:
            axis.append(next(a for a, end in enumerate(ends) if n < end))
    turns = torch.complex(s["cos"].double(), s["sin"].double())
    turn = torch.stack([turns[s["positions"][a], n] for n, a in enumerate(axis)], -1).unsqueeze(1)
    outs = []
    for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
        y = x.double()
        if w is not None:
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / y.size(-1) + s["eps"]) * w.double()
        n = torch.arange(half, device="cuda")
        first, second = (2 * n, 2 * n + 1) if c["interleaved"] else (n, n + half)
        z = torch.complex(y[..., first], y[..., second]) * turn
        out = y.clone()
        out[..., first], out[..., second] = z.real, z.imag
        outs.append(out)
    return tuple(outs)


def _exact_held(side):
    n, step, zero = side
    return (n.double() - zero.double().unsqueeze(-1)) * step.double().unsqueeze(-1)


def _exact_append(s):
    """A row's span, in fp32, over 15, up to the next multiple of 2^-6 of its power of two."""
    bs = s["case"]["bs"]
    to, back = s["slots"].long(), s["read"].long()
    outs = []
    for x, side in ((s["k"], s["k4"]), (s["v"], s["v4"])):
        x = x.double()
        zero = torch.zeros((), device="cuda", dtype=torch.float64)
        low = torch.minimum(x.min(-1).values, zero)
        span = (torch.maximum(x.max(-1).values, zero) - low).float().double()
        least = (span / 15).clamp(min=2.0 ** -30)
        unit = (least / torch.frexp(least).mantissa / 128).clamp(min=2.0 ** -20)
        step = (torch.ceil(least / unit) * unit).clamp(2.0 ** -20, 4352)
        down = torch.round(low / step).clamp(min=-15)
        number = (torch.round(x / step.unsqueeze(-1)) - down.unsqueeze(-1)).clamp(0, 15)
        held = _exact_held(side)
        held[to // bs, :, to % bs] = (number + down.unsqueeze(-1)) * step.unsqueeze(-1)
        outs.append(held[back // bs, :, back % bs])
    return tuple(outs)


def _exact_read(s):
    bs, at = s["case"]["bs"], s["read"].long()
    return tuple(_exact_held(side)[at // bs, :, at % bs] for side in (s["k4"], s["v4"]))


def _exact_attend(s):
    """Request by request and head by head, each over the tokens that its queries see."""
    c = s["case"]
    hk, bs = s["k4"][0].size(1), c["bs"]
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
            k, v = (_exact_held([x[blocks, h] for x in s[side]]).flatten(0, 1)[:length] for side in ("k4", "v4"))
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
    global own
    was, own = own, False   # (the definition reads the numbers, whoever runs)
    try:
        state = _STATE[case["kind"]](case, seed)
    finally:
        own = was
    return {"rope": _exact_rope, "append": _exact_append, "read": _exact_read, "attend": _exact_attend}[case["kind"]](state)
