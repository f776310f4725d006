"""Ragged batches over the 4-bit cache whose tiles are cut into shares, and calls whose
offsets are not in order (MI355X only): against oracle/kv4.py, to the tolerances of
test_gpu_kv4.py, and to the bit from call to call."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import rhinoforge_amd as rf
from rhinoforge_amd import capi
from test_gpu_kv4 import DEV, _cache, _check, _filled, _rng, _say, _table

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


def _ragged(b, most_new, seed, longest=3000, long=3):
    """Most requests short or empty, a few long; (lens, news)."""
    r = np.random.default_rng(seed)
    lens = r.integers(0, 60, b)
    lens[r.integers(0, b, long)] = r.integers(longest // 2, longest + 1, long)
    news = [1] * b if most_new == 1 else [int(x) for x in r.integers(0, most_new + 1, b)]
    return [int(x) for x in lens], news


# (shares of tiles of 4 and 8 rows, with heads of 64 also of 16, from 130 requests on of 32)
@pytest.mark.parametrize("b", [48, 63, 64, 65, 130, 511])
@pytest.mark.parametrize("hq,hk,d", [(4, 1, 64), (8, 1, 64), (4, 1, 128), (8, 1, 128), (16, 2, 128)])
@pytest.mark.parametrize("new,window", [(1, 0), (1, 2000), (3, 0)])
def test_batches_in_shares(b, hq, hk, d, new, window):
    _say("shares", b, hq, hk, d, new, window)
    lens, news = _ragged(b, new, b * 7 + new)
    nb = sum(-(-n // 64) for n in lens) + 1
    k, v = _filled(nb, hk, 64, d, 60), _filled(nb, hk, 64, d, 61)
    q = torch.randn(sum(news), hq, d, generator=_rng(b)).half()
    table = _table(lens, 64, nb, _rng(b + 1))
    kw = dict(window=window, max_q_len=max(news), max_kv_len=max(lens))
    out, lse = _check(q, k, v, table, lens, news, **kw)
    cache, args = _cache(k, v), (table.to(DEV), _i32(lens), _i32(np.concatenate(([0], np.cumsum(news)))))
    for _ in range(3):
        again = rf.kv4_attention(q.to(DEV), cache, *args, return_lse=True, **kw)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)


# (48 x one query, 64 + 8 heads: fewer shares than the grid has room for tiles; 80 x 12 + 12 and 60 x up to 4: few
# shares for each tile; the others: whole tiles, and splits that the second kernel adds)
@pytest.mark.parametrize("b,hq,hk,d,new", [(48, 64, 8, 128, 1), (80, 12, 12, 64, 1), (60, 64, 8, 128, 4), (130, 12, 12, 64, 1),
                                           (100, 8, 1, 256, 1), (50, 8, 1, 256, 5)])
@pytest.mark.parametrize("window", [0, 700])
def test_batches_of_many_tiles(b, hq, hk, d, new, window):
    _say("many tiles", b, hq, hk, d, new, window)
    lens, news = _ragged(b, new, b, 2500, 6)
    nb = sum(-(-n // 64) for n in lens) + 1
    k, v = _filled(nb, hk, 64, d, 62), _filled(nb, hk, 64, d, 63)
    q = torch.randn(sum(news), hq, d, generator=_rng(b)).bfloat16()
    table = _table(lens, 64, nb, _rng(b + 1))
    kw = dict(window=window, max_q_len=max(news), max_kv_len=max(lens))
    out, lse = _check(q, k, v, table, lens, news, **kw)
    again, lse2 = _check(q, k, v, table, lens, news, **kw)
    assert torch.equal(again, out) and torch.equal(lse2, lse)


@pytest.mark.parametrize("n", [1, 6, 150])
def test_tokens_behind_the_batch_change_nothing(n):
    """Of the same launch the same bits; of another one the same result to its tolerance."""
    k, v = _filled(9, 1, 32, 64, 13), _filled(9, 1, 32, 64, 14)
    q = torch.randn(n + 7, 4, 64, generator=_rng(22)).half()
    table = _table([n + 50], 32, 9, _rng(23))
    want, _ = _check(q[:n], k, v, table, [n + 50], [n], max_q_len=n)
    out, lse = rf.kv4_attention(q.to(DEV), _cache(k, v), table.to(DEV), _i32([n + 50]), _i32([0, n]), max_q_len=n,
                                return_lse=True)
    assert torch.equal(out[:n], want)
    assert (out[n:] == 0).all() and torch.isneginf(lse[n:]).all()


# ---- offsets that are not in order ---------------------------------------------------------

MARGIN = 4096   # bytes on either side of what a call may write


class _Call:
    """A call through the C ABI, whose outputs and partial results lie between margins."""

    def __init__(self, b, new, hq, hk, d, context, max_q):
        bs = 32
        lens = [context] * b
        nb = sum(-(-n // bs) for n in lens)
        self.tokens, self.hq, self.d = b * new, hq, d
        self.cache = _cache(_filled(nb, hk, bs, d, 64), _filled(nb, hk, bs, d, 65))
        self.table, self.lens = _table(lens, bs, nb, _rng(66)).to(DEV), _i32(lens)
        self.q = torch.randn(self.tokens, hq, d, generator=_rng(67)).half().to(DEV)
        self.cu = _i32(np.arange(0, self.tokens + 1, new))
        c = self.cache
        self.args = capi.KV4AttentionArgs(
            cache=capi.KV4Cache(k=c.k.data_ptr(), v=c.v.data_ptr(), rows=c.rows.data_ptr(), num_blocks=c.num_blocks,
                                kv_heads=hk, head_dim=d, block_size=bs),
            q=capi.KV8Heads(data=self.q.data_ptr(), token_stride=hq * d, head_stride=d, heads=hq),
            kv_lens=self.lens.data_ptr(), block_table=self.table.data_ptr(), cu_q=self.cu.data_ptr(), out=self.q.data_ptr(),
            tokens=self.tokens, requests=b, width=self.table.size(1), table_stride=self.table.size(1), max_q_len=max_q,
            max_kv_len=context, dtype=0, causal=1, window=0, scale=0.1)
        self.need = capi.load().rf_kv4_attention_workspace(ctypes.byref(self.args))
        assert self.need > 0
        sizes = dict(out=self.q.numel() * 2, lse=self.tokens * hq * 4, part=self.need, counters=capi.WS_COUNTER_BYTES)
        self.held = {k: torch.full((n + 2 * MARGIN,), 0xa5, dtype=torch.uint8, device=DEV) for k, n in sizes.items()}
        self.inner("counters").zero_()
        at = lambda k: self.inner(k).data_ptr()  # noqa: E731
        self.scratch = capi.Scratch(at("counters"), at("part"), self.need)
        self.args.out, self.args.lse, self.args.scratch = at("out"), at("lse"), ctypes.pointer(self.scratch)

    def inner(self, name):
        return self.held[name][MARGIN:-MARGIN]

    def run(self, cu):
        """(out, lse) of a call with these offsets; the margins and the counters are as they were."""
        self.args.cu_q = cu.data_ptr()
        st = capi.load().rf_kv4_attention(ctypes.byref(self.args), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        assert st == capi.OK
        for name, x in self.held.items():
            assert (x[:MARGIN] == 0xa5).all() and (x[-MARGIN:] == 0xa5).all(), name
        assert not self.inner("counters").any()
        return self.inner("out").clone(), self.inner("lse").clone()


# requests, queries, heads, kv_heads, head_dim, context, max_q_len
CALLS = [(40, 1, 8, 1, 128, 2000, 1), (3, 1, 8, 2, 128, 9000, 1), (48, 4, 64, 8, 128, 2000, 4), (70, 1, 4, 1, 64, 1500, 0),  # shares
         (1, 1, 8, 2, 128, 9000, 0), (1, 1, 4, 1, 256, 20000, 0),                           # splits joined in the launch
         (40, 9, 4, 2, 64, 2000, 9), (1, 3, 4, 1, 128, 20000, 0), (2, 20, 16, 1, 128, 6000, 0),   # by the second kernel
         (1, 300, 16, 2, 128, 6300, 0)]                                                     # of a prompt


@pytest.mark.parametrize("call", CALLS, ids=str)
def test_offsets_that_are_not_in_order(call):
    """What they give is not said, but they stay inside and leave the next call right."""
    _say("offsets", call)
    c = _Call(*call)
    good = c.cu
    want = c.run(good)
    b, t = call[0], c.tokens
    bad = [good.flip(0), torch.full_like(good, t), torch.zeros_like(good), good - t // 2, good * 2, good.roll(1)]
    up = good.clone()
    up[1:b:2] = t
    far = good.clone()
    far[::2], far[1::2] = -2 ** 31, 2 ** 31 - 1
    for cu in (*bad, up, far):
        c.run(cu.contiguous())
        got = c.run(good)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
