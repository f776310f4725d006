"""The scratch of the int8 cache's attention behind the torch op: what it holds as
calls need more and more (MI355X only)."""
from __future__ import annotations

import ctypes

import pytest
import torch

import rhinoforge_amd as rf
from rhinoforge_amd import capi
from conftest import fresh_hip_stream

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _need(q, cache, table, lens, cu, new):
    """Bytes of partial results of one call, as the C ABI states them."""
    hq, d = q.shape[1:]
    a = capi.KV8AttentionArgs(
        cache=capi.KV8Cache(k=cache.k.data_ptr(), v=cache.v.data_ptr(), k_scale=cache.k_scale.data_ptr(),
                            v_scale=cache.v_scale.data_ptr(), num_blocks=cache.num_blocks,
                            kv_heads=cache.kv_heads, head_dim=d, block_size=cache.block_size),
        q=capi.KV8Heads(data=q.data_ptr(), token_stride=hq * d, head_stride=d, heads=hq),
        cu_q=cu.data_ptr(), kv_lens=lens.data_ptr(), block_table=table.data_ptr(), out=q.data_ptr(), lse=None,
        scratch=None, tokens=q.size(0), requests=1, width=table.size(1), table_stride=table.size(1),
        max_q_len=new, max_kv_len=0, dtype=0, causal=1, window=0, scale=0.1)
    return capi.load().rf_kv8_attention_workspace(ctypes.byref(a))


def test_partials_that_grow_hold_a_bounded_multiple():
    """Chunks of 90 to 200 tokens, each a little longer than the one before: buffers
    that a captured graph may still use are kept, so the next one is at least twice
    the last, and all together stay below four times the largest need."""
    hq, hk, d, n = 64, 4, 256, 1500
    cache = rf.KV8Cache(48, hk, d, 32)
    kv = torch.randn(n, hk, d, generator=torch.Generator().manual_seed(0)).half().to(DEV)
    cache.append(kv, kv.flip(0), torch.arange(n, dtype=torch.int32, device=DEV))
    table = torch.arange(48, dtype=torch.int32, device=DEV)[None]
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    most, outs = 0, []
    news = list(range(90, 201, 2))
    qs = torch.randn(max(news), hq, d, generator=torch.Generator().manual_seed(1)).half().to(DEV)
    cus = [torch.tensor([0, new], dtype=torch.int32, device=DEV) for new in news]
    with fresh_hip_stream() as stream:
        stream.wait_stream(torch.cuda.current_stream())
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        with torch.cuda.stream(stream):
            for new, cu in zip(news, cus):
                most = max(most, _need(qs[:new], cache, table, lens, cu, new))
                out = rf.kv8_attention(qs[:new], cache, table, lens, cu, max_q_len=new, scale=0.1)
            outs.append(out.clone())
            del out
        torch.cuda.synchronize()
        held = torch.cuda.memory_allocated() - before - sum(x.numel() * x.element_size() for x in outs)
    print(f"largest need {most / 2 ** 20:.1f} MB, held {held / 2 ** 20:.1f} MB", flush=True)
    assert most > 32 << 20   # (past the least size, more than once)
    assert held <= 4 * most
    again = rf.kv8_attention(qs[:news[-1]], cache, table, lens, cus[-1], max_q_len=news[-1], scale=0.1)
    assert torch.equal(again, outs[0])


def test_partials_that_cannot_double_grow_to_the_need():
    """A cache that leaves little memory: 32 MB of partials, then 39 MB where 64 do not fit."""
    hq, hk, d, n = 64, 4, 256, 1500
    cache = rf.KV8Cache(48, hk, d, 32)
    kv = torch.randn(n, hk, d, generator=torch.Generator().manual_seed(0)).half().to(DEV)
    cache.append(kv, kv.flip(0), torch.arange(n, dtype=torch.int32, device=DEV))
    table = torch.arange(48, dtype=torch.int32, device=DEV)[None]
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    q = torch.randn(200, hq, d, generator=torch.Generator().manual_seed(1)).half().to(DEV)
    args = {new: (q[:new], cache, table, lens, torch.tensor([0, new], dtype=torch.int32, device=DEV))
            for new in (140, 200)}
    want = rf.kv8_attention(*args[200], max_q_len=200)
    total = torch.cuda.get_device_properties(0).total_memory
    with fresh_hip_stream() as stream:
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            rf.kv8_attention(*args[140], max_q_len=140)
            torch.cuda.synchronize()
            torch.cuda.empty_cache()
            torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (62 << 20)) / total)
            try:
                got = rf.kv8_attention(*args[200], max_q_len=200)
            finally:
                torch.cuda.set_per_process_memory_fraction(1.0)
        torch.cuda.synchronize()
    assert torch.equal(got, want)
