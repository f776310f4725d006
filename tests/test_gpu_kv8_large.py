"""Calls of the int8 paged cache's ops that need more than one launch: HIP takes
fewer than 2^32 threads along x, so fewer than 2^24 workgroups of 256 (MI355X only).
Each is compared, bit for bit, with small calls on its parts."""
from __future__ import annotations

import pytest
import torch

import rhinoforge_amd as rf

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _memory():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


@pytest.mark.parametrize("positions", [None, torch.int32, torch.int64])
def test_norm_rope(positions):
    t, d = 2 ** 25 + 3, 16
    print("rope", positions, flush=True)
    q, k = (torch.randn(t, 1, d, generator=_gen(s), device=DEV, dtype=torch.float16) for s in (0, 1))
    w = torch.rand(d, generator=_gen(2), device=DEV).half()
    rows = t if positions is None else 1000
    cos, sin = (torch.rand(rows, d // 2, generator=_gen(s), device=DEV) for s in (3, 4))
    pos = None if positions is None else torch.randint(0, rows, (t,), generator=_gen(5), device=DEV).to(positions)
    got = rf.qk_norm_rope(q, k, w, None, cos, sin, pos)
    for lo in range(0, t, 2 ** 23):
        part = slice(lo, min(lo + 2 ** 23, t))
        want = rf.qk_norm_rope(q[part], k[part], w, None, cos[part] if pos is None else cos,
                               sin[part] if pos is None else sin, None if pos is None else pos[part])
        assert torch.equal(got[0][part], want[0]) and torch.equal(got[1][part], want[1]), lo


HEADS, D, BS = 4096, 64, 32


def _few(t):
    """Tokens in use among t: the first, the last, and runs around where launches of
    whole parts of 32 or 64 tokens would begin."""
    return [(0, 40), (130990, 131072), (t - 20, t)]


def test_append():
    t = 2 ** 17 + 130
    print("append", flush=True)
    x = [torch.randn(t, 1, D, generator=_gen(s), device=DEV).half().expand(t, HEADS, D) for s in (0, 1)]
    slots = torch.full((t,), -1, dtype=torch.int32, device=DEV)
    at = 7
    for lo, hi in _few(t):
        slots[lo:hi] = torch.arange(at, at + hi - lo, dtype=torch.int32, device=DEV)
        at = (at + hi - lo + BS) // BS * BS + 5
    nb = at // BS + 1
    many, few = rf.KV8Cache(nb, HEADS, D, BS), rf.KV8Cache(nb, HEADS, D, BS)
    many.append(*x, slots)
    for lo, hi in _few(t):
        few.append(x[0][lo:hi], x[1][lo:hi], slots[lo:hi])
    for a, b in zip(many.tensors(), few.tensors()):
        assert torch.equal(a, b)
    assert (many.k_scale > 0).any()


def test_read():
    if torch.cuda.mem_get_info()[0] < 160 << 30:
        pytest.skip("needs 160 GB")
    t = 2 ** 17 + 130
    print("read", flush=True)
    cache = rf.KV8Cache(4, HEADS, D, BS)
    kv = torch.randn(4 * BS, HEADS, D, generator=_gen(0), device=DEV).half()
    cache.append(kv, kv.flip(0), torch.arange(4 * BS, dtype=torch.int32, device=DEV))
    slots = torch.full((t,), -1, dtype=torch.int32, device=DEV)
    for lo, hi in _few(t):
        slots[lo:hi] = torch.arange(hi - lo, dtype=torch.int32, device=DEV) % (4 * BS)
    got = cache.read(slots)
    for lo, hi in _few(t) + [(1000, 1100), (131072, 131100)]:
        want = cache.read(slots[lo:hi])
        assert torch.equal(got[0][lo:hi], want[0]) and torch.equal(got[1][lo:hi], want[1])


@pytest.mark.parametrize("offsets", [False, True])
def test_attention(offsets):
    b = 2 ** 24 + 5
    print("attention", offsets, flush=True)
    cache = rf.KV8Cache(3, 1, D, BS)
    kv = torch.randn(3 * BS, 1, D, generator=_gen(0), device=DEV).half()
    cache.append(kv, kv.flip(0), torch.arange(3 * BS, dtype=torch.int32, device=DEV))
    q = torch.randn(b, 1, D, generator=_gen(1), device=DEV, dtype=torch.float16)
    table = torch.randint(0, 3, (b, 1), generator=_gen(2), device=DEV, dtype=torch.int32)
    lens = torch.randint(0, BS + 1, (b,), generator=_gen(3), device=DEV, dtype=torch.int32)
    cu = torch.arange(b + 1, dtype=torch.int32, device=DEV) if offsets else None
    got, lse = rf.kv8_attention(q, cache, table, lens, cu, max_q_len=1, return_lse=True)
    step = 2 ** 22
    for lo in range(0, b, step):
        part = slice(lo, min(lo + step, b))
        want, wlse = rf.kv8_attention(q[part], cache, table[part], lens[part], return_lse=True)
        assert torch.equal(got[part], want) and torch.equal(lse[part], wlse), lo
