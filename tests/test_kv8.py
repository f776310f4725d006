"""CPU tests of the int8 paged cache: tile order, oracle, op registration and
shape inference, refusals of the torch ops and of the C ABI."""
from __future__ import annotations

import ctypes
import re
from pathlib import Path

import numpy as np
import pytest
import torch
from torch.library import opcheck

import rhinoforge_amd as rf
from oracle import kv8 as o
from rhinoforge_amd import capi

ROOT = Path(__file__).resolve().parents[1]


def _meta(shape, dtype, **kw):
    return torch.empty(shape, dtype=dtype, device="meta", **kw)


# ---- the tile order -----------------------------------------------------------------

@pytest.mark.parametrize("bs", [32, 64, 128])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_tile_order(bs, d):
    """from_quantized against the byte positions that include/kv8.h defines."""
    g = torch.Generator().manual_seed(bs + d)
    k, v = (torch.randint(-127, 128, (2, 3, bs, d), dtype=torch.int8, generator=g) for _ in range(2))
    c = rf.KV8Cache.from_quantized(k, torch.rand(2, 3), v, torch.rand(2, 3))
    kb, vb = (t.reshape(2, 3, bs // 32, 32 * d).numpy() for t in (c.k, c.v))
    token, dim = np.meshgrid(np.arange(bs), np.arange(d), indexing="ij")
    gr, t = token // 32, token % 32
    at = (t // 16 * (d // 64) + dim // 64) * 1024 + ((dim % 64 // 16) * 16 + t % 16) * 16 + dim % 16
    assert np.array_equal(kb[:, :, gr, at], (k.numpy().astype(int) + 128))
    lane = (t % 16 // 4) * 16 + dim % 16
    at = dim // 32 * 1024 + lane * 16 + (dim % 32 // 16) * 8 + t // 16 * 4 + t % 4
    assert np.array_equal(vb[:, :, gr, at], (v.numpy().astype(int) + 128))
    k2, ks2, v2, vs2 = c.to_quantized()
    assert torch.equal(k2, k) and torch.equal(v2, v)
    assert torch.equal(ks2, c.k_scale) and torch.equal(vs2, c.v_scale)
    assert (c.num_blocks, c.kv_heads, c.block_size, c.head_dim) == (2, 3, bs, d)


def test_from_quantized_takes_minus_128_as_minus_127_and_copies():
    k = torch.full((1, 1, 32, 64), -128, dtype=torch.int8)
    s = torch.ones(1, 1)
    c = rf.KV8Cache.from_quantized(k, s, k, s)
    assert (c.to_quantized()[0] == -127).all() and (k == -128).all()
    s.fill_(5)
    assert c.k_scale.item() == 1 and c.v_scale.item() == 1


def test_cache_arguments():
    for args in ((1, 1, 64, 16), (1, 1, 96, 32), (0, 1, 64, 32), (1, 0, 64, 32), (2 ** 25, 1, 64, 64)):
        with pytest.raises(ValueError):
            rf.KV8Cache(*args, device="meta")
    k = torch.zeros(2, 1, 32, 64, dtype=torch.int8)
    s = torch.ones(2, 1)
    with pytest.raises(ValueError, match="int8"):
        rf.KV8Cache.from_quantized(k.float(), s, k, s)
    with pytest.raises(ValueError, match="float32"):
        rf.KV8Cache.from_quantized(k, s.half(), k, s)
    with pytest.raises(ValueError, match="block_size"):
        rf.KV8Cache.from_quantized(k[:, :, :16], s, k[:, :, :16], s)
    empty = rf.KV8Cache(2, 1, 64, 32, device="cpu")
    assert (empty.to_quantized()[0] == 0).all() and (empty.k_scale == 0).all()


# ---- the oracle ---------------------------------------------------------------------

def test_oracle_attention_against_softmax_in_torch():
    g = torch.Generator().manual_seed(1)
    hk, d, bs = 2, 8, 4
    kq, vq = (torch.randint(-127, 128, (5, hk, bs, d), dtype=torch.int8, generator=g).numpy() for _ in range(2))
    ks, vs = (torch.rand(5, hk, generator=g).double().numpy() * 0.02 for _ in range(2))
    table = np.array([[3, 1, -1], [4, 0, 2]])
    lens, cu = [6, 11], [0, 2, 6]
    q = torch.randn(6, 6, d, generator=g).double().numpy()
    out, lse, mass, size = o.attention(q, kq, ks, vq, vs, table, lens, cu, window=5, scale=0.7)
    for r, n in enumerate(lens):
        k = np.concatenate([kq[b] * ks[b][:, None, None] for b in table[r] if b >= 0], 1)[:, :n]
        v = np.concatenate([vq[b] * vs[b][:, None, None] for b in table[r] if b >= 0], 1)[:, :n]
        nq = cu[r + 1] - cu[r]
        pos = torch.arange(n - nq, n)[:, None]
        at = torch.arange(n)[None]
        hide = (at > pos) | (at <= pos - 5)
        qq = torch.from_numpy(q[cu[r]:cu[r + 1]]).permute(1, 0, 2)
        s = qq @ torch.from_numpy(k).double().repeat_interleave(3, 0).transpose(1, 2) * 0.7
        s = s.masked_fill(hide, -torch.inf)
        ref = torch.softmax(s, -1) @ torch.from_numpy(v).double().repeat_interleave(3, 0)
        assert np.allclose(out[cu[r]:cu[r + 1]], ref.permute(1, 0, 2).numpy(), atol=1e-12)
        assert np.allclose(lse[cu[r]:cu[r + 1]], torch.logsumexp(s, -1).T.numpy(), atol=1e-12)
    assert (mass >= np.abs(out) - 1e-12).all() and (size > 0).all()
    none = o.attention(q[:4], kq, ks, vq, vs, table[:1], [2], [0, 4], scale=1.0)
    assert (none[0][:2] == 0).all() and np.isneginf(none[1][:2]).all()
    assert np.isfinite(none[1][2:]).all()


def test_oracle_rope_is_a_rotation_and_a_norm():
    r = np.random.default_rng(0)
    x = r.standard_normal((4, 2, 32))
    ang = r.random((9, 8)) * 6
    for inter in (False, True):
        y = o.norm_rope(x, None, np.cos(ang), np.sin(ang), [0, 8, 3, 5], 1e-6, inter)
        assert np.allclose((y ** 2).sum(-1), (x ** 2).sum(-1)) and np.allclose(y[..., 16:], x[..., 16:])
        pair = (0, 1) if inter else (0, 8)
        z = (x[1, 0, pair[0]] + 1j * x[1, 0, pair[1]]) * np.exp(1j * ang[8, 0])
        assert np.allclose(y[1, 0, list(pair)], [z.real, z.imag])
    y = o.norm_rope(x, np.full(32, 2.0), None, None, None, 0.0, False)
    assert np.allclose((y ** 2).mean(-1), 4.0)


def test_oracle_append_keeps_the_largest_magnitude():
    q, s = np.zeros((2, 1, 4, 2)), np.zeros((2, 1))
    q, s, _ = o.append(q, s, np.array([[[1.0, -0.5]], [[0.25, 0.0]]]), [4, 5])
    assert s[1, 0] == 1 / 127 and q[1, 0, :2].tolist() == [[127, -64], [32, 0]]
    q, s, _ = o.append(q, s, np.array([[[2.0, 0.0]]]), [6])
    assert s[1, 0] == 2 / 127 and q[1, 0, :3].tolist() == [[64, -32], [16, 0], [127, 0]]
    q, s, _ = o.append(q, s, np.array([[[0.5, 0.0]]]), [7])
    assert s[1, 0] == 2 / 127 and q[1, 0, 3].tolist() == [32, 0]
    q, s, _ = o.append(q, s, np.array([[[0.5, 0.0]]]), [4])  # a block begun again
    assert s[1, 0] == 0.5 / 127


def test_oracle_plan():
    table, slots, pos, cu, lens, nxt = o.plan(
        np.array([[7, -1], [-1, -1]]), [3, 0], [2, 5], [10, 11, 12, 13], 1, 9, 4)
    assert table.tolist() == [[7, 11], [12, 13]] and nxt == 4
    assert slots.tolist() == [31, 44, 48, 49, 50, 51, 52, -1, -1]
    assert pos.tolist() == [3, 4, 0, 1, 2, 3, 4, 0, 0]
    assert cu.tolist() == [0, 2, 7] and lens.tolist() == [5, 5]


# ---- registration and shapes ----------------------------------------------------------

def _cache_meta(nb=3, hk=2, bs=64, d=128, device="meta"):
    z = lambda s, t: torch.zeros(s, dtype=t, device=device)  # noqa: E731
    tiles = (nb, hk, bs // 32, d // 32, 1024)
    return (z(tiles, torch.uint8), z(tiles, torch.uint8), z((nb, hk), torch.float32),
            z((nb, hk), torch.float32))


def _cases(dev="meta"):
    z = lambda s, t: torch.zeros(s, dtype=t, device=dev)  # noqa: E731
    h, i = torch.float16, torch.int32
    c = _cache_meta(device=dev)
    q, k = z((5, 6, 128), h), z((5, 2, 128), h)
    w, cos = z((128,), h), z((50, 64), torch.float32)
    ops = torch.ops.kv8
    return {
        "kv8::qk_norm_rope": (ops.qk_norm_rope.default, (q, k, w, w, cos, cos, z((5,), torch.int64), 1e-6, False)),
        "kv8::qk_norm_rope plain": (ops.qk_norm_rope.default, (q, k, None, None, None, None, None, 1e-6, True)),
        "kv8::plan": (ops.plan.default, (z((2, 4), i), z((2,), i), z((2,), i), z((9,), i), z((1,), i), 7, 64)),
        "kv8::append": (ops.append.default, (*c, k, k, z((5,), i))),
        "kv8::read": (ops.read.default, (*c, z((3,), i), torch.bfloat16)),
        "kv8::attention": (ops.attention.default,
                           (q, *c, z((2, 4), i), z((2,), i), z((3,), i), 0, 0, True, 0, 0.1, False)),
        "kv8::attention lse": (ops.attention.default,
                               (q, *c, z((1, 4), i), z((1,), i), None, 5, 99, True, 8, 0.1, True)),
    }


@pytest.mark.parametrize("name", sorted(_cases()))
def test_opcheck_every_schema(name):
    op, args = _cases()[name]
    report = opcheck(op, args, raise_exception=False)
    failed = {k: v for k, v in report.items() if v != "SUCCESS"}
    assert not failed, f"{name}: {failed}"


def test_every_schema_is_covered():
    registered = {n for n in torch._C._dispatch_get_all_op_names() if n.startswith("kv8::")}
    assert registered == {n.split(" ")[0] for n in _cases()}


def test_shapes_and_no_graph():
    c = _cases()
    out, lse = c["kv8::attention lse"][0](*c["kv8::attention lse"][1])
    assert out.shape == (5, 6, 128) and out.dtype == torch.float16
    assert lse.shape == (5, 6) and lse.dtype == torch.float32
    out, lse = c["kv8::attention"][0](*c["kv8::attention"][1])
    assert lse.shape == (0,)
    k, v = c["kv8::read"][0](*c["kv8::read"][1])
    assert k.shape == v.shape == (3, 2, 128) and k.dtype == torch.bfloat16
    p = c["kv8::plan"][0](*c["kv8::plan"][1])
    assert [tuple(x.shape) for x in p] == [(7,), (7,), (3,), (2,), (1,)]
    q = _meta((5, 6, 128), torch.float16, requires_grad=True)
    y, _ = torch.ops.kv8.qk_norm_rope(q, q, None, None, None, None, None, 1e-6, False)
    assert not y.requires_grad


@pytest.mark.parametrize("name", sorted(_cases()))
def test_there_is_no_cpu_computation(name):
    op, args = _cases("cpu")[name]
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        op(*args)


# ---- refusals ---------------------------------------------------------------------------

def _refused(name, match, **change):
    """The op of that name with arguments replaced by position."""
    op, args = _cases()[name]
    args = list(args)
    for at, v in change.items():
        args[int(at[1:])] = v
    with pytest.raises(RuntimeError, match=match):
        op(*args)


def test_refusals():
    h, i, f = torch.float16, torch.int32, torch.float32
    n = "kv8::qk_norm_rope"
    _refused(n, "float16 or bfloat16", a0=_meta((5, 6, 128), f))
    _refused(n, "as q", a1=_meta((5, 2, 128), torch.bfloat16))
    _refused(n, "same tokens and head_dim", a1=_meta((4, 2, 128), h))
    _refused(n, "same tokens and head_dim", a1=_meta((5, 2, 64), h))
    _refused(n, "same tokens and head_dim", a0=_meta((5, 768), h))
    _refused(n, "norm weight", a2=_meta((64,), h))
    _refused(n, "norm weight", a3=_meta((128,), f))
    _refused(n, "go together", a5=None)
    _refused(n, "float32", a4=_meta((50, 64), h))
    _refused(n, "differ in shape", a4=_meta((49, 64), f))
    _refused(n, "multiple of 16", a4=_meta((50, 68), f), a5=_meta((50, 68), f))
    _refused(n, "multiple of 16", a4=_meta((50, 4), f), a5=_meta((50, 4), f))
    _refused(n, "no rows", a4=_meta((0, 64), f), a5=_meta((0, 64), f))
    _refused(n, "positions must", a6=_meta((5,), f))
    _refused(n, "positions must", a6=_meta((4,), i))
    _refused(n, "a row for each token", a6=None, a4=_meta((4, 64), f), a5=_meta((4, 64), f))
    with pytest.raises(RuntimeError, match="multiple of 8"):
        rf.qk_norm_rope(_meta((1, 1, 12), h), _meta((1, 1, 12), h), None, None, None, None)
    n = "kv8::plan"
    _refused(n, "int32", a0=_meta((2, 4), torch.int64))
    _refused(n, "dimension", a1=_meta((2, 1), i))
    _refused(n, "differ in requests", a2=_meta((3,), i))
    _refused(n, "contiguous", a1=_meta((4,), i)[::2])
    _refused(n, "unit stride", a0=_meta((4, 2), i).t())
    _refused(n, "one element", a4=_meta((2,), i))
    _refused(n, "num_tokens", a5=-1)
    _refused(n, "block_size", a6=48)
    _refused(n, "requests", a0=_meta((8193, 4), i), a1=_meta((8193,), i), a2=_meta((8193,), i))
    n = "kv8::append"
    _refused(n, "uint8", a0=_meta((3, 2, 2, 4, 1024), torch.int8))
    _refused(n, "one shape", a1=_meta((3, 2, 4, 4, 1024), torch.uint8))
    _refused(n, "float32", a2=_meta((3, 2), h))
    _refused(n, "float32", a3=_meta((2, 3), f))
    _refused(n, "kv_heads", a4=_meta((5, 3, 128), h))
    _refused(n, "kv_heads", a5=_meta((4, 2, 128), h))
    _refused(n, "as k", a5=_meta((5, 2, 128), torch.bfloat16))
    _refused(n, "int32", a6=_meta((5,), torch.int64))
    bad = _cache_meta()
    for k in ((3, 2, 3, 4, 1024), (3, 2, 2, 3, 1024), (0, 2, 2, 4, 1024)):
        t = _meta(k, torch.uint8)
        _refused(n, "block_size|head_dim|empty", a0=t, a1=t, a2=_meta(k[:2], f), a3=_meta(k[:2], f))
    _refused("kv8::read", "dtype", a5=torch.float64)
    _refused("kv8::read", "int32", a4=_meta((3,), torch.int64))
    n = "kv8::attention"
    _refused(n, "float16 or bfloat16", a0=_meta((5, 6, 128), f))
    _refused(n, "tokens, heads, 128", a0=_meta((5, 6, 64), h))
    _refused(n, "multiple of the cache's", a0=_meta((5, 5, 128), h))
    _refused(n, "differ in requests", a5=_meta((3, 4), i))
    _refused(n, "cu_q must have", a7=_meta((2,), i))
    _refused(n, "multiple of the requests", a7=None)
    _refused(n, "negative", a8=-1)
    _refused(n, "negative", a9=-1)
    _refused(n, "window", a11=-1)
    _refused(n, "window", a10=False, a11=5)
    for s in (0.0, -1.0, float("inf"), float("nan"), 1e-60):
        _refused(n, "scale", a12=s)


# ---- the C ABI ----------------------------------------------------------------------------

def _declared():
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "kv8.h").read_text(), flags=re.S)
    return sorted(set(re.findall(r"\b(rf_kv8_\w+)\s*\(", text)))


def test_header_and_binding_agree():
    assert _declared() == sorted(capi.KV8_SIGNATURES)
    lib = ctypes.CDLL(str(capi.LIB_PATH))
    assert all(hasattr(lib, n) for n in _declared())


P = 1 << 20  # a 16-byte aligned address that nothing reads: every call is refused


def _c_cache(**kw):
    return capi.KV8Cache(**{**dict(k=P, v=P, k_scale=P, v_scale=P, num_blocks=4, kv_heads=2,
                                   head_dim=128, block_size=64), **kw})


def _c_heads(heads=2, **kw):
    return capi.KV8Heads(**{**dict(data=P, token_stride=heads * 128, head_stride=128, heads=heads), **kw})


def _c_attention(cache=None, q=None, **kw):
    a = dict(cu_q=P, kv_lens=P, block_table=P, out=P, lse=None, scratch=None,
             tokens=4, requests=2, width=3, table_stride=3, max_q_len=0, max_kv_len=0, dtype=0, causal=1,
             window=0, scale=0.1)
    return capi.KV8AttentionArgs(cache=cache or _c_cache(), q=q or _c_heads(4), **{**a, **kw})


@pytest.mark.parametrize("want,args", [
    (capi.EINVAL, dict(cache=dict(head_dim=96))), (capi.EINVAL, dict(cache=dict(block_size=16))),
    (capi.EINVAL, dict(cache=dict(k=None))), (capi.EINVAL, dict(cache=dict(v_scale=None))),
    (capi.EINVAL, dict(cache=dict(num_blocks=0))), (capi.EINVAL, dict(cache=dict(num_blocks=2 ** 26))),
    (capi.EALIGN, dict(cache=dict(v=P + 8))), (capi.EINVAL, dict(q=dict(heads=3))),
    (capi.EINVAL, dict(q=dict(data=None))), (capi.EALIGN, dict(q=dict(data=P + 2))),
    (capi.EALIGN, dict(q=dict(token_stride=12))), (capi.EINVAL, dict(dtype=2)),
    (capi.EINVAL, dict(kv_lens=None)), (capi.EINVAL, dict(out=None)), (capi.EALIGN, dict(out=P + 8)),
    (capi.EALIGN, dict(lse=P + 2)), (capi.EINVAL, dict(tokens=-1)), (capi.EINVAL, dict(tokens=2 ** 29 + 2)),
    (capi.EINVAL, dict(width=2 ** 25, table_stride=2 ** 25)),
    (capi.EINVAL, dict(tokens=5, cu_q=None)), (capi.EINVAL, dict(requests=0)), (capi.EINVAL, dict(width=0)),
    (capi.EINVAL, dict(table_stride=2)), (capi.EINVAL, dict(scale=0.0)), (capi.EINVAL, dict(scale=float("nan"))),
    (capi.EINVAL, dict(scale=float("inf"))), (capi.EINVAL, dict(window=-1)),
    (capi.EINVAL, dict(window=4, causal=0)), (capi.EINVAL, dict(max_q_len=-1)),
])
def test_attention_refusals_of_the_c_abi(want, args):
    args = dict(args)
    cache = _c_cache(**args.pop("cache", {}))
    q = _c_heads(**{"heads": 4, **args.pop("q", {})})
    a = _c_attention(cache, q, **args)
    assert capi.load().rf_kv8_attention(ctypes.byref(a), None) == want
    assert capi.load().rf_kv8_attention_workspace(ctypes.byref(a)) == 0


def test_other_refusals_of_the_c_abi():
    lib, ref = capi.load(), ctypes.byref
    assert lib.rf_kv8_attention(None, None) == capi.EINVAL
    assert lib.rf_kv8_attention(ref(_c_attention(tokens=0)), None) == capi.OK
    rope = dict(q=_c_heads(4), k=_c_heads(), q_out=P, k_out=P, cos=P, sin=P, positions=P, tokens=3,
                table_rows=9, head_dim=128, rot=128, dtype=0, positions64=1, interleaved=0, eps=1e-6)
    for want, kw in ((capi.EINVAL, dict(head_dim=12)), (capi.EINVAL, dict(head_dim=520)), (capi.EINVAL, dict(rot=24)),
                     (capi.EINVAL, dict(rot=144)), (capi.EINVAL, dict(cos=None)), (capi.EINVAL, dict(dtype=2)),
                     (capi.EINVAL, dict(q_out=None)), (capi.EALIGN, dict(k_out=P + 8)), (capi.EALIGN, dict(sin=P + 4)),
                     (capi.EALIGN, dict(positions=P + 4)), (capi.EINVAL, dict(positions=None, table_rows=2)),
                     (capi.EINVAL, dict(tokens=-1)), (capi.EALIGN, dict(k=_c_heads(head_stride=4))),
                     (capi.EALIGN, dict(q_weight=P + 2)), (capi.OK, dict(tokens=0))):
        assert lib.rf_kv8_qk_norm_rope(ref(capi.KV8RopeArgs(**{**rope, **kw})), None) == want, kw
    plan = dict(block_table=P, cached=P, fresh=P, free_blocks=P, free_start=P, slots=P, positions=P, cu=P,
                kv_lens=P, free_next=P, requests=2, width=4, table_stride=4, num_free=3, tokens=5, block_size=64)
    for want, kw in ((capi.EINVAL, dict(requests=0)), (capi.EINVAL, dict(requests=8193)), (capi.EINVAL, dict(width=0)),
                     (capi.EINVAL, dict(table_stride=3)), (capi.EINVAL, dict(block_size=256)),
                     (capi.EINVAL, dict(cu=None)), (capi.EINVAL, dict(free_blocks=None)),
                     (capi.EINVAL, dict(slots=None)), (capi.EALIGN, dict(slots=P + 2)), (capi.EINVAL, dict(tokens=-1))):
        assert lib.rf_kv8_plan(ref(capi.KV8PlanArgs(**{**plan, **kw})), None) == want, kw
    c, h = _c_cache(), _c_heads()
    assert lib.rf_kv8_append(ref(c), ref(h), ref(_c_heads(4)), 0, P, 3, None) == capi.EINVAL
    assert lib.rf_kv8_append(ref(c), ref(h), ref(h), 2, P, 3, None) == capi.EINVAL
    assert lib.rf_kv8_append(ref(c), ref(h), ref(h), 0, None, 3, None) == capi.EINVAL
    assert lib.rf_kv8_append(ref(c), ref(h), ref(h), 0, P + 2, 3, None) == capi.EALIGN
    assert lib.rf_kv8_append(ref(c), ref(h), ref(h), 0, P, 0, None) == capi.OK
    assert lib.rf_kv8_append(ref(c), None, ref(h), 0, P, 1, None) == capi.EINVAL
    assert lib.rf_kv8_read(ref(c), P, 3, 3, P, P, None) == capi.EINVAL
    assert lib.rf_kv8_read(ref(c), P, 3, 0, None, P, None) == capi.EINVAL
    assert lib.rf_kv8_read(ref(c), P, 3, 2, P, P + 16, None) == capi.EALIGN
    assert lib.rf_kv8_read(ref(c), P, -1, 0, P, P, None) == capi.EINVAL
    assert lib.rf_kv8_read(ref(c), None, 0, 0, None, None, None) == capi.OK
