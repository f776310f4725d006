"""CPU tests of the 4-bit paged cache and of the rotation by several axes: bit order,
oracle, op registration and shape inference, refusals of the torch ops and of the C
ABI."""
from __future__ import annotations

import ctypes
import re
from pathlib import Path

import numpy as np
import pytest
import torch
from torch.library import opcheck

import rhinoforge_amd as rf
from oracle import kv4 as o
from rhinoforge_amd import capi

ROOT = Path(__file__).resolve().parents[1]


def _meta(shape, dtype, **kw):
    return torch.empty(shape, dtype=dtype, device="meta", **kw)


def _numbers(shape, seed):
    g = torch.Generator().manual_seed(seed)
    n = torch.randint(0, 16, shape, generator=g).to(torch.uint8)
    step = (torch.randint(0x10, 0x6c40, shape[:3], generator=g) & ~15).to(torch.int16).view(torch.float16)
    return n, step, torch.randint(0, 16, shape[:3], generator=g).to(torch.uint8)


# ---- the order of the bits ------------------------------------------------------------

@pytest.mark.parametrize("bs", [32, 64, 128])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_bit_order(bs, d):
    """from_quantized against the positions that include/kv4.h defines."""
    k, v = _numbers((2, 3, bs, d), bs + d), _numbers((2, 3, bs, d), bs + d + 1)
    c = rf.KV4Cache.from_quantized(*k, *v)
    assert (c.num_blocks, c.kv_heads, c.block_size, c.head_dim) == (2, 3, bs, d)
    kw, vw = (t.reshape(2, 3, bs // 32, 16 * d).numpy().view("<u4").astype(np.int64) for t in (c.k, c.v))
    token, dim = np.meshgrid(np.arange(bs), np.arange(d), indexing="ij")
    gr, t, tile, x = token // 32, token % 32, dim // 64, dim % 64
    lane, w, e = x // 16 * 16 + t // 8 * 4 + t % 4, t // 4 % 2 * 2 + x % 16 // 8, x % 8
    assert np.array_equal(kw[:, :, gr, tile * 256 + lane * 4 + w] >> 4 * (e // 2 + 4 * (e % 2)) & 15, k[0].numpy())
    lane, w = t // 8 * 16 + x // 4, t % 8 // 2
    assert np.array_equal(vw[:, :, gr, tile * 256 + lane * 4 + w] >> 16 * (t % 2) + 4 * (x % 4) & 15, v[0].numpy())
    for side, (_, s, z) in enumerate((k, v)):
        word = c.rows.transpose(2, 3)[:, :, side].reshape(2, 3, bs)
        assert torch.equal(word & 15, z.to(torch.int16)) and torch.equal((word & ~15).view(torch.float16), s)
    for got, want in zip(c.to_quantized(), (*k, *v)):
        assert got.dtype == want.dtype and torch.equal(got, want)


def test_a_new_cache_holds_zeros():
    c = rf.KV4Cache(2, 1, 64, 32, device="cpu")
    k, ks, kz, v, vs, vz = c.to_quantized()
    assert not k.any() and not v.any() and not kz.any() and not vz.any()
    assert (ks == 2.0 ** -20).all() and (vs == 2.0 ** -20).all()


def test_from_quantized_takes_copies_and_nan_marks():
    k, v = _numbers((2, 1, 32, 64), 1), _numbers((2, 1, 32, 64), 2)
    k[1][0, 0, 5] = float("nan")
    c = rf.KV4Cache.from_quantized(*k, *v)
    assert int((c.rows == 0x7e00).sum()) == 1
    back = c.to_quantized()
    assert torch.isnan(back[1][0, 0, 5]) and int(torch.isnan(back[1]).sum()) == 1
    k[0].fill_(0)
    assert c.k.any()


def test_cache_arguments():
    for args in ((1, 1, 64, 16), (1, 1, 96, 32), (0, 1, 64, 32), (1, 0, 64, 32), (2 ** 25, 1, 64, 64)):
        with pytest.raises(ValueError):
            rf.KV4Cache(*args, device="meta")
    k, s, z = _numbers((2, 1, 32, 64), 3)
    make = rf.KV4Cache.from_quantized
    for match, args in (("uint8", (k.float(), s, z, k, s, z)), ("float16", (k, s.float(), z, k, s, z)),
                        ("zero points", (k, s, z, k, s, z.int())), ("float16", (k, s[:1], z, k, s, z)),
                        ("block_size", (k[:, :, :16], s[:, :, :16], z[:, :, :16], k[:, :, :16], s[:, :, :16], z[:, :, :16])),
                        ("0..15", (k + 16, s, z, k, s, z)), ("0..15", (k, s, z + 16, k, s, z)),
                        ("four", (k, s, z, k, torch.full_like(s, 1 + 2 ** -10), z)),
                        ("steps", (k, -s, z, k, s, z)), ("steps", (k, s, z, k, s * 0, z)),
                        ("steps", (k, s, z, k, s * float("nan"), z)),
                        ("steps", (k, torch.full_like(s, 8192.0), z, k, s, z))):
        with pytest.raises(ValueError, match=match):
            make(*args)


# ---- the oracle -----------------------------------------------------------------------

@pytest.mark.parametrize("span,step", [
    (0.0, 2.0 ** -20), (15.0, 1.0), (15.1, 1.015625), (15 * 127 / 64, 127 / 64), (29.9, 2.0), (30.0, 2.0),
    (15 * 2.0 ** -14, 2.0 ** -14), (14.9 * 2.0 ** -16, 2.0 ** -16), (15.01 * 2.0 ** -16, 2.0 ** -16 + 2.0 ** -20),
    (1e6, 4352.0), (65280.0, 4352.0), (65000.0, 4352.0)])
def test_oracle_step(span, step):
    assert o.step_of(0.0, span)[1] == step and o.step_of(-span, 0.0)[1] == step


def test_oracle_quantizer_is_off_by_half_a_step_at_most():
    r = np.random.default_rng(0)
    x = (r.standard_normal((500, 64)) * np.exp(r.standard_normal((500, 1)) * 3)).astype(np.float16).clip(-3e4, 3e4)
    x[:50] = np.abs(x[:50])
    x[50] = 0
    n, s, z = o.quantize(x)
    assert (np.abs(o.values(n, s, z) - x) <= s[:, None] / 2).all()
    assert np.array_equal(o.values(n, s, z), o.values(n, s, z).astype(np.float16).astype(np.float64))
    assert ((s.astype(np.float16).view(np.int16) & 15) == 0).all()
    assert n.min() == 0 and n.max() == 15 and (s[:50] * 15 >= x[:50].max(-1)).all()


def test_oracle_axes():
    assert o.axis_of_pairs([3, 1, 2], False) == [0, 0, 0, 1, 2, 2]
    assert o.axis_of_pairs([4, 2, 2], True) == [0, 1, 2, 0, 1, 2, 0, 0]
    assert o.axis_of_pairs([2, 1, 2], True) == [0, 1, 2, 0, 0]   # (the last pair has no place of its own)
    assert o.axis_of_pairs([2, 2], True) == [0, 1, 0, 1]


def test_oracle_attention_against_softmax_in_torch():
    g = torch.Generator().manual_seed(1)
    hk, d, bs = 2, 8, 4
    k, v = (torch.randn(5, hk, bs, d, generator=g, dtype=torch.float64).numpy() for _ in range(2))
    table, lens, cu = np.array([[3, 1, -1], [4, 0, 2]]), [6, 11], [0, 2, 6]
    q = torch.randn(6, 6, d, generator=g).double().numpy()
    out, lse, mass, size = o.attention(q, k, v, table, lens, cu, window=5, scale=0.7)
    for r, n in enumerate(lens):
        kk, vv = (np.concatenate([x[b] for b in table[r] if b >= 0], 1)[:, :n] for x in (k, v))
        nq = cu[r + 1] - cu[r]
        pos, at = torch.arange(n - nq, n)[:, None], torch.arange(n)[None]
        qq = torch.from_numpy(q[cu[r]:cu[r + 1]]).permute(1, 0, 2)
        s = qq @ torch.from_numpy(kk).repeat_interleave(3, 0).transpose(1, 2) * 0.7
        s = s.masked_fill((at > pos) | (at <= pos - 5), -torch.inf)
        ref = torch.softmax(s, -1) @ torch.from_numpy(vv).repeat_interleave(3, 0)
        assert np.allclose(out[cu[r]:cu[r + 1]], ref.permute(1, 0, 2).numpy(), atol=1e-12)
        assert np.allclose(lse[cu[r]:cu[r + 1]], torch.logsumexp(s, -1).T.numpy(), atol=1e-12)
    assert (mass >= np.abs(out) - 1e-12).all() and (size > 0).all()
    none = o.attention(q[:4], k, v, table[:1], [2], [0, 4], scale=1.0)
    assert (none[0][:2] == 0).all() and np.isneginf(none[1][:2]).all() and np.isfinite(none[1][2:]).all()


# ---- registration and shapes ------------------------------------------------------------

def _cache(nb=3, hk=2, bs=64, d=128, device="meta"):
    tiles = (nb, hk, bs // 32, d // 64, 1024)
    z = lambda s, t: torch.zeros(s, dtype=t, device=device)  # noqa: E731
    return z(tiles, torch.uint8), z(tiles, torch.uint8), z((*tiles[:3], 2, 32), torch.int16)


def _cases(dev="meta"):
    z = lambda s, t: torch.zeros(s, dtype=t, device=dev)  # noqa: E731
    h, i = torch.float16, torch.int32
    c = _cache(device=dev)
    q, k = z((5, 6, 128), h), z((5, 2, 128), h)
    w, cos = z((128,), h), z((50, 64), torch.float32)
    kv4, rope = torch.ops.kv4, torch.ops.rope
    return {
        "rope::qk_norm_mrope": (rope.qk_norm_mrope.default,
                                (q, k, w, w, cos, cos, z((3, 5), torch.int64), [24, 20, 20], True, 1e-6, False)),
        "rope::qk_norm_mrope plain": (rope.qk_norm_mrope.default,
                                      (q, k, None, None, cos, cos, z((2, 5), i), [30, 34], False, 1e-6, True)),
        "kv4::append": (kv4.append.default, (*c, k, k, z((5,), i))),
        "kv4::read": (kv4.read.default, (*c, z((3,), i), torch.bfloat16)),
        "kv4::attention": (kv4.attention.default,
                           (q, *c, z((2, 4), i), z((2,), i), z((3,), i), 0, 0, True, 0, 0.1, False)),
        "kv4::attention lse": (kv4.attention.default,
                               (q, *c, z((1, 4), i), z((1,), i), None, 5, 99, True, 8, 0.1, True)),
    }


@pytest.mark.parametrize("name", sorted(_cases()))
def test_opcheck_every_schema(name):
    op, args = _cases()[name]
    failed = {k: v for k, v in opcheck(op, args, raise_exception=False).items() if v != "SUCCESS"}
    assert not failed, f"{name}: {failed}"


def test_every_schema_is_covered():
    registered = {n for n in torch._C._dispatch_get_all_op_names() if n.startswith(("kv4::", "rope::"))}
    assert registered == {n.split(" ")[0] for n in _cases()}


def test_shapes_and_no_graph():
    c = _cases()
    out, lse = c["kv4::attention lse"][0](*c["kv4::attention lse"][1])
    assert out.shape == (5, 6, 128) and out.dtype == torch.float16
    assert lse.shape == (5, 6) and lse.dtype == torch.float32
    assert c["kv4::attention"][0](*c["kv4::attention"][1])[1].shape == (0,)
    k, v = c["kv4::read"][0](*c["kv4::read"][1])
    assert k.shape == v.shape == (3, 2, 128) and k.dtype == torch.bfloat16
    q = _meta((5, 6, 128), torch.float16, requires_grad=True)
    cos = _meta((9, 64), torch.float32)
    y, z = rf.qk_norm_mrope(q, q, None, None, cos, cos, _meta((1, 5), torch.int32), [64])
    assert y.shape == q.shape and not y.requires_grad and z.shape == q.shape


@pytest.mark.parametrize("name", sorted(_cases()))
def test_there_is_no_cpu_computation(name):
    op, args = _cases("cpu")[name]
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        op(*args)


# ---- refusals -----------------------------------------------------------------------------

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
    n = "rope::qk_norm_mrope"
    _refused(n, "float16 or bfloat16", a0=_meta((5, 6, 128), f))
    _refused(n, "as q", a1=_meta((5, 2, 128), torch.bfloat16))
    _refused(n, "norm weight", a2=_meta((64,), h))
    _refused(n, "differ in shape", a4=_meta((49, 64), f))
    _refused(n, "no rows", a4=_meta((0, 64), f), a5=_meta((0, 64), f))
    _refused(n, "positions must", a6=_meta((3, 5), f))
    _refused(n, "positions must", a6=_meta((5,), i))
    _refused(n, "positions must", a6=_meta((2, 5), i))
    _refused(n, "positions must", a6=_meta((3, 4), i))
    _refused(n, "sections", a7=[])
    _refused(n, "sections", a6=_meta((5, 5), i), a7=[24, 10, 10, 10, 10])
    _refused(n, "add up", a7=[24, 20, 19])
    _refused(n, "negative", a7=[84, 0, -20])
    _refused(n, "mixed", a7=[20, 22, 22])
    n = "kv4::append"
    _refused(n, "uint8", a0=_meta((3, 2, 2, 2, 1024), torch.int8))
    _refused(n, "one shape", a1=_meta((3, 2, 4, 2, 1024), torch.uint8))
    _refused(n, "int16", a2=_meta((3, 2, 2, 2, 32), h))
    _refused(n, "int16", a2=_meta((3, 2, 2, 32, 2), torch.int16))
    _refused(n, "kv_heads", a3=_meta((5, 3, 128), h))
    _refused(n, "kv_heads", a4=_meta((4, 2, 128), h))
    _refused(n, "as k", a4=_meta((5, 2, 128), torch.bfloat16))
    _refused(n, "int32", a5=_meta((5,), torch.int64))
    for k in ((3, 2, 3, 2, 1024), (3, 2, 2, 3, 1024), (0, 2, 2, 2, 1024)):
        t = _meta(k, torch.uint8)
        _refused(n, "block_size|head_dim|empty", a0=t, a1=t)
    _refused("kv4::read", "dtype", a4=torch.float64)
    _refused("kv4::read", "int32", a3=_meta((3,), torch.int64))
    n = "kv4::attention"
    _refused(n, "float16 or bfloat16", a0=_meta((5, 6, 128), f))
    _refused(n, "tokens, heads, 128", a0=_meta((5, 6, 64), h))
    _refused(n, "multiple of the cache's", a0=_meta((5, 5, 128), h))
    _refused(n, "differ in requests", a4=_meta((3, 4), i))
    _refused(n, "cu_q must have", a6=_meta((2,), i))
    _refused(n, "multiple of the requests", a6=None)
    _refused(n, "negative", a7=-1)
    _refused(n, "negative", a8=-1)
    _refused(n, "window", a10=-1)
    _refused(n, "window", a9=False, a10=5)
    for s in (0.0, -1.0, float("inf"), float("nan"), 1e-60):
        _refused(n, "scale", a11=s)


# ---- the C ABI ------------------------------------------------------------------------------

def _declared():
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "kv4.h").read_text(), flags=re.S)
    return sorted(set(re.findall(r"\b(rf_kv4_\w+)\s*\(", text)))


def test_header_and_binding_agree():
    assert _declared() == sorted(capi.KV4_SIGNATURES)
    lib = ctypes.CDLL(str(capi.LIB_PATH))
    assert all(hasattr(lib, n) for n in _declared())


P = 1 << 20  # a 16-byte aligned address that nothing reads: every call is refused


def _c_cache(**kw):
    return capi.KV4Cache(**{**dict(k=P, v=P, rows=P, num_blocks=4, kv_heads=2, head_dim=128, block_size=64), **kw})


def _c_heads(heads=2, **kw):
    return capi.KV8Heads(**{**dict(data=P, token_stride=heads * 128, head_stride=128, heads=heads), **kw})


@pytest.mark.parametrize("want,args", [
    (capi.EINVAL, dict(cache=dict(head_dim=96))), (capi.EINVAL, dict(cache=dict(block_size=16))),
    (capi.EINVAL, dict(cache=dict(k=None))), (capi.EINVAL, dict(cache=dict(rows=None))),
    (capi.EINVAL, dict(cache=dict(num_blocks=0))), (capi.EINVAL, dict(cache=dict(num_blocks=2 ** 26))),
    (capi.EALIGN, dict(cache=dict(v=P + 8))), (capi.EALIGN, dict(cache=dict(rows=P + 2))),
    (capi.EINVAL, dict(q=dict(heads=3))), (capi.EINVAL, dict(q=dict(data=None))),
    (capi.EALIGN, dict(q=dict(data=P + 2))), (capi.EALIGN, dict(q=dict(token_stride=12))),
    (capi.EINVAL, dict(dtype=2)), (capi.EINVAL, dict(kv_lens=None)), (capi.EINVAL, dict(out=None)),
    (capi.EALIGN, dict(out=P + 8)), (capi.EALIGN, dict(lse=P + 2)), (capi.EINVAL, dict(tokens=-1)),
    (capi.EINVAL, dict(tokens=2 ** 29 + 2)), (capi.EINVAL, dict(width=2 ** 25, table_stride=2 ** 25)),
    (capi.EINVAL, dict(tokens=5, cu_q=None)), (capi.EINVAL, dict(requests=0)), (capi.EINVAL, dict(width=0)),
    (capi.EINVAL, dict(table_stride=2)), (capi.EINVAL, dict(scale=0.0)), (capi.EINVAL, dict(scale=float("nan"))),
    (capi.EINVAL, dict(scale=float("inf"))), (capi.EINVAL, dict(window=-1)),
    (capi.EINVAL, dict(window=4, causal=0)), (capi.EINVAL, dict(max_q_len=-1)),
])
def test_attention_refusals_of_the_c_abi(want, args):
    args = dict(args)
    a = dict(cu_q=P, kv_lens=P, block_table=P, out=P, lse=None, scratch=None, tokens=4, requests=2, width=3,
             table_stride=3, max_q_len=0, max_kv_len=0, dtype=0, causal=1, window=0, scale=0.1)
    cache = _c_cache(**args.pop("cache", {}))
    q = _c_heads(**{"heads": 4, **args.pop("q", {})})
    call = capi.KV4AttentionArgs(cache=cache, q=q, **{**a, **args})
    assert capi.load().rf_kv4_attention(ctypes.byref(call), None) == want
    assert capi.load().rf_kv4_attention_workspace(ctypes.byref(call)) == 0


def test_other_refusals_of_the_c_abi():
    lib, ref = capi.load(), ctypes.byref
    assert lib.rf_kv4_attention(None, None) == capi.EINVAL
    c, h = _c_cache(), _c_heads()
    assert lib.rf_kv4_append(ref(c), ref(h), ref(_c_heads(4)), 0, P, 3, None) == capi.EINVAL
    assert lib.rf_kv4_append(ref(c), ref(h), ref(h), 2, P, 3, None) == capi.EINVAL
    assert lib.rf_kv4_append(ref(c), ref(h), ref(h), 0, None, 3, None) == capi.EINVAL
    assert lib.rf_kv4_append(ref(c), ref(h), ref(h), 0, P + 2, 3, None) == capi.EALIGN
    assert lib.rf_kv4_append(ref(c), ref(h), ref(h), 0, P, 0, None) == capi.OK
    assert lib.rf_kv4_append(ref(c), None, ref(h), 0, P, 1, None) == capi.EINVAL
    assert lib.rf_kv4_append(None, ref(h), ref(h), 0, P, 1, None) == capi.EINVAL
    assert lib.rf_kv4_read(ref(c), P, 3, 3, P, P, None) == capi.EINVAL
    assert lib.rf_kv4_read(ref(c), P, 3, 0, None, P, None) == capi.EINVAL
    assert lib.rf_kv4_read(ref(c), P, 3, 2, P, P + 16, None) == capi.EALIGN
    assert lib.rf_kv4_read(ref(c), P, -1, 0, P, P, None) == capi.EINVAL
    assert lib.rf_kv4_read(ref(c), None, 0, 0, None, None, None) == capi.OK
    rope = dict(q=_c_heads(4), k=_c_heads(), q_out=P, k_out=P, cos=P, sin=P, positions=P, tokens=3,
                table_rows=9, head_dim=128, rot=128, dtype=0, positions64=1, interleaved=0, eps=1e-6)
    mrope = dict(axis_stride=3, axes=3, mixed=1, sections=(24, 20, 20, 0))
    for want, kw, inner in ((capi.EINVAL, dict(axes=0), {}), (capi.EINVAL, dict(axes=5), {}),
                            (capi.EINVAL, dict(axis_stride=2), {}), (capi.EINVAL, dict(sections=(24, 20, 19, 0)), {}),
                            (capi.EINVAL, dict(sections=(84, -20, 0, 0)), {}),
                            (capi.EINVAL, dict(sections=(20, 22, 22, 0)), {}), (capi.EINVAL, {}, dict(rot=0)),
                            (capi.EINVAL, {}, dict(positions=None)), (capi.EALIGN, {}, dict(positions=P + 4)),
                            (capi.EALIGN, {}, dict(sin=P + 4)), (capi.EINVAL, {}, dict(q_out=None)),
                            (capi.OK, dict(mixed=0, sections=(20, 22, 22, 0)), dict(tokens=0)), (capi.OK, {}, dict(tokens=0))):
        m = {**mrope, **kw}
        m["sections"] = (ctypes.c_int32 * 4)(*m["sections"])
        call = capi.KV8MropeArgs(rope=capi.KV8RopeArgs(**{**rope, **inner}), **m)
        assert lib.rf_kv8_qk_norm_mrope(ref(call), None) == want, (kw, inner)
    assert lib.rf_kv8_qk_norm_mrope(None, None) == capi.EINVAL
