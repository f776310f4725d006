"""Operands of the int8 paged cache's ops in layouts that the kernels do not read in
place (MI355X only): strides that are not multiples of eight, innermost strides
other than one, addresses that are not multiples of 16."""
from __future__ import annotations

import pytest
import torch

import rhinoforge_amd as rf

pytestmark = pytest.mark.gpu
DEV = "cuda"

FORMS = ["odd stride", "unit stride elsewhere", "off by one value", "broadcast"]


def _laid_out(x, form):
    """x [tokens, heads, d] in another layout, same values."""
    t, h, d = x.shape
    if form == "odd stride":
        y = torch.zeros(t, h, d + 3, dtype=x.dtype, device=DEV)[..., 1:d + 1]
    elif form == "unit stride elsewhere":
        y = torch.zeros(t, d, h, dtype=x.dtype, device=DEV).transpose(1, 2)
    elif form == "off by one value":
        y = torch.zeros(t * h * d + 1, dtype=x.dtype, device=DEV)[1:].view(t, h, d)
    else:
        y = x[:1].expand(t, h, d)
        return y
    y.copy_(x)
    return y


def _shifted(x):
    """A contiguous copy one element past a 16-byte boundary."""
    y = torch.zeros(x.numel() + 1, dtype=x.dtype, device=DEV)[1:].view(x.shape)
    return y.copy_(x)


def _made(t, h, d, seed):
    return torch.randn(t, h, d, generator=torch.Generator().manual_seed(seed)).half().to(DEV)


@pytest.mark.parametrize("form", FORMS)
def test_norm_rope(form):
    q, k = _laid_out(_made(7, 4, 128, 0), form), _laid_out(_made(7, 2, 128, 1), form)
    w = torch.rand(128, generator=torch.Generator().manual_seed(2)).half().to(DEV)
    angle = torch.rand(7, 32, generator=torch.Generator().manual_seed(3)).to(DEV)
    cos, sin = angle.cos(), angle.sin()
    want = rf.qk_norm_rope(q.clone(memory_format=torch.contiguous_format),
                           k.clone(memory_format=torch.contiguous_format), w, w, cos, sin)
    got = rf.qk_norm_rope(q, k, _shifted(w), _shifted(w), _shifted(cos), _shifted(sin))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("tokens", [3, 45])
def test_append(form, tokens):
    k, v = _laid_out(_made(tokens, 2, 64, 4), form), _laid_out(_made(tokens, 2, 64, 5), form)
    slots = torch.arange(30, 30 + tokens, dtype=torch.int32, device=DEV)
    a, b = rf.KV8Cache(4, 2, 64, 32), rf.KV8Cache(4, 2, 64, 32)
    a.append(k, v, _shifted(slots))
    b.append(k.clone(memory_format=torch.contiguous_format), v.clone(memory_format=torch.contiguous_format), slots)
    for x, y in zip(a.tensors(), b.tensors()):
        assert torch.equal(x, y)
    for x, y in zip(a.read(_shifted(slots)), b.read(slots)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("tokens,heads", [(2, 4), (90, 32)])
def test_attention(form, tokens, heads):
    cache = rf.KV8Cache(5, 2, 128, 32)
    cache.append(_made(150, 2, 128, 6), _made(150, 2, 128, 7), torch.arange(150, dtype=torch.int32, device=DEV))
    q = _laid_out(_made(tokens, heads, 128, 8), form)
    table = torch.arange(5, dtype=torch.int32, device=DEV)[None]
    lens = torch.tensor([150], dtype=torch.int32, device=DEV)
    want = rf.kv8_attention(q.clone(memory_format=torch.contiguous_format), cache, table, lens)
    assert torch.equal(rf.kv8_attention(q, cache, _shifted(table), _shifted(lens)), want)


def test_plan_of_operands_off_by_one_value():
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    table = torch.full((3, 4), -1, dtype=torch.int32, device=DEV)
    cached, new, free, start = i32(5, 0, 60), i32(40, 3, 1), i32(9, 8, 7, 6, 5, 4), i32(1)
    table[0, 0], table[2, :2] = 2, i32(0, 1)
    other = _shifted(table)
    a = rf.kv8_plan(table, cached, new, free, start, 44, 32)
    b = rf.kv8_plan(other, _shifted(cached), _shifted(new), _shifted(free), _shifted(start), 44, 32)
    assert torch.equal(table, other)
    for x, y in zip(a, b):
        assert torch.equal(x, y)
