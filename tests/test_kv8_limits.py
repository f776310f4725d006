"""CPU tests of the int8 paged cache: layouts that KV8Cache takes, and operands that
the C ABI refuses."""
from __future__ import annotations

import ctypes

import pytest
import torch

import rhinoforge_amd as rf
from rhinoforge_amd import capi


@pytest.mark.parametrize("form", ["transposed", "strided", "broadcast"])
def test_from_quantized_of_scales_that_are_not_contiguous(form):
    nb, hk = 5, 3
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randint(-127, 128, (nb, hk, 32, 64), dtype=torch.int8, generator=g) for _ in range(2))
    if form == "transposed":
        s = torch.rand(hk, nb, generator=g).t()
    elif form == "strided":
        s = torch.rand(nb, 2 * hk, generator=g)[:, ::2]
    else:
        s = torch.rand(nb, 1, generator=g).expand(nb, hk)
    c = rf.KV8Cache.from_quantized(k, s, v, s)
    assert c.k_scale.is_contiguous() and c.v_scale.is_contiguous()
    assert torch.equal(c.k_scale, s) and torch.equal(c.v_scale, s)
    assert c.k_scale.data_ptr() != s.data_ptr()
    # every op takes the cache as far as there is something to run on
    slots = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        rf.kv8_read(c, slots)
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        rf.kv8_append(c, torch.zeros(1, hk, 64).half(), torch.zeros(1, hk, 64).half(), slots)
    # and its own way back
    assert all(torch.equal(a, b) for a, b in zip(c.to_quantized(), (k, s, v, s)))


# ---- the C ABI: rf_kv8_plan's outputs apart from its inputs ---------------------------

IN = {"cached": 5, "fresh": 5, "free_blocks": 9, "free_start": 1}    # elements, for 5 requests
OUT = {"slots": 40, "positions": 40, "cu": 6, "kv_lens": 5, "free_next": 1}


def _plan(**at):
    """The status of a call whose arrays are at made-up addresses, 4 KB apart."""
    names = ["block_table", *IN, *OUT]
    where = {n: (1 << 20) + 4096 * i for i, n in enumerate(names)}
    a = capi.KV8PlanArgs(**{**where, **at}, requests=5, width=3, table_stride=3, num_free=9, tokens=40,
                         block_size=32)
    if at == {}:
        return where
    return capi.load().rf_kv8_plan(ctypes.byref(a), None)


@pytest.mark.parametrize("out", sorted(OUT))
@pytest.mark.parametrize("inp", sorted(IN))
def test_plan_refuses_outputs_over_its_inputs(out, inp):
    """A workgroup may read an input after another has written its outputs."""
    where = _plan()
    assert _plan(**{out: where[inp]}) == capi.EINVAL
    assert _plan(**{out: where[inp] + 4 * (IN[inp] - 1)}) == capi.EINVAL
    assert _plan(**{out: where[inp] - 4 * (OUT[out] - 1)}) == capi.EINVAL


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are made up: nothing may run on them")
@pytest.mark.parametrize("out", sorted(OUT))
@pytest.mark.parametrize("inp", sorted(IN))
def test_plan_takes_outputs_right_beside_its_inputs(out, inp):
    """Refused later, for want of a device."""
    where = _plan()
    assert _plan(**{out: where[inp] + 4 * IN[inp]}) not in (capi.OK, capi.EINVAL)
    assert _plan(**{out: where[inp] - 4 * OUT[out]}) not in (capi.OK, capi.EINVAL)
