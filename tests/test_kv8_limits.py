"""CPU tests of the int8 paged cache: layouts that KV8Cache takes, and sizes that the
C ABI takes or refuses."""
from __future__ import annotations

import pytest
import torch

import rhinoforge_amd as rf


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
