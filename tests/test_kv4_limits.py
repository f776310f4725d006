"""What the 4-bit cache takes and promises at the edges, on the CPU."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import rhinoforge_amd as rf
from oracle import kv4 as o


def _parts():
    n = torch.full((1, 1, 32, 64), 3, dtype=torch.uint8)
    step, zero = torch.ones(1, 1, 32, dtype=torch.float16), torch.zeros(1, 1, 32, dtype=torch.uint8)
    return dict(k=n, k_step=step, k_zero=zero, v=n.clone(), v_step=step.clone(), v_zero=zero.clone())


@pytest.mark.parametrize("key_step", [1.0, float("nan")])
@pytest.mark.parametrize("value_step", [1 + 9 * 2.0 ** -10, 1 + 2.0 ** -10, 2.0 ** -21, 5000.0, float("nan"), -1.0])
def test_value_steps_beside_a_key_that_stands_for_nan(key_step, value_step):
    """The mark is the key's: it excuses no value step that the cache cannot hold."""
    p = _parts()
    p["k_step"][0, 0, 5] = key_step
    rf.KV4Cache.from_quantized(**p)
    p["v_step"][0, 0, 5] = value_step
    with pytest.raises(ValueError, match="steps"):
        rf.KV4Cache.from_quantized(**p)


@pytest.mark.parametrize("key_step", [1 + 9 * 2.0 ** -10, 2.0 ** -21, 5000.0])
def test_key_steps_that_the_cache_cannot_hold(key_step):
    p = _parts()
    p["k_step"][0, 0, 5] = key_step
    with pytest.raises(ValueError, match="steps"):
        rf.KV4Cache.from_quantized(**p)


def test_nan_keys_with_any_payload_are_the_mark():
    """A NaN of other low bits is taken, and reads back as the one mark."""
    p = _parts()
    p["k_step"].view(torch.int16)[0, 0, 7] = 0x7fff
    q = rf.KV4Cache.from_quantized(**p).to_quantized()
    assert torch.isnan(q[1][0, 0, 7]) and torch.isnan(q[1]).sum() == 1
    assert all(torch.equal(a, b) for a, b in zip(q[3:], (p["v"], p["v_step"], p["v_zero"])))


def test_half_a_step_is_within_its_bound():
    """At most 1/30 of the span and 2^-6 of that more; steps below 2^-14: 2^-21 more."""
    r = np.random.default_rng(0)
    worst = dict(large=0.0, small=0.0)
    for e in np.concatenate((r.uniform(-30, 16, 4000), np.arange(-30, 17))):
        x = np.sort(r.standard_normal(16)) * 2.0 ** e
        x = x.astype(np.float32).astype(np.float64)
        low, high = min(x[0], 0.0), max(x[-1], 0.0)
        span, step = o.step_of(low, high)
        if span > 65280:
            continue
        small = step < 2.0 ** -14
        bound = span / 30 + 2.0 ** -21 if small else span / 30 * (1 + 2.0 ** -6)
        assert span / 30 <= step / 2 <= bound
        worst["small" if small else "large"] = max(worst["small" if small else "large"], step / 2 / (span / 30))
        n, s, z = o.quantize(x[None])
        assert (np.abs(o.values(n, s, z)[0] - x) <= step / 2).all()
    assert worst["large"] > 1.01 and worst["small"] > 2   # (1/30 of the span alone is no bound)
