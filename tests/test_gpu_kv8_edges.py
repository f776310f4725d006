"""The int8 paged cache's ops at the edges of what they accept (MI355X only)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import rhinoforge_amd as rf
from oracle import kv8 as o

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _rng(seed):
    return torch.Generator().manual_seed(seed)


def _np(t):
    return t.detach().cpu().double().numpy()


# ---- norms and rotation: values that are not finite --------------------------------

@pytest.mark.parametrize("d,rot", [(128, 64), (128, 128), (64, 16), (40, 0), (256, 128), (512, 256), (80, 48)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_rotation_beside_values_that_are_not_finite(d, rot, interleaved, dt, bad):
    """One such value in each token, at every dimension in turn: it reaches its own
    pair, or where it is not rotated nothing else, bit for bit."""
    x = torch.randn(d, 2, d, generator=_rng(d + rot)).to(dt)
    for t in range(d):
        x[t, t % 2, t] = bad
    cos = sin = None
    if rot:
        angle = torch.rand(d, rot // 2, generator=_rng(rot)) * 6 + 0.1
        cos, sin = angle.cos(), angle.sin()
    on = lambda v: None if v is None else v.to(DEV)  # noqa: E731
    got = rf.qk_norm_rope(x.to(DEV), x[:, :1].contiguous().to(DEV), None, None, on(cos), on(sin),
                          interleaved=interleaved)
    for y, part in ((got[0], x), (got[1], x[:, :1])):
        y = y.cpu()
        assert torch.equal(y[..., rot:].view(torch.int16), part[..., rot:].contiguous().view(torch.int16)) \
            or (bad != bad and torch.equal(y[..., rot:].isnan(), part[..., rot:].isnan())
                and torch.equal(y[..., rot:].nan_to_num(), part[..., rot:].nan_to_num()))
        with np.errstate(invalid="ignore"):
            ref = o.norm_rope(_np(part), None, None if cos is None else _np(cos), None if sin is None else _np(sin),
                              None, 0.0, interleaved)
        assert np.array_equal(np.isnan(_np(y)), np.isnan(ref))
        assert np.array_equal(np.isinf(_np(y)) * np.sign(np.nan_to_num(_np(y))),
                              np.isinf(ref) * np.sign(np.nan_to_num(ref)))
        fin = np.isfinite(ref)
        assert (np.abs(_np(y)[fin] - ref[fin]) <= UNIT[dt] * np.abs(ref[fin]) + 2.0 ** -20).all()


def test_norm_beside_values_that_are_not_finite():
    """An infinity makes its head's mean infinite: 0 for the finite values that are
    not rotated, NaN for itself; other heads keep theirs."""
    d, rot = 128, 64
    x = torch.randn(3, 2, d, generator=_rng(0)).half()
    x[0, 0, 100] = float("inf")
    x[1, 1, 3] = float("nan")
    w = torch.ones(d, dtype=torch.float16)
    angle = torch.rand(3, rot // 2, generator=_rng(1))
    y, _ = (t.cpu() for t in rf.qk_norm_rope(x.to(DEV), x.to(DEV), w.to(DEV), None, angle.cos().to(DEV),
                                             angle.sin().to(DEV)))
    want = torch.zeros(d)
    want[100] = float("nan")
    assert torch.equal(y[0, 0].isnan(), want.isnan()) and (y[0, 0].nan_to_num() == 0).all()
    assert y[1, 1].isnan().all()
    assert y[0, 1].isfinite().all() and y[1, 0].isfinite().all() and y[2].isfinite().all()


# ---- windows of every size -----------------------------------------------------------

@pytest.mark.parametrize("window", [2 ** 31, 2 ** 40, 2 ** 63 - 1])
def test_a_window_past_every_length_launches_as_none(window):
    """The same launch, so the same bits, for one token behind a long context."""
    hk, d, n = 2, 128, 20000
    cache = rf.KV8Cache(320, hk, d, 64)
    kv = torch.randn(n, hk, d, generator=_rng(0)).half().to(DEV)
    cache.append(kv, kv.flip(0), torch.arange(n, dtype=torch.int32, device=DEV))
    q = torch.randn(1, 8, d, generator=_rng(1)).half().to(DEV)
    table = torch.arange(320, dtype=torch.int32, device=DEV)[None]
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    want = rf.kv8_attention(q, cache, table, lens, return_lse=True)
    got = rf.kv8_attention(q, cache, table, lens, window=window, return_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
