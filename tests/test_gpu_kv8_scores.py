"""Attention over the int8 cache where a score's factor is very small or zero: the
decode and the prefill kernel against the same bound (MI355X only)."""
from __future__ import annotations

import pytest
import torch

from test_gpu_kv8_scales import DEV, SHAPES, _check, _made, _on

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scale", [1e-44, 1e-38, 1e-20])
def test_a_scale_that_leaves_nothing_of_the_scores(shape, dt, scale):
    """Every score is 0 to any precision: the mean of what a row sees."""
    print("scale", shape, dt, scale, flush=True)
    q, cache, table = _made(shape, dt, 11)
    _check(q.to(DEV), _on(cache), table, [shape[0]], [shape[1]], scale=scale)


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("low", [2.0 ** -115, 2.0 ** -125, 2.0 ** -133])
def test_bf16_query_rows_near_the_least_magnitude(shape, low):
    print("rows", shape, low, flush=True)
    q, (kq, ks, vq, vs), table = _made(shape, torch.bfloat16, 12)
    q[::3] = (q[::3].double() * low).bfloat16()
    q[:, ::5] = 0
    ks = ks * 2.0 ** -4
    _check(q.to(DEV), _on((kq, ks, vq, vs)), table, [shape[0]], [shape[1]])


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("least", [0.0, 2.0 ** -140, 2.0 ** -107])
def test_key_scales_of_zero_or_nearly(shape, least):
    """A key scale of 0 makes the keys 0 whatever the bytes."""
    print("key scales", shape, least, flush=True)
    q, (kq, ks, vq, vs), table = _made(shape, torch.float16, 13)
    ks[table[0, 1::3]] = least
    _check(q.to(DEV), _on((kq, ks, vq, vs)), table, [shape[0]], [shape[1]])


@pytest.mark.parametrize("size", [1e-37, 1e-20, 1e20, 1e30])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_bf16_queries_past_the_range_of_fp16_in_both_kernels(shape, size):
    print("range", shape, size, flush=True)
    q, cache, table = _made(shape, torch.bfloat16, 14)
    q = (q.double() * size).bfloat16()
    _check(q.to(DEV), _on(cache), table, [shape[0]], [shape[1]], scale=1.0 / size)
