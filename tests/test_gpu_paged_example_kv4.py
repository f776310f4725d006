"""examples/paged_qwen3.py over the 4-bit paged cache (MI355X only): a pass over a ragged
batch, what its first layer holds, and the captured steps against the eager ones."""
from __future__ import annotations

import pytest
import torch

pytest.importorskip("transformers")

import rhinoforge_amd as rf  # noqa: E402
from test_gpu_paged_example import _example, _prompts, model  # noqa: E402,F401

pytestmark = pytest.mark.gpu
DEV = "cuda"


@torch.no_grad()
def test_a_ragged_batch(model):  # noqa: F811
    paged = _example().PagedQwen3(model, num_blocks=64, block_size=32, bits=4)
    assert all(isinstance(c, rf.KV4Cache) for c in paged.caches)
    prompts = _prompts([1, 77, 130, 32, 33])
    i32 = dict(dtype=torch.int32, device=DEV)
    table, zero = torch.full((5, 8), -1, **i32), torch.zeros(5, **i32)
    lens = torch.tensor([len(p) for p in prompts], **i32)
    flat = torch.tensor([t for p in prompts for t in p], device=DEV)
    logits, plan = paged.logits(flat, table, zero, lens, torch.zeros(1, **i32), 130)
    assert torch.isfinite(logits).all() and torch.equal(plan.kv_lens, lens)
    # the first layer's cache holds the model's own keys and values, to half a step: 1/30
    # of the span from the least (or 0) to the largest (or 0), and 2^-6 more for a step
    # of six mantissa bits; 2^-9 for the rotation in another order
    layer = model.model.layers[0]
    at = layer.self_attn
    h = layer.input_layernorm(model.model.embed_tokens(flat))
    k = at.k_norm(at.k_proj(h).unflatten(-1, (2, -1)))
    cos, sin = model.model.rotary_emb(k, plan.positions[None].long())
    half = k.size(-1) // 2
    turned = torch.cat([-k[..., half:], k[..., :half]], -1)
    k = k.float() * cos[0, :, None].float() + turned.float() * sin[0, :, None].float()
    v = at.v_proj(h).unflatten(-1, (2, -1)).float()
    for got, want in zip(paged.caches[0].read(plan.slots, torch.float32), (k, v)):
        span = want.amax(-1).clamp(min=0) - want.amin(-1).clamp(max=0)
        bound = span[..., None] / 30 * (1 + 2.0 ** -6) + 2.0 ** -9 * want.abs().amax()
        assert ((got - want).abs() <= bound).all()
    more, plan2 = paged.logits(logits.argmax(-1), table, plan.kv_lens, torch.ones(5, **i32), plan.free_next, 1)
    assert torch.isfinite(more).all() and torch.equal(plan2.kv_lens, lens + 1)


@pytest.mark.parametrize("lens", [[5], [40, 3, 64, 1, 90, 17]])
def test_captured_steps_are_the_eager_ones(model, lens):  # noqa: F811
    ex = _example()
    runs = [ex.PagedQwen3(model, num_blocks=64, block_size=32, bits=4).generate(_prompts(lens), 40, graph=g)
            for g in (True, False)]
    assert torch.equal(*runs) and ((runs[0] >= 0) & (runs[0] < 1000)).all()


def test_other_widths_are_refused(model):  # noqa: F811
    with pytest.raises(ValueError, match="bits"):
        _example().PagedQwen3(model, num_blocks=4, bits=5)
