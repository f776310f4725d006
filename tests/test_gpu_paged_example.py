"""examples/paged_qwen3.py: a W8A16 Qwen3 checkpoint over the int8 paged cache,
against the same loaded model's own attention in fp16 (MI355X only).

An int8 value differs from its key or value by at most half a step, amax / 254
(uniform: 0.23% of amax, about 0.9% of the rms), so scores of unit-norm heads move by
about 1% and outputs by as much before the residual stream dilutes it: logits
within 3% of their rms per row (l2), cos >= 0.999.  A greedy token equals the
model's argmax where that leads the runner-up by more than four times the row's
largest logit error.
"""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

transformers = pytest.importorskip("transformers")

import rhinoforge_amd as rf  # noqa: E402
from rhinoforge_amd.quant import convert, load  # noqa: E402
from ckpt_util import write_source  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"
PATH = Path(__file__).resolve().parents[1] / "examples" / "paged_qwen3.py"


def _example():
    spec = importlib.util.spec_from_file_location("paged_qwen3", PATH)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.fixture(scope="module", params=[64, 128])
def model(request, tmp_path_factory):
    root = tmp_path_factory.mktemp(f"paged_{request.param}")
    write_source(root / "src", seed=11, vocab_size=1000, hidden_size=256, intermediate_size=704,
                 num_attention_heads=8, num_key_value_heads=2, head_dim=request.param,
                 max_position_embeddings=512)
    convert.convert_checkpoint(root / "src", root / "dst", quant_lm_head=True, log=lambda *a: None)
    return load.load_w8a16_model(None, root / "dst", device=DEV)


def _prompts(lens, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 1000, (n,), generator=g).tolist() for n in lens]


def _last_logits(model, rows):
    return torch.stack([model(torch.tensor([r], device=DEV)).logits[0, -1].float() for r in rows])


def _close(got, ref):
    got, ref = got.double(), ref.double()
    rel = ((got - ref).norm(dim=-1) / ref.norm(dim=-1)).max().item()
    cos = torch.nn.functional.cosine_similarity(got, ref, dim=-1).min().item()
    print(f"  rel {rel:.4f} cos {cos:.6f}", flush=True)
    assert rel <= 0.03 and cos >= 0.999


@torch.no_grad()
def test_logits_of_a_ragged_batch(model):
    ex = _example()
    paged = ex.PagedQwen3(model, num_blocks=64, block_size=32)
    prompts = _prompts([1, 77, 130, 32, 33])
    i32 = dict(dtype=torch.int32, device=DEV)
    table = torch.full((5, 8), -1, **i32)
    zero, start = torch.zeros(5, **i32), torch.zeros(1, **i32)
    lens = torch.tensor([len(p) for p in prompts], **i32)
    flat = torch.tensor([t for p in prompts for t in p], device=DEV)
    logits, plan = paged.logits(flat, table, zero, lens, start, 130)
    _close(logits, _last_logits(model, prompts))
    # the first layer's cache holds the model's own keys and values, to half a step
    layer = model.model.layers[0]
    h = layer.input_layernorm(model.model.embed_tokens(flat))
    at = layer.self_attn
    k = at.k_norm(at.k_proj(h).unflatten(-1, (2, -1)))
    cos, sin = model.model.rotary_emb(k, plan.positions[None].long())
    half = k.size(-1) // 2
    turned = torch.cat([-k[..., half:], k[..., :half]], -1)
    k = k.float() * cos[0, :, None].float() + turned.float() * sin[0, :, None].float()
    v = at.v_proj(h).unflatten(-1, (2, -1)).float()
    rk, rv = paged.caches[0].read(plan.slots, torch.float32)
    block = (plan.slots // 32).long()
    for got, want, scale in ((rk, k, paged.caches[0].k_scale), (rv, v, paged.caches[0].v_scale)):
        step = scale[block][..., None]
        assert ((got - want).abs() <= 0.51 * step + 2.0 ** -9 * want.abs().amax()).all()
    # one more token for each, behind the cache
    token = logits.argmax(-1)
    more, plan2 = paged.logits(token, table, plan.kv_lens, torch.ones(5, **i32), plan.free_next, 1)
    assert torch.equal(plan2.kv_lens, lens + 1)
    _close(more, _last_logits(model, [p + [t] for p, t in zip(prompts, token.tolist())]))


@torch.no_grad()
@pytest.mark.parametrize("lens", [[5], [40, 3, 64, 1, 90, 17]])
def test_generate_agrees_with_the_model(model, lens):
    ex = _example()
    paged = ex.PagedQwen3(model, num_blocks=64, block_size=32)
    prompts = _prompts(lens, seed=len(lens))
    out = paged.generate(prompts, 40)
    eager = ex.PagedQwen3(model, num_blocks=64, block_size=32).generate(prompts, 40, graph=False)
    assert torch.equal(out, eager)
    for p, row in zip(prompts, out.tolist()):
        ref = model(torch.tensor([p + row], device=DEV)).logits[0, len(p) - 1:-1].float()
        top = ref.topk(2, -1).values
        sure = top[:, 0] - top[:, 1] > 4 * 0.03 * ref.norm(dim=-1) / ref.size(-1) ** 0.5
        same = ref.argmax(-1).cpu() == torch.tensor(row)
        print(f"  {int(sure.sum())} of 40 sure, {int(same.sum())} the same", flush=True)
        assert (same | ~sure.cpu()).all()


def test_generate_refuses_what_does_not_fit(model):
    paged = _example().PagedQwen3(model, num_blocks=4, block_size=32)
    with pytest.raises(ValueError, match="blocks"):
        paged.generate(_prompts([100, 30]), 10)
    with pytest.raises(ValueError, match="positions"):
        paged.generate(_prompts([500]), 100)
    with pytest.raises(ValueError, match="prompt"):
        paged.generate([[]], 3)
