"""examples/paged_qwen3.py with a scaled rotation (YaRN: cos and sin times a factor)
against the loaded model's own attention, in the bounds of
test_gpu_paged_example.py (MI355X only)."""
from __future__ import annotations

import pytest
import torch

transformers = pytest.importorskip("transformers")

from rhinoforge_amd.quant import convert, load  # noqa: E402
from ckpt_util import write_source  # noqa: E402
from test_gpu_paged_example import DEV, _close, _example, _last_logits, _prompts  # noqa: E402

pytestmark = pytest.mark.gpu


@torch.no_grad()
@pytest.mark.parametrize("factor", [4.0, 16.0])
def test_logits_with_a_yarn_table(factor, tmp_path):
    write_source(tmp_path / "src", seed=11, vocab_size=1000, hidden_size=256, intermediate_size=704,
                 num_attention_heads=8, num_key_value_heads=2, head_dim=64, max_position_embeddings=512,
                 rope_parameters={"rope_type": "yarn", "factor": factor, "rope_theta": 1e6,
                                  "original_max_position_embeddings": int(512 / factor)})
    convert.convert_checkpoint(tmp_path / "src", tmp_path / "dst", quant_lm_head=True, log=lambda *a: None)
    model = load.load_w8a16_model(None, tmp_path / "dst", device=DEV)
    assert model.model.rotary_emb.attention_scaling > 1.1
    paged = _example().PagedQwen3(model, num_blocks=64, block_size=32)
    prompts = _prompts([1, 77, 300, 32])
    i32 = dict(dtype=torch.int32, device=DEV)
    table, zero = torch.full((4, 12), -1, **i32), torch.zeros(4, **i32)
    lens = torch.tensor([len(p) for p in prompts], **i32)
    flat = torch.tensor([t for p in prompts for t in p], device=DEV)
    logits, plan = paged.logits(flat, table, zero, lens, torch.zeros(1, **i32), 300)
    _close(logits, _last_logits(model, prompts))
    token = logits.argmax(-1)
    more, _ = paged.logits(token, table, plan.kv_lens, torch.ones(4, **i32), plan.free_next, 1)
    _close(more, _last_logits(model, [p + [t] for p, t in zip(prompts, token.tolist())]))
