"""examples/paged_qwen3.py on the CPU: the rotation table it builds from a model."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

transformers = pytest.importorskip("transformers")

from ckpt_util import tiny_config  # noqa: E402

PATH = Path(__file__).resolve().parents[1] / "examples" / "paged_qwen3.py"

ROPES = {
    "default": {"rope_type": "default", "rope_theta": 1e6},
    "linear": {"rope_type": "linear", "factor": 2.0, "rope_theta": 1e6},
    "dynamic": {"rope_type": "dynamic", "factor": 2.0, "rope_theta": 1e6},
    "yarn": {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32, "rope_theta": 1e6},
    "yarn, its own factor": {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32,
                             "rope_theta": 1e6, "attention_factor": 0.7},
    "llama3": {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
               "original_max_position_embeddings": 32, "rope_theta": 1e6},
}


def _paged(rope):
    spec = importlib.util.spec_from_file_location("paged_qwen3", PATH)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    torch.manual_seed(0)
    model = transformers.Qwen3ForCausalLM(tiny_config(head_dim=64, rope_parameters=rope)).eval()
    return model, mod.PagedQwen3(model, num_blocks=2, block_size=32)


@pytest.mark.parametrize("name", sorted(ROPES))
def test_the_table_is_the_models(name):
    """cos and sin of every position as the model's own rotary embedding gives them:
    its angles are fp32 products of up to 127, off by 2^-18 at most."""
    model, paged = _paged(ROPES[name])
    cos, sin = model.model.rotary_emb(torch.zeros(1, 1, 64), torch.arange(128)[None])
    for mine, theirs in ((paged.cos, cos), (paged.sin, sin)):
        assert mine.shape == (128, 32) and mine.dtype == torch.float32
        assert (mine - theirs[0, :, :32]).abs().max() <= 2.0 ** -16


def test_a_table_that_changes_with_the_length_is_refused():
    with pytest.raises(ValueError, match="longrope"):
        _paged({"rope_type": "longrope", "factor": 4.0, "short_factor": [1.0] * 32, "long_factor": [2.0] * 32,
                "original_max_position_embeddings": 32, "rope_theta": 1e6})
