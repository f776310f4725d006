"""Tensors of the paged caches' ops that are not on the device of the others: refused with
the argument's name, before anything is allocated or launched (MI355X only)."""
from __future__ import annotations

import pytest
import torch

import rhinoforge_amd as rf

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _calls():
    """name -> (op, arguments, which of them are tensors)."""
    c4, c8 = rf.KV4Cache(2, 2, 64, 32, device=DEV), rf.KV8Cache(2, 2, 64, 32, device=DEV)
    q, kv = (torch.zeros(3, h, 64, dtype=torch.float16, device=DEV) for h in (4, 2))
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    cos, pos, w = torch.ones(4, 32, device=DEV), i32(0, 1, 2).expand(3, 3).contiguous(), torch.ones(64, device=DEV).half()
    tail = (i32(0, 1)[None], i32(3), i32(0, 3), 3, 3, True, 0, 0.1, True)
    ops = torch.ops
    calls = {
        "kv4 append": (ops.kv4.append, (*c4.tensors(), kv, kv, i32(0, 1, 2))),
        "kv4 read": (ops.kv4.read, (*c4.tensors(), i32(0, 1, 2), torch.float16)),
        "kv4 attention": (ops.kv4.attention, (q, *c4.tensors(), *tail)),
        "kv8 append": (ops.kv8.append, (*c8.tensors(), kv, kv, i32(0, 1, 2))),
        "kv8 read": (ops.kv8.read, (*c8.tensors(), i32(0, 1, 2), torch.float16)),
        "kv8 attention": (ops.kv8.attention, (q, *c8.tensors(), *tail)),
        "mrope": (ops.rope.qk_norm_mrope, (q, kv, w, w, cos, cos, pos, [12, 10, 10], True, 1e-6, False)),
    }
    return calls


CASES = [(n, i) for n, k in (("kv4 append", 6), ("kv4 read", 4), ("kv4 attention", 7), ("kv8 append", 7), ("kv8 read", 5),
                             ("kv8 attention", 8), ("mrope", 7)) for i in range(k)]


@pytest.mark.parametrize("name,at", CASES)
def test_a_tensor_on_the_host_among_tensors_on_the_device(name, at):
    print("refused", name, at, flush=True)
    op, args = _calls()[name]
    op(*args)
    args = list(args)
    args[at] = args[at].cpu()
    with pytest.raises(RuntimeError, match=r"(kv4|kv8|rope)::\w+: .* must be on"):
        op(*args)
