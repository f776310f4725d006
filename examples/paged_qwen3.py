"""Greedy generation with a W8A16 Qwen3 checkpoint over the int8 paged cache.

    python examples/paged_qwen3.py CHECKPOINT --prompts "9707,11,1879" "785,3974" --new 64

``CHECKPOINT`` is a W8A16 directory as ``python -m rhinoforge_amd.quant.convert``
writes it; prompts are token ids.  All prompts run as one ragged batch: one pass
fills the cache, then every step decodes one token for each request.  The decode
step (plan, projections, norms and rotation, append, attention, argmax) depends
on no value on the host, so it is captured once and replayed.
"""
from __future__ import annotations

import argparse
import time

import torch

import rhinoforge_amd as rf
from rhinoforge_amd.quant.load import load_w8a16_model


class PagedQwen3:
    """A loaded model's layers around one :class:`rf.KV8Cache` each."""

    def __init__(self, model, num_blocks: int, block_size: int = 64) -> None:
        cfg = model.config
        self.model, self.block_size = model, block_size
        self.heads, self.kv_heads = cfg.num_attention_heads, cfg.num_key_value_heads
        self.head_dim, self.eps = cfg.head_dim, cfg.rms_norm_eps
        self.device = model.model.norm.weight.device
        self.caches = [rf.KV8Cache(num_blocks, self.kv_heads, self.head_dim, block_size, device=self.device)
                       for _ in model.model.layers]
        rope = model.model.rotary_emb
        if getattr(rope, "rope_type", "default") == "longrope":
            raise ValueError("longrope's frequencies depend on the length of the sequence: one table cannot hold them")
        # (YaRN and its like also scale cos and sin; 1 elsewhere)
        factor = getattr(rope, "attention_scaling", 1.0)
        self.cos, self.sin = (t * factor for t in rf.rope_table(rope.inv_freq.to(self.device),
                                                               cfg.max_position_embeddings))
        self.free = torch.arange(num_blocks, dtype=torch.int32, device=self.device)

    def logits(self, ids, table, cached, new, free_start, max_new: int, max_kv: int = 0):
        """One pass over a ragged batch of new tokens ``ids`` [tokens]: the logits
        of each request's last token, and the pass's plan."""
        m = self.model.model
        plan = rf.kv8_plan(table, cached, new, self.free, free_start, ids.numel(), self.block_size)
        cu = None if max_new == 1 else plan.cu_new
        h = m.embed_tokens(ids)
        for layer, cache in zip(m.layers, self.caches):
            at = layer.self_attn
            projections = (at.q_proj, at.k_proj, at.v_proj)
            q, k, v = rf.linear_multi(layer.input_layernorm(h), [p.weight for p in projections],
                                      [p.weight_scale for p in projections], [p.bias for p in projections])
            q, k, v = (t.unflatten(-1, (n, self.head_dim))
                       for t, n in ((q, self.heads), (k, self.kv_heads), (v, self.kv_heads)))
            q, k = rf.qk_norm_rope(q, k, at.q_norm.weight, at.k_norm.weight, self.cos, self.sin,
                                   plan.positions, eps=self.eps)
            cache.append(k, v, plan.slots)
            o = rf.kv8_attention(q, cache, table, plan.kv_lens, cu, max_q_len=max_new, max_kv_len=max_kv,
                                 window=at.sliding_window or 0, scale=at.scaling)
            h = h + at.o_proj(o.flatten(1))
            h = h + layer.mlp(layer.post_attention_layernorm(h))
        last = h if max_new == 1 else h[plan.cu_new[1:].long() - 1]
        return self.model.lm_head(m.norm(last)), plan

    @torch.no_grad()
    def generate(self, prompts, new_tokens: int, graph: bool = True):
        """Greedy token ids [requests, new_tokens] for lists of prompt ids."""
        dev, b = self.device, len(prompts)
        lens = [len(p) for p in prompts]
        if min(lens) < 1 or new_tokens < 1:
            raise ValueError("every prompt needs a token, and at least one is generated")
        if max(lens) + new_tokens > self.cos.size(0):
            raise ValueError(f"{max(lens) + new_tokens} tokens exceed the model's {self.cos.size(0)} positions")
        longest = max(lens) + new_tokens
        blocks = sum(-(-(n + new_tokens) // self.block_size) for n in lens)
        if blocks > self.free.numel():
            raise ValueError(f"{blocks} blocks needed, the cache has {self.free.numel()}")
        i32 = dict(dtype=torch.int32, device=dev)
        table = torch.full((b, -(-longest // self.block_size)), -1, **i32)
        cached, free_start, one = torch.zeros(b, **i32), torch.zeros(1, **i32), torch.ones(b, **i32)
        out = torch.zeros(b, new_tokens, dtype=torch.long, device=dev)

        ids = torch.tensor([t for p in prompts for t in p], device=dev)
        logits, plan = self.logits(ids, table, cached, torch.tensor(lens, **i32), free_start, max(lens),
                                   max(lens))
        token = logits.argmax(-1)
        out[:, 0] = token
        cached.copy_(plan.kv_lens)
        free_start.copy_(plan.free_next)

        def step():
            logits, plan = self.logits(token, table, cached, one, free_start, 1, longest)
            token.copy_(logits.argmax(-1))
            cached.copy_(plan.kv_lens)
            free_start.copy_(plan.free_next)

        run, done = step, 1
        if graph and new_tokens > 2:
            stream = torch.cuda.Stream()
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                step()                      # (allocations and library handles, before the capture)
                out[:, 1] = token
                done = 2
            torch.cuda.current_stream().wait_stream(stream)
            captured = torch.cuda.CUDAGraph()
            with torch.cuda.graph(captured):
                step()
            run = captured.replay
        for i in range(done, new_tokens):
            run()
            out[:, i] = token
        return out


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("checkpoint")
    ap.add_argument("--prompts", nargs="+", default=["1,2,3"], help="token ids, separated by commas")
    ap.add_argument("--new", type=int, default=32, help="tokens to generate for each prompt")
    ap.add_argument("--blocks", type=int, default=1024, help="blocks of each layer's cache")
    args = ap.parse_args()
    paged = PagedQwen3(load_w8a16_model(None, args.checkpoint), args.blocks)
    prompts = [[int(t) for t in p.split(",")] for p in args.prompts]
    paged.generate(prompts, min(args.new, 4))
    torch.cuda.synchronize()
    begin = time.perf_counter()
    out = paged.generate(prompts, args.new)
    torch.cuda.synchronize()
    took = time.perf_counter() - begin
    for row in out.tolist():
        print(",".join(map(str, row)))
    print(f"{out.numel()} tokens, {out.numel() / took:.1f} tokens/s")


if __name__ == "__main__":
    main()
