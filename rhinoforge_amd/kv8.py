"""Attention over an int8 paged cache: what a decoder layer does between its
q/k/v projections and its o projection (``torch.ops.kv8``, csrc/kv8_*).

The reference runs these steps inside its fused decoder (head norms, RoPE, KV
insert, SDPA: src/fused/rpu_qwen3_model.h:3310-3517).  Here they are five ops
that share one cache:

* :func:`qk_norm_rope`   head norms and position rotation of q and k, one launch;
* :func:`kv8_plan`       block tables, slots and positions from request lengths;
* :func:`kv8_append`     quantizes new keys and values into the cache;
* :func:`kv8_attention`  ragged batches of single tokens, drafted tokens or prompts;
* :func:`kv8_read`       cached tokens as the values they stand for.

Everything runs on the current HIP stream, without synchronization, and can be
captured into a graph.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

# (resolved once: single-token calls are bound by the host)
_ops = torch.ops.kv8
_qk_norm_rope, _plan, _append = _ops.qk_norm_rope.default, _ops.plan.default, _ops.append.default
_read, _attention = _ops.read.default, _ops.attention.default

GROUP = 32          # tokens of one group of tiles
BLOCK_SIZES = (32, 64, 128)
HEAD_DIMS = (64, 128, 256)


class KV8Plan(NamedTuple):
    """What :func:`kv8_plan` gives, all int32 on the device."""
    slots: torch.Tensor      # [num_tokens]
    positions: torch.Tensor  # [num_tokens]
    cu_new: torch.Tensor     # [requests + 1]
    kv_lens: torch.Tensor    # [requests]
    free_next: torch.Tensor  # [1]


class KV8Cache:
    """The int8 cache of one decoder layer: ``num_blocks`` blocks of
    ``block_size`` tokens, each with one fp32 scale per key/value head for keys
    and one for values (``x = q * scale``, q in [-127, 127]).

    ``k`` and ``v`` hold the values in the kernels' tile order (uint8
    ``[num_blocks, kv_heads, block_size / 32, head_dim / 32, 1024]``, see
    include/kv8.h); :meth:`to_quantized` and :meth:`from_quantized` convert to
    and from row-major int8 ``[num_blocks, kv_heads, block_size, head_dim]``.
    Scales are zero or positive; :func:`kv8_attention` gives NaN to queries that
    see tokens of a block whose scale is negative, infinite or NaN.
    """

    def __init__(self, num_blocks: int, kv_heads: int, head_dim: int, block_size: int = 64, *,
                 device="cuda") -> None:
        if block_size not in BLOCK_SIZES:
            raise ValueError(f"block_size must be one of {BLOCK_SIZES}, got {block_size}")
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        if num_blocks < 1 or kv_heads < 1:
            raise ValueError("num_blocks and kv_heads must be at least 1")
        if num_blocks * block_size > 0x7fffffff:
            raise ValueError("the cache's slots must fit int32")
        shape = (num_blocks, kv_heads, block_size // GROUP, head_dim // 32, 1024)
        self.k = torch.full(shape, 128, dtype=torch.uint8, device=device)
        self.v = torch.full(shape, 128, dtype=torch.uint8, device=device)
        self.k_scale = torch.zeros(num_blocks, kv_heads, dtype=torch.float32, device=device)
        self.v_scale = torch.zeros_like(self.k_scale)

    num_blocks = property(lambda self: self.k.size(0))
    kv_heads = property(lambda self: self.k.size(1))
    block_size = property(lambda self: self.k.size(2) * GROUP)
    head_dim = property(lambda self: self.k.size(3) * 32)
    device = property(lambda self: self.k.device)

    def tensors(self):
        """(k, v, k_scale, v_scale), as the ops of ``torch.ops.kv8`` take them."""
        return self.k, self.v, self.k_scale, self.v_scale

    @classmethod
    def from_quantized(cls, k: torch.Tensor, k_scale: torch.Tensor, v: torch.Tensor,
                       v_scale: torch.Tensor) -> "KV8Cache":
        """A cache of row-major int8 k, v [num_blocks, kv_heads, block_size, head_dim]
        and fp32 scales [num_blocks, kv_heads]; -128 is taken as -127."""
        if k.dtype != torch.int8 or v.dtype != torch.int8 or k.dim() != 4 or k.shape != v.shape:
            raise ValueError("k and v must be int8 [num_blocks, kv_heads, block_size, head_dim], "
                             f"got {k.dtype} {list(k.shape)} and {v.dtype} {list(v.shape)}")
        for s in (k_scale, v_scale):
            if s.dtype != torch.float32 or s.shape != k.shape[:2]:
                raise ValueError(f"scales must be float32 {list(k.shape[:2])}, got {s.dtype} {list(s.shape)}")
        nb, heads, bs, d = k.shape
        c = cls.__new__(cls)
        if bs not in BLOCK_SIZES or d not in HEAD_DIMS:
            raise ValueError(f"block_size must be one of {BLOCK_SIZES} and head_dim one of "
                             f"{HEAD_DIMS}, got {bs} and {d}")
        # k: token 32 gr + 16 tt + l, dimension 64 kb + 16 g + j
        t = k.clamp(min=-127).view(torch.uint8).bitwise_xor_(0x80)
        t = t.view(nb, heads, bs // 32, 2, 16, d // 64, 4, 16).permute(0, 1, 2, 3, 5, 6, 4, 7)
        c.k = t.reshape(nb, heads, bs // 32, d // 32, 1024).contiguous()
        # v: token 32 gr + 16 h + 4 g + c, dimension 32 dt + 16 e + l
        t = v.clamp(min=-127).view(torch.uint8).bitwise_xor_(0x80)
        t = t.view(nb, heads, bs // 32, 2, 4, 4, d // 32, 2, 16).permute(0, 1, 2, 6, 4, 8, 7, 3, 5)
        c.v = t.reshape(nb, heads, bs // 32, d // 32, 1024).contiguous()
        # (a clone alone would keep a transposed tensor's strides)
        c.k_scale, c.v_scale = (s.clone(memory_format=torch.contiguous_format) for s in (k_scale, v_scale))
        return c

    def to_quantized(self):
        """(k, k_scale, v, v_scale) with k and v row-major int8, as
        :meth:`from_quantized` takes them."""
        nb, heads, gr, dt, _ = self.k.shape
        t = self.k.bitwise_xor(0x80).view(nb, heads, gr, 2, dt // 2, 4, 16, 16)
        k = t.permute(0, 1, 2, 3, 6, 4, 5, 7).reshape(nb, heads, gr * 32, dt * 32)
        t = self.v.bitwise_xor(0x80).view(nb, heads, gr, dt, 4, 16, 2, 2, 4)
        v = t.permute(0, 1, 2, 7, 4, 8, 3, 6, 5).reshape(nb, heads, gr * 32, dt * 32)
        return (k.contiguous().view(torch.int8), self.k_scale.clone(),
                v.contiguous().view(torch.int8), self.v_scale.clone())

    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """:func:`kv8_append` into this cache."""
        kv8_append(self, k, v, slots)

    def read(self, slots: torch.Tensor, dtype: torch.dtype = torch.float16):
        """:func:`kv8_read` from this cache."""
        return kv8_read(self, slots, dtype)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor | None,
                 k_weight: torch.Tensor | None, cos: torch.Tensor | None, sin: torch.Tensor | None,
                 positions: torch.Tensor | None = None, *, eps: float = 1e-6,
                 interleaved: bool = False):
    """RMS norm of each query and key head, then the position rotation.

    q [tokens, heads, head_dim], k [tokens, kv_heads, head_dim], fp16 or bf16
    (views of the projections' outputs are read in place); weights [head_dim]
    of that type or None (no norm).  cos, sin: fp32 [rows, rot / 2], rot a
    multiple of 16 up to head_dim (the first rot dimensions of a head are
    rotated), or None (no rotation).  Token t uses row ``positions[t]`` (int32
    or int64), or row t without positions; a position outside the table gives
    NaN.  Pairs are (i, i + rot / 2), with ``interleaved`` (2i, 2i + 1).
    fp32 throughout, one rounding.  Returns new contiguous (q, k).
    """
    return _qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)


def rope_table(inv_freq: torch.Tensor, rows: int):
    """(cos, sin) fp32 [rows, rot / 2] of positions 0 .. rows - 1 for
    :func:`qk_norm_rope`, from angles in fp64."""
    angle = torch.arange(rows, device=inv_freq.device, dtype=torch.float64)[:, None] * inv_freq.double()
    return angle.cos().float(), angle.sin().float()


def kv8_plan(block_table: torch.Tensor, cached_lens: torch.Tensor, new_lens: torch.Tensor,
             free_blocks: torch.Tensor, free_start: torch.Tensor, num_tokens: int,
             block_size: int) -> KV8Plan:
    """Block tables and slots of a batch from its lengths, in one launch.

    All tensors int32 on the device.  Request i holds ``cached_lens[i]`` tokens
    and gets ``new_lens[i]`` more; the blocks it lacks are taken from
    ``free_blocks`` in order, from index ``free_start[0]`` on, and entered into
    ``block_table[i]`` (in place).  ``num_tokens``: the batch's new tokens, or
    more (a captured graph's fixed size): slots past them are -1.

    ``free_next[0] > free_blocks.numel()`` says that the blocks ran out; tokens
    without a block have slot -1, which :func:`kv8_append` skips.
    """
    return KV8Plan(*_plan(block_table, cached_lens, new_lens, free_blocks, free_start, num_tokens,
                          block_size))


def kv8_append(cache: KV8Cache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantizes k, v [tokens, kv_heads, head_dim] (fp16 or bf16) into
    ``slots`` [tokens] (int32, slot = block * block_size + token in the block;
    negative or past the cache: skipped).

    A block's scale is the largest magnitude it holds over 127: where new
    tokens raise it, the block's earlier tokens are rounded again to the new
    step.  The new tokens of one block must be consecutive slots and
    consecutive in the batch, as :func:`kv8_plan` makes them.  A block that
    gets an infinity or NaN reads back as NaN (that head, k or v).
    """
    _append(*cache.tensors(), k, v, slots)


def kv8_read(cache: KV8Cache, slots: torch.Tensor, dtype: torch.dtype = torch.float16):
    """Cached tokens as values: (k, v), each [n, kv_heads, head_dim] of fp16,
    bf16 or fp32, for int32 ``slots`` [n]; a slot outside the cache gives zeros."""
    return _read(*cache.tensors(), slots, dtype)


def kv8_attention(q: torch.Tensor, cache: KV8Cache, block_table: torch.Tensor,
                  kv_lens: torch.Tensor, cu_q: torch.Tensor | None = None, *, max_q_len: int = 0,
                  max_kv_len: int = 0, causal: bool = True, window: int = 0,
                  scale: float | None = None, return_lse: bool = False):
    """softmax(scale q k^T) v over the cache, for a ragged batch.

    q [tokens, heads, head_dim] fp16 or bf16, heads a multiple of the cache's;
    request i's queries are tokens ``cu_q[i] .. cu_q[i + 1] - 1`` (int32
    [requests + 1]; None: the same number each) and are the last of its
    ``kv_lens[i]`` cached tokens, whose blocks ``block_table[i]`` lists.
    ``causal``: a query sees the tokens up to its own; ``window`` > 0: only the
    last ``window`` of those.  A query that sees none gives zeros and a
    log-sum-exp of -inf; a block id outside the cache gives NaN.  Tokens past
    ``cu_q[-1]`` give zeros.

    ``max_q_len`` and ``max_kv_len``: the largest of the batch where the caller
    knows them; they choose the launch, never the result's meaning.  ``scale``
    defaults to head_dim ** -0.5.  Returns out [tokens, heads, head_dim] in q's
    type, with ``return_lse`` also the natural log-sum-exp, fp32 [tokens, heads].
    """
    scale = cache.head_dim ** -0.5 if scale is None else scale
    out, lse = _attention(q, *cache.tensors(), block_table, kv_lens, cu_q, max_q_len, max_kv_len,
                          causal, window, scale, return_lse)
    return (out, lse) if return_lse else out
