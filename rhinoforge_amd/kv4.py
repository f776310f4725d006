"""Attention over a 4-bit paged cache: the int8 paged cache's steps (``kv8.py``) with
keys and values in half the bytes (``torch.ops.kv4``, csrc/kv4_*).

* :func:`kv4_append`     quantizes new keys and values into the cache;
* :func:`kv4_attention`  ragged batches of single tokens, drafted tokens or prompts;
* :func:`kv4_read`       cached tokens as the values they stand for.

Block tables, slots and positions come from :func:`~rhinoforge_amd.kv8.kv8_plan`, norms
and rotation from :func:`~rhinoforge_amd.kv8.qk_norm_rope` or
:func:`~rhinoforge_amd.kv8.qk_norm_mrope`, as for the int8 cache.  Everything runs on
the current HIP stream, without synchronization, and can be captured into a graph.
"""
from __future__ import annotations

import torch

from .kv8 import BLOCK_SIZES, GROUP, HEAD_DIMS

# (resolved once: single-token calls are bound by the host)
_ops = torch.ops.kv4
_append, _read, _attention = _ops.append.default, _ops.read.default, _ops.attention.default

_EMPTY = 0x0010   # the word of the least step, 2^-20, and zero point 0
_NAN = 0x7e00     # the word of a token that stands for NaN
MAX_STEP = 4352.0


class KV4Cache:
    """The 4-bit cache of one decoder layer: ``num_blocks`` blocks of ``block_size``
    tokens.  Each token, key/value head and side (keys, values) holds ``head_dim``
    numbers n of 0..15, a step s and a zero point z of 0..15, and stands for
    ``(n - z) * s``.  Steps are fp16 numbers whose last four mantissa bits are 0, from
    2^-20 to 4352: all of these values are fp16 numbers.

    ``k`` and ``v`` hold the numbers in the kernels' order (uint8 ``[num_blocks,
    kv_heads, block_size / 32, head_dim / 64, 1024]``, see include/kv4.h), ``rows`` the
    steps and zero points (int16 ``[num_blocks, kv_heads, block_size / 32, 2, 32]``);
    :meth:`to_quantized` and :meth:`from_quantized` convert to and from row-major
    numbers.
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
        shape = (num_blocks, kv_heads, block_size // GROUP, head_dim // 64, 1024)
        self.k = torch.zeros(shape, dtype=torch.uint8, device=device)
        self.v = torch.zeros_like(self.k)
        self.rows = torch.full((*shape[:3], 2, GROUP), _EMPTY, dtype=torch.int16, device=device)

    num_blocks = property(lambda self: self.k.size(0))
    kv_heads = property(lambda self: self.k.size(1))
    block_size = property(lambda self: self.k.size(2) * GROUP)
    head_dim = property(lambda self: self.k.size(3) * 64)
    device = property(lambda self: self.k.device)

    def tensors(self):
        """(k, v, rows), as the ops of ``torch.ops.kv4`` take them."""
        return self.k, self.v, self.rows

    @classmethod
    def from_quantized(cls, k: torch.Tensor, k_step: torch.Tensor, k_zero: torch.Tensor, v: torch.Tensor,
                       v_step: torch.Tensor, v_zero: torch.Tensor) -> "KV4Cache":
        """A cache of row-major numbers k, v (uint8 [num_blocks, kv_heads, block_size,
        head_dim], 0..15), fp16 steps and uint8 zero points [num_blocks, kv_heads,
        block_size].  Raises where a number, step or zero point is none that the cache
        can hold; a key step of NaN marks a token that stands for NaN, keys and values.
        (Looks at the values, so it waits for the device.)
        """
        if k.dtype != torch.uint8 or v.dtype != torch.uint8 or k.dim() != 4 or k.shape != v.shape:
            raise ValueError("k and v must be uint8 [num_blocks, kv_heads, block_size, head_dim], "
                             f"got {k.dtype} {list(k.shape)} and {v.dtype} {list(v.shape)}")
        nb, heads, bs, d = k.shape
        if bs not in BLOCK_SIZES or d not in HEAD_DIMS:
            raise ValueError(f"block_size must be one of {BLOCK_SIZES} and head_dim one of "
                             f"{HEAD_DIMS}, got {bs} and {d}")
        for step, zero in ((k_step, k_zero), (v_step, v_zero)):
            if step.dtype != torch.float16 or zero.dtype != torch.uint8 or not step.shape == zero.shape == k.shape[:3]:
                raise ValueError(f"steps must be float16 and zero points uint8 {list(k.shape[:3])}, got "
                                 f"{step.dtype} {list(step.shape)} and {zero.dtype} {list(zero.shape)}")
        words = [(s.contiguous().view(torch.int16), z) for s, z in ((k_step, k_zero), (v_step, v_zero))]
        nan = torch.isnan(k_step)
        wrong = torch.stack([((words[0][0] & 15) != 0).logical_and(~nan).any(), ((words[1][0] & 15) != 0).any()] +
                            [~((k_step >= 2.0 ** -20) & (k_step <= MAX_STEP) | nan).all(),
                             ~((v_step >= 2.0 ** -20) & (v_step <= MAX_STEP)).all()] +
                            [(x > 15).any() for x in (k, v, k_zero, v_zero)]).any()
        if bool(wrong):
            raise ValueError("numbers and zero points must be 0..15, steps 2^-20 to 4352 with the last four "
                             "bits 0 (keys: or NaN)")
        c = cls.__new__(cls)
        # k: token 32 gr + 8 a + 4 tt + b, dimension 64 t + 16 g + 8 j + 2 p + h
        t = k.reshape(nb, heads, bs // 32, 4, 2, 4, d // 64, 4, 2, 4, 2)
        t = t.permute(0, 1, 2, 6, 7, 3, 5, 4, 8, 10, 9)   # [.., t, g, a, b, tt, j, h, p]
        c.k = _packed(t).reshape(nb, heads, bs // 32, d // 64, 1024)
        # v: token 32 gr + 8 g + 2 w + h, dimension 64 t + 4 c + b
        t = v.reshape(nb, heads, bs // 32, 4, 4, 2, d // 64, 16, 4)
        t = t.permute(0, 1, 2, 6, 3, 7, 4, 5, 8)          # [.., t, g, c, w, h, b]
        c.v = _packed(t).reshape(nb, heads, bs // 32, d // 64, 1024)
        kw = torch.where(nan, _NAN, words[0][0] | k_zero)
        rows = torch.stack((kw, words[1][0] | v_zero), 2).to(torch.int16)   # [nb, heads, 2, bs]
        c.rows = rows.view(nb, heads, 2, bs // 32, 32).transpose(2, 3).contiguous()
        return c

    def to_quantized(self):
        """(k, k_step, k_zero, v, v_step, v_zero), as :meth:`from_quantized` takes them."""
        nb, heads, gr, dt, _ = self.k.shape
        t = _unpacked(self.k).view(nb, heads, gr, dt, 4, 4, 4, 2, 2, 2, 4)
        k = t.permute(0, 1, 2, 5, 7, 6, 3, 4, 8, 10, 9).reshape(nb, heads, gr * 32, dt * 64)
        t = _unpacked(self.v).view(nb, heads, gr, dt, 4, 16, 4, 2, 4)
        v = t.permute(0, 1, 2, 4, 6, 7, 3, 5, 8).reshape(nb, heads, gr * 32, dt * 64)
        rows = self.rows.transpose(2, 3).reshape(nb, heads, 2, gr * 32)
        step, zero = (rows & ~15).view(torch.float16), (rows & 15).to(torch.uint8)
        return (k, step[:, :, 0].contiguous(), zero[:, :, 0].contiguous(),
                v, step[:, :, 1].contiguous(), zero[:, :, 1].contiguous())

    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """:func:`kv4_append` into this cache."""
        kv4_append(self, k, v, slots)

    def read(self, slots: torch.Tensor, dtype: torch.dtype = torch.float16):
        """:func:`kv4_read` from this cache."""
        return kv4_read(self, slots, dtype)

    def attention(self, q: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor,
                  cu_q: torch.Tensor | None = None, **kw):
        """:func:`kv4_attention` over this cache."""
        return kv4_attention(q, self, block_table, kv_lens, cu_q, **kw)


def _packed(t: torch.Tensor) -> torch.Tensor:
    """Two numbers a byte, the first in the low bits."""
    t = t.reshape(-1, 2)
    return t[:, 0] | t[:, 1] << 4


def _unpacked(t: torch.Tensor) -> torch.Tensor:
    return torch.stack((t & 15, t >> 4), -1)


def kv4_append(cache: KV4Cache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantizes k, v [tokens, kv_heads, head_dim] (fp16 or bf16) into ``slots``
    [tokens] (int32, slot = block * block_size + token in the block, no two the same;
    negative or past the cache: skipped).

    Each token's head has a step of its own, the least with 15 steps from its
    smallest value (or 0) to its largest (or 0): values are off by at most half a
    step, and tokens held before are not touched.  Steps are rounded up to seven
    significant bits, below 2^-14 to multiples of 2^-20: half a step is at most 1/30 of
    the span and 2^-6 of that more, or 2^-21 more.  A span over 65280 is cut.  A token
    with an infinity or NaN among the keys or values of a head reads back as NaN there,
    keys and values.
    """
    _append(*cache.tensors(), k, v, slots)


def kv4_read(cache: KV4Cache, slots: torch.Tensor, dtype: torch.dtype = torch.float16):
    """Cached tokens as values: (k, v), each [n, kv_heads, head_dim] of fp16 (exact),
    bf16 or fp32, for int32 ``slots`` [n]; a slot outside the cache gives zeros."""
    return _read(*cache.tensors(), slots, dtype)


def kv4_attention(q: torch.Tensor, cache: KV4Cache, block_table: torch.Tensor,
                  kv_lens: torch.Tensor, cu_q: torch.Tensor | None = None, *, max_q_len: int = 0,
                  max_kv_len: int = 0, causal: bool = True, window: int = 0,
                  scale: float | None = None, return_lse: bool = False):
    """softmax(scale q k^T) v over the cache, for a ragged batch: the arguments, masks and
    results of :func:`~rhinoforge_amd.kv8.kv8_attention`.  A query that sees a token
    which stands for NaN gives NaN.
    """
    scale = cache.head_dim ** -0.5 if scale is None else scale
    out, lse = _attention(q, *cache.tensors(), block_table, kv_lens, cu_q, max_q_len, max_kv_len,
                          causal, window, scale, return_lse)
    return (out, lse) if return_lse else out
