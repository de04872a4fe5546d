"""The 8-bit K/V cache that decode attention reads (no counterpart in the
reference, which has no cache).

Every full block of 64 tokens of a K/V head is held in e4m3 with one
power-of-two scale; the last, unfinished block of each sequence is held in
BF16 (its tail).  A token is thus rounded once, with its whole block known,
and the cache's contents do not depend on how tokens were split into calls.
"""

from __future__ import annotations

import torch

from . import _C

BLOCK_TOKENS = _C.FU_KV_BLOCK


class KvCache:
    """The tensors of one layer's cache on one rank.

    ==============  ==========================  ==================================
    ``k_blocks``    ``float8_e4m3fn``           ``[num_blocks, kv_heads, 64, 128]``
    ``v_blocks``    ``float8_e4m3fn``           ``[num_blocks, kv_heads, 128, 64]``
    ``k_scales``    ``float32``                 ``[num_blocks, kv_heads]``
    ``v_scales``    ``float32``                 ``[num_blocks, kv_heads]``
    ``k_tail``      ``bfloat16``                ``[max_seqs, kv_heads, 64, 128]``
    ``v_tail``      ``bfloat16``                ``[max_seqs, kv_heads, 64, 128]``
    ``block_table`` ``int32``                   ``[max_seqs, max_blocks]``
    ==============  ==========================  ==================================

    A value of a full block is its e4m3 value times the block's scale;
    ``v_blocks`` holds dims by tokens.  A sequence occupies one slot, a row of
    ``block_table`` and of the tails; block ``b`` of its tokens is cache block
    ``block_table[slot, b]``.  Which blocks a slot uses is the caller's to
    decide (one table may serve the caches of several layers): entries up to
    the sequence's length must be in place before the call that completes
    them.  Tokens in the tail belong to the slot until their block is
    complete.  The tensors are the caller's too, and may be read at any time.
    """

    __slots__ = ("k_blocks", "v_blocks", "k_scales", "v_scales", "k_tail", "v_tail",
                 "block_table", "device", "num_blocks", "kv_heads", "max_seqs", "max_blocks",
                 "_desc", "_address")

    def __init__(self, k_blocks, v_blocks, k_scales, v_scales, k_tail, v_tail, block_table):
        if k_blocks.dim() != 4 or k_tail.dim() != 4 or block_table.dim() != 2:
            raise ValueError("k_blocks and k_tail have 4 dimensions, block_table has 2")
        num_blocks, heads = k_blocks.shape[:2]
        max_seqs, max_blocks = block_table.shape
        e4m3, block, dim = torch.float8_e4m3fn, BLOCK_TOKENS, _C.FU_HEAD_DIM
        tensors = dict(k_blocks=(k_blocks, e4m3, (num_blocks, heads, block, dim)),
                       v_blocks=(v_blocks, e4m3, (num_blocks, heads, dim, block)),
                       k_scales=(k_scales, torch.float32, (num_blocks, heads)),
                       v_scales=(v_scales, torch.float32, (num_blocks, heads)),
                       k_tail=(k_tail, torch.bfloat16, (max_seqs, heads, block, dim)),
                       v_tail=(v_tail, torch.bfloat16, (max_seqs, heads, block, dim)),
                       block_table=(block_table, torch.int32, (max_seqs, max_blocks)))
        if min(num_blocks, heads, max_seqs, max_blocks) < 1:
            raise ValueError("a cache has at least one block, head, slot and table column")
        if max_blocks * block >= 2 ** 31 or num_blocks >= 2 ** 31 or max_seqs >= 2 ** 31:
            raise ValueError("cache sizes must stay below 2^31")
        for name, (t, dtype, shape) in tensors.items():
            if (t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous()
                    or t.device != k_blocks.device or t.data_ptr() % 16):
                raise ValueError(f"{name} must be a contiguous, 16-byte aligned {dtype} tensor "
                                 f"of shape {shape} on {k_blocks.device}")
            setattr(self, name, t)
        self.device = k_blocks.device
        self.num_blocks, self.kv_heads = num_blocks, heads
        self.max_seqs, self.max_blocks = max_seqs, max_blocks
        d = _C.KvCacheDesc()
        d.device = -1 if self.device.index is None else self.device.index
        d.kv_heads, d.num_blocks, d.max_seqs, d.max_blocks = heads, num_blocks, max_seqs, max_blocks
        for name, (t, _, _) in tensors.items():
            setattr(d, name, t.data_ptr())
        self._desc = d
        self._address = _C.address_of(d)

    def __setattr__(self, name, value):
        # Calls read the addresses that the constructor took.
        if hasattr(self, "_address"):
            raise AttributeError("a KvCache's tensors are fixed; copy into them instead")
        super().__setattr__(name, value)

    @classmethod
    def allocate(cls, num_blocks, max_seqs, max_blocks, kv_heads, device):
        """A zeroed cache."""
        block, dim = BLOCK_TOKENS, _C.FU_HEAD_DIM

        def zeros(dtype, *shape):
            return torch.zeros(shape, dtype=dtype, device=device)

        return cls(k_blocks=zeros(torch.uint8, num_blocks, kv_heads, block, dim)
                   .view(torch.float8_e4m3fn),
                   v_blocks=zeros(torch.uint8, num_blocks, kv_heads, dim, block)
                   .view(torch.float8_e4m3fn),
                   k_scales=zeros(torch.float32, num_blocks, kv_heads),
                   v_scales=zeros(torch.float32, num_blocks, kv_heads),
                   k_tail=zeros(torch.bfloat16, max_seqs, kv_heads, block, dim),
                   v_tail=zeros(torch.bfloat16, max_seqs, kv_heads, block, dim),
                   block_table=zeros(torch.int32, max_seqs, max_blocks))
