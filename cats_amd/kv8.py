"""A cache of keys and values in 8 bits for one attention layer: the tensors that ``flash_gemv.cats_kv8_append`` and ``cats_kv8_attention`` share.

Blocks of 64 tokens are held as e4m3 numbers with one power of two as scale for each head's keys and values; a row's last block, complete or not, is
kept as it was given.  So a token is rounded once, and a cache holds the same whatever pieces the tokens came in.  Half the memory of a
16-bit cache and half the bytes a decode step reads; a number is off by at most 2^-4 of itself.

    cache = Kv8Cache(rows, kv_heads, max_len, head_dim, torch.float16)
    cache.append(k, v, start)              # k, v (rows, T, kv_heads, head_dim); start: where each row ends, int64 on the GPU
    out = cache.attend(q, start)           # q (rows, T, heads, head_dim), causal; the same start and count
    cache.reorder(parents, start + T)      # beam search: rows become what their parents were

A row ends where the last call left it.  Tokens are taken back by a smaller start, as far as the start of the block that holds the last one, or
to the start of any block: tokens of an earlier block are there as e4m3 only, and the rest of that block has to be given again.

Drafted tokens may pass the end of a block before they are checked.  Who wants to go on from inside that block keeps the tails (64 tokens a row) over the
draft, and after it puts them back and stores the accepted tokens again:

    kept = cache.k_tail.clone(), cache.v_tail.clone()
    cache.append(k, v, start)              # five drafted tokens from 62, say: a block is completed, and the tails begin the next one
    out = cache.attend(q, start)           # one is accepted
    cache.k_tail.copy_(kept[0]), cache.v_tail.copy_(kept[1])
    cache.append(k, v, start, accepted)    # int64 on the GPU, one for all rows or one each; the row ends at start + accepted

Nothing tells a cache from which block its tails are: a start further back than that makes a wrong block of what they hold.

For fp16 and bf16 on the GPU, heads of 32, 64, 128 or 256 elements, without gradients.
"""
from __future__ import annotations

import torch

BLOCK = 64


class Kv8Cache:
    FIELDS = ("k8", "v8", "k_scale", "v_scale", "k_tail", "v_tail")
    SLOTS = (BLOCK, BLOCK, BLOCK, BLOCK, 0, 0)  # tokens an entry of each holds, as cats_cache_reorder takes them

    def __init__(self, rows, kv_heads, max_len, head_dim, dtype=torch.float16, device="cuda"):
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"a cache in 8 bits is for float16 and bfloat16 models, not {dtype}")
        if head_dim not in (32, 64, 128, 256):
            raise ValueError(f"heads of 32, 64, 128 or 256 elements, not {head_dim}")
        if min(rows, kv_heads, max_len) < 1:
            raise ValueError("a cache needs at least one row, one head and one token")
        self.blocks = -(-max_len // BLOCK)
        shape = (rows, kv_heads, self.blocks)
        zeros = lambda *s, dtype: torch.zeros(s, dtype=dtype, device=device)
        # zeros in e4m3 by way of bytes: 0 is 0
        self.k8 = zeros(*shape, BLOCK, head_dim, dtype=torch.uint8).view(torch.float8_e4m3fn)
        self.v8 = zeros(*shape, head_dim, BLOCK, dtype=torch.uint8).view(torch.float8_e4m3fn)
        self.k_scale, self.v_scale = (torch.ones(shape, dtype=torch.float32, device=device) for _ in range(2))  # tokens that were never stored are zeros
        self.k_tail = zeros(rows, kv_heads, BLOCK, head_dim, dtype=dtype)
        self.v_tail = zeros(rows, kv_heads, head_dim, BLOCK, dtype=dtype)

    def tensors(self):
        return [getattr(self, f) for f in self.FIELDS]

    def append(self, k, v, start, count=None):
        """Store k, v (rows, T, kv_heads, head_dim) at positions start .. of each row, the first `count` of them."""
        import flash_gemv

        flash_gemv.cats_kv8_append(k, v, start, count, *self.tensors())

    def attend(self, q, start, count=None, scale=None, window=0):
        """Causal attention of q (rows, T, heads, head_dim), whose tokens have been appended at start."""
        import flash_gemv

        return flash_gemv.cats_kv8_attention(q, start, count, *self.tensors(), q.shape[-1] ** -0.5 if scale is None else scale, window)

    def reorder(self, parents, lengths):
        """Rows (groups of beams) become what their parents were; lengths: tokens they hold."""
        import flash_gemv

        flash_gemv.cats_cache_reorder(self.tensors(), self.SLOTS, parents, lengths)
