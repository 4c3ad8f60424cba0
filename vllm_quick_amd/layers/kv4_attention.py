"""Attention of a decoder layer over a paged cache that holds keys and values in 4 bits.

What stands between a layer's qkv product and its output product: the rotation of queries and keys, the append to the
cache and the attention over it, two launches of `ops.rope_append_kv4` and `ops.paged_attention_kv4`.  The same module
serves a prompt, a chunk of one, drafted tokens and single tokens; only `KV4Metadata` differs.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from .._C import ops


@dataclass
class KV4Metadata:
    """Where a step's tokens stand; the same for all layers.  Device tensors, so that a captured step is replayed with
    new contents; the two host integers size launches (see `ops.paged_attention_kv4`)."""
    positions: torch.Tensor  # int64 [tokens]
    slots: torch.Tensor  # int64 [tokens], -1: padding, nothing is stored
    block_tables: torch.Tensor  # int32 [sequences, blocks]
    seq_lens: torch.Tensor  # int32 [sequences], the step's own tokens among them
    max_seq_len: int
    query_start: Optional[torch.Tensor] = None  # int32 [sequences + 1]; None: one token for each sequence
    max_query_len: int = 1


def slots_of(block_tables: torch.Tensor, positions: torch.Tensor, block_size: int,
             sequences: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Slots of tokens at `positions` of their sequences (row of block_tables for each token; None: token i is of sequence
    i): block * block_size + place in the block; -1, which stores nothing, for a position that the row has no block for
    (a padded token's -1)."""
    rows = block_tables if sequences is None else block_tables[sequences]
    if rows.shape[1] == 0:
        return torch.full_like(positions, -1)
    page = torch.div(positions, block_size, rounding_mode="floor")
    block = rows.long().gather(1, page.clamp(0, rows.shape[1] - 1)[:, None])[:, 0]
    held = (page >= 0) & (page < rows.shape[1]) & (block >= 0)
    return torch.where(held, block * block_size + positions % block_size, -1)


def rope_table(positions: int, rotary: int, base: float = 10000.0, device: Optional[torch.device] = None) -> torch.Tensor:
    """fp32 [positions, rotary]: cosines of rotary / 2 angles, then their sines, from angles in 64 bits (in 32 a far
    position's angle has lost the digits that its cosine depends on)."""
    inv = float(base)**(-torch.arange(0, rotary, 2, dtype=torch.float64, device=device) / max(rotary, 1))
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * inv
    return torch.cat([angle.cos(), angle.sin()], 1).float()


class KV4Attention(torch.nn.Module):
    """query [T, heads * D], key and value [T, kv_heads * D] (views of one qkv tensor will do) -> [T, heads * D].

    Args: `scale` defaults to D ** -0.5; `window` > 0 lets a token see the last `window` tokens only; `interleaved`
    rotates neighbouring elements instead of halves.
    """

    def __init__(self, num_heads: int, head_size: int, num_kv_heads: Optional[int] = None, scale: Optional[float] = None,
                 window: int = 0, interleaved: bool = False):
        super().__init__()
        self.num_heads = num_heads
        self.head_size = head_size
        self.num_kv_heads = num_heads if num_kv_heads is None else num_kv_heads
        if self.num_kv_heads <= 0 or num_heads % self.num_kv_heads:
            raise ValueError(f"{num_heads} heads cannot share {self.num_kv_heads} kv heads")
        self.scale = head_size**-0.5 if scale is None else scale
        self.window = window
        self.interleaved = interleaved

    def make_cache(self, num_blocks: int, block_size: int, device: torch.device) -> torch.Tensor:
        return ops.kv4_cache(num_blocks, block_size, self.num_kv_heads, self.head_size, device)

    def forward(self, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, cache: torch.Tensor, cos_sin: torch.Tensor,
                meta: KV4Metadata) -> torch.Tensor:
        tokens, d = query.shape[0], self.head_size
        query = ops.rope_append_kv4(meta.positions, query.view(tokens, self.num_heads, d), key.view(tokens, self.num_kv_heads, d),
                                    value.view(tokens, self.num_kv_heads, d), cos_sin, cache, meta.slots, self.interleaved)
        out = ops.paged_attention_kv4(query, cache, meta.block_tables, meta.seq_lens, self.scale, meta.max_seq_len,
                                      meta.query_start, meta.max_query_len, self.window)
        return out.view(tokens, self.num_heads * d)
