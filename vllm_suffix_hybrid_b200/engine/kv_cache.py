"""Paged KV cache: block pool and per-layer cache tensors.

Cache layout per layer: K and V each [num_blocks, kv_heads, block, head_dim]
(one contiguous 16 KB page per (block, head) at head_dim 128), the layout the
attention kernel streams; with kv_format "nvfp4" each is uint8 [num_blocks,
kv_heads, page bytes] (4.5 KB a page).  Blocks are counted: a fork shares its
parent's full blocks, and one returns to the pool when its last holder
releases it.  Block 0 is reserved as the scratch page that
padded batch rows write into and read from, so a fixed-shape (CUDA-graph)
batch never touches a live request's cache.
"""
from __future__ import annotations

from typing import Dict, List

import torch


class BlockPool:
    def __init__(self, num_blocks: int):
        if num_blocks < 2:
            raise ValueError("the KV cache needs at least 2 blocks")
        self.num_blocks = num_blocks
        self._free = list(range(num_blocks - 1, 0, -1))  # block 0 reserved
        self._refs = [0] * num_blocks  # holders of each block

    @property
    def free(self) -> int:
        return len(self._free)

    def allocate(self, n: int) -> List[int]:
        if n > len(self._free):
            raise MemoryError(f"KV cache exhausted: need {n} blocks, {len(self._free)} free")
        out = self._free[-n:][::-1] if n else []
        del self._free[len(self._free) - n:]
        for b in out:
            self._refs[b] = 1
        return out

    def share(self, blocks: List[int]) -> None:
        """One more holder for each of these allocated blocks."""
        if any(self._refs[b] < 1 for b in blocks):
            raise ValueError("only allocated blocks can be shared")
        for b in blocks:
            self._refs[b] += 1

    def release(self, blocks: List[int]) -> None:
        """Give up one hold on each block; those without a holder return to the pool."""
        for b in reversed(blocks):
            if self._refs[b] < 1:
                raise ValueError(f"block {b} is not allocated")
            self._refs[b] -= 1
            if self._refs[b] == 0:
                self._free.append(b)

    def compaction(self) -> Dict[int, int]:
        """Moves {from: to} that bring the allocated blocks to the lowest ids (from and to share no id)."""
        live = [b for b in range(1, self.num_blocks) if self._refs[b]]
        holes = [b for b in range(1, len(live) + 1) if not self._refs[b]]
        return dict(zip([b for b in live if b > len(live)], holes))

    def moved(self, moves: Dict[int, int]) -> None:
        """The contents of `compaction`'s blocks have been copied and their tables rewritten."""
        for a, b in moves.items():
            self._refs[b], self._refs[a] = self._refs[a], 0
        self._free = [b for b in range(self.num_blocks - 1, 0, -1) if not self._refs[b]]


def allocate_caches(num_layers: int, shape, dtype, device) -> List[tuple]:
    caches = []
    for _ in range(num_layers):
        k = torch.zeros(shape, dtype=dtype, device=device)
        v = torch.zeros(shape, dtype=dtype, device=device)
        caches.append((k, v))
    return caches


def blocks_for(tokens: int, block_size: int) -> int:
    return (tokens + block_size - 1) // block_size
