"""A paged 8-bit key/value cache that runs the serving operators together.

One `PagedCache` holds the blocks of every layer, one row of the block table
for each request, and the stack of free blocks.  A step is

    step = cache.begin(new_lens)              # tokens that each request gains: tables, slots
    for layer in range(layers):
        out = cache.prefill(layer, q, k, v)   # whole prompts (requests that held nothing), or
        out = cache.decode(layer, q, k, v)    # one token for each request that gains one

A step is one or the other: `prefill` and `decode` refuse what is not theirs, and
`cancel` takes back a step that was begun and is not to be.
`begin` works out the step's lengths on the host (the caller knows them) and
everything else on the GPU; nothing synchronises.  The keys and values of a
prompt are attended to in 16 bits as they come and kept in 8 bits for the
tokens that follow.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import List, Optional, Sequence, Tuple

import torch

from . import ops

CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


@dataclass
class Step:
    """What `PagedCache.begin` found out: device tensors, and the host's lists."""
    new_lens: List[int]
    contexts: List[int]            # tokens before the step
    slots: torch.Tensor            # each new token's place in the cache
    cu_seqlens: torch.Tensor       # new tokens before each request
    seq_lens: torch.Tensor         # tokens after the step
    # Where some requests gain one token and the others none: the former's table rows and lengths.
    gaining: Optional[Tuple[torch.Tensor, torch.Tensor]]
    before: Tuple[torch.Tensor, torch.Tensor, int]   # lengths, free blocks (device, host) before the step


class PagedCache:
    def __init__(self, layers: int, requests: int, max_tokens: int, blocks: int, kv_heads: int,
                 dim: int, block_size: int = 16, codes: str = "int8", device=None):
        if codes not in CODES:
            raise ValueError(f"codes must be one of {sorted(CODES)}, got {codes!r}")
        if min(layers, requests, max_tokens, blocks, kv_heads) < 1:
            raise ValueError("layers, requests, max_tokens, blocks and kv_heads must be positive")
        if block_size not in (16, 32, 64, 128, 256):
            raise ValueError("block_size must be a power of two from 16 to 256")
        if dim % 16 or not 0 < dim <= 128:
            raise ValueError("dim must be a multiple of 16, at most 128")
        device = torch.device("cuda" if device is None else device)
        self.block_size, self.blocks, self.max_tokens = block_size, blocks, max_tokens
        shape = (layers, blocks, kv_heads, block_size, dim)
        ints = dict(dtype=torch.int32, device=device)
        self.k_cache = torch.zeros(shape, dtype=torch.uint8, device=device).view(CODES[codes])
        self.v_cache = torch.zeros(shape, dtype=torch.uint8, device=device).view(CODES[codes])
        self.k_scale = torch.zeros(shape[:3], dtype=torch.float32, device=device)
        self.v_scale = torch.zeros(shape[:3], dtype=torch.float32, device=device)
        self.block_table = torch.full((requests, -(-max_tokens // block_size)), -1, **ints)
        self.free_blocks = torch.arange(blocks - 1, -1, -1, **ints)
        self.free_count = torch.full((1,), blocks, **ints)
        self.lens = torch.zeros(requests, **ints)
        self.lengths = [0] * requests      # the same on the host
        self.free = blocks
        self.step = None

    def _held(self, tokens: int) -> int:
        return -(-tokens // self.block_size)

    def _open(self) -> Step:
        if self.step is None:
            raise RuntimeError("begin() opens a step first")
        return self.step

    def begin(self, new_lens: Sequence[int]) -> Step:
        """Make room for `new_lens[r]` more tokens of each request r."""
        new_lens = [int(n) for n in new_lens]
        if len(new_lens) != len(self.lengths):
            raise ValueError(f"new_lens must have {len(self.lengths)} values, got {len(new_lens)}")
        if min(new_lens) < 0:
            raise ValueError("new_lens must not be negative")
        after = [a + n for a, n in zip(self.lengths, new_lens)]
        if max(after) > self.max_tokens:
            raise ValueError(f"a request would hold {max(after)} tokens, the cache allows {self.max_tokens}")
        need = sum(self._held(b) - self._held(a) for a, b in zip(self.lengths, after))
        if need > self.free:
            raise RuntimeError(f"the step needs {need} blocks, {self.free} are free")
        gained = torch.tensor(new_lens, dtype=torch.int32, pin_memory=True).to(
            self.lens.device, non_blocking=True)
        slots, cu, lens, left = ops.block_tables(self.lens, gained, self.block_table, self.free_blocks,
                                                 self.free_count, sum(new_lens), self.block_size)
        gaining = None
        if min(new_lens) == 0 and max(new_lens) <= 1:
            rows = torch.tensor([r for r, n in enumerate(new_lens) if n], dtype=torch.int64,
                                pin_memory=True).to(lens.device, non_blocking=True)
            gaining = self.block_table[rows], lens[rows]
        self.step = Step(new_lens, self.lengths, slots, cu, lens, gaining,
                         (self.lens, self.free_count, self.free))
        self.lens, self.free_count = lens, left
        self.lengths, self.free = after, self.free - need
        return self.step

    def cancel(self) -> None:
        """Take back the step that `begin` opened: the requests hold what they held before it, and its
        blocks are free.  (Codes that it wrote count for nothing; the scale of a block that was partly
        filled stays as its tokens may have raised it.)"""
        step = self._open()
        self.lens, self.free_count, self.free = step.before
        self.lengths = step.contexts
        self.step = None

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """Keep the step's keys and values (tokens, kv_heads, dim)."""
        ops.cache_append(k, v, self._open().slots, self.k_cache[layer], self.v_cache[layer],
                         self.k_scale[layer], self.v_scale[layer])

    def prefill(self, layer: int, q, k, v, scale=None) -> torch.Tensor:
        """The step's prompts: keep their keys and values, and attend to them."""
        step = self._open()
        if any(n and c for n, c in zip(step.new_lens, step.contexts)):
            raise RuntimeError("prefill() is for requests that held no token (cancel() takes the step back)")
        self.append(layer, k, v)
        return ops.prompt_attention(q, k, v, self.step.cu_seqlens, scale=scale)

    def decode(self, layer: int, q, k, v, scale=None) -> torch.Tensor:
        """One token of each request that gains one: keep its key and value, and attend to all
        that the request holds."""
        step = self._open()
        if max(step.new_lens) > 1:
            raise RuntimeError("decode() is for steps of one token a request (cancel() takes the step back)")
        self.append(layer, k, v)
        table, lens = step.gaining or (self.block_table, step.seq_lens)
        return ops.cache_attention(q, self.k_cache[layer], self.v_cache[layer], self.k_scale[layer],
                                   self.v_scale[layer], table, lens, scale)

    def release(self, request: int) -> None:
        """Give a finished request's blocks back; its row is free for another."""
        if not 0 <= request < len(self.lengths):
            raise IndexError(f"request must be from 0 to {len(self.lengths) - 1}, got {request}")
        n = self._held(self.lengths[request])
        self.free_blocks[self.free:self.free + n] = self.block_table[request, :n]
        self.free += n
        self.lengths = [0 if r == request else a for r, a in enumerate(self.lengths)]
        self.free_count = self.free_count + n
        self.lens = self.lens.clone()
        self.lens[request] = 0
        self.step = None
