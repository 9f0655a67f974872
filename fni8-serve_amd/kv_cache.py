"""The paged key/value cache of one attention layer (fni8serve/engine/kv_cache.py:409-830).

`PagedKVCache(num_pages, page_size, num_kv_heads, head_dim, dtype)` holds keys and
values [pages, heads, page_size, head_dim], in fp16 or, as the reference's serving
default, in int8 with one fp32 scale a row.  A head's rows of a page lie together, so
attention reads each page as one run of memory.  Which page holds which tokens is the
caller's (a block table a sequence); a token's slot is page * page_size + offset.

    step = cache.step(block_tables, new=[5, 1], total=[5, 300])
    q = cache.append(q, k, v, step, cos_sin, q_weight=..., k_weight=...)
    out = cache.attend(q, step)

The arithmetic runs in `ops.rope_append` and `ops.paged_attention`; nothing here waits for
the GPU (`step` sends what lies on the host, its block tables among it, from pinned memory in
one copy), and a step's tensors may be filled anew between replays of a graph.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import ops


@dataclass
class Step:
    """One call's tokens: `positions` and `slots` a token; `block_tables`, `context_lens`
    and `cu_seqlens` as in ops.paged_attention; `max_seqlen` new tokens a sequence at most."""
    positions: torch.Tensor
    slots: torch.Tensor
    block_tables: torch.Tensor
    context_lens: torch.Tensor
    cu_seqlens: torch.Tensor | None = None
    max_seqlen: int | None = None


class PagedKVCache:
    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.float16, device="cuda"):
        if dtype not in (torch.float16, torch.int8):
            raise ValueError(f"the cache holds fp16 or int8 (got {dtype})")
        if page_size < 16 or page_size > 65536 or page_size & (page_size - 1):
            raise ValueError(f"page_size {page_size} must be a power of two from 16 to 65536")
        if num_pages < 1 or num_kv_heads < 1 or num_pages * page_size >= 1 << 31:
            raise ValueError(f"{num_pages} pages of {page_size} for {num_kv_heads} heads: at least "
                             "one of each and fewer than 2^31 slots")
        if head_dim % 16 or not 16 <= head_dim <= 256:
            raise ValueError(f"head_dim {head_dim} must be a multiple of 16, at most 256")
        shape = (num_pages, num_kv_heads, page_size, head_dim)
        # what was never written may be read as part of a page, and is masked: any contents
        # do, zeros keep a dump of the cache readable
        self.k, self.v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
        self.k_scale = self.v_scale = None
        if dtype == torch.int8:
            self.k_scale, self.v_scale = (torch.zeros(shape[:3], device=device) for _ in range(2))
        self.num_pages, self.page_size = num_pages, page_size
        self.num_kv_heads, self.head_dim, self.dtype = num_kv_heads, head_dim, dtype

    def step(self, block_tables: torch.Tensor, new: list[int], total: list[int]) -> Step:
        """The step that brings `new[s]` tokens to sequence s, the last of its `total[s]`.
        block_tables [sequences, pages], on the GPU or the host: the pages of each sequence's
        tokens, in order."""
        if len(new) != len(total) or len(new) != block_tables.shape[0]:
            raise ValueError(f"{len(new)} new and {len(total)} total lengths for "
                             f"{block_tables.shape[0]} block tables")
        if any(n < 0 or t < n for n, t in zip(new, total)):
            raise ValueError("a sequence has no fewer than 0 new tokens and no fewer in all")
        if any(-(-t // self.page_size) > block_tables.shape[1] for t in total):
            raise ValueError(f"a sequence of {max(total)} tokens needs more than "
                             f"{block_tables.shape[1]} pages of {self.page_size}")
        dev, width, shift = self.k.device, block_tables.shape[1], self.page_size.bit_length() - 1
        pos, at = [], []  # positions, and the place of each token's page in the tables
        for s, (n, t) in enumerate(zip(new, total)):
            first = s * width
            pos += range(t - n, t)
            at += [first + (p >> shift) for p in range(t - n, t)]
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        # one copy to the device, from pinned memory: places, positions, lengths, bounds, tables
        # that lie on the host
        host = torch.tensor(at + pos + list(total) + cu, dtype=torch.int32)
        tables = ops._int32(block_tables)
        packed = tables.device != dev and tables.device.type == "cpu"
        if packed:
            host = torch.cat([host, tables.reshape(-1)])
        ints = (host.pin_memory() if dev.type == "cuda" else host).to(dev, non_blocking=True)
        at, pos, lens, cu, flat = ints.split([len(at), len(at), len(total), len(cu),
                                              len(ints) - 2 * len(at) - len(total) - len(cu)])
        tables = flat.view(tables.shape) if packed else tables.to(dev)
        slots = self._place(tables.reshape(-1).index_select(0, at), pos)
        return Step(pos, slots, tables, lens, cu, max(new, default=0))

    def slots(self, block_tables: torch.Tensor, sequences: torch.Tensor,
              positions: torch.Tensor) -> torch.Tensor:
        """int32 slots of tokens at `positions` of `sequences` (rows of block_tables).  A token
        that has none gets one outside the cache, which append drops: its position is negative
        (padding) or past the table, its sequence not in the table or its page not in the
        cache."""
        if block_tables.numel() == 0:
            return torch.full_like(positions, -1, dtype=torch.int32)
        rows, width = block_tables.shape
        shift = self.page_size.bit_length() - 1
        column, sequences = positions.long() >> shift, sequences.long()
        row, at = sequences.clamp(0, rows - 1), column.clamp(0, width - 1)
        page = torch.where((row == sequences) & (at == column), block_tables[row, at], -1)
        return self._place(page, positions)

    def _place(self, page: torch.Tensor, position: torch.Tensor) -> torch.Tensor:
        """int32 slots of tokens in their pages.  A page that is not in the cache counts as the
        one before the first or behind the last, whose slots 32 bits hold too: a larger number
        could wrap to a valid slot."""
        page = page.clamp(-1, self.num_pages).to(torch.int32)
        offset = (position & (self.page_size - 1)).to(torch.int32)
        return torch.add(offset, page, alpha=self.page_size)

    def append(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, step: Step,
               cos_sin: torch.Tensor | None = None, q_weight: torch.Tensor | None = None,
               k_weight: torch.Tensor | None = None, eps: float = 1e-6, interleaved: bool = False,
               unit_offset: bool = False) -> torch.Tensor:
        """Norm and rotation of q and k (ops.qk_norm_rope; without cos_sin no rotation), keys
        and values into their slots; returns the queries."""
        return ops.rope_append(q, k, v, None if cos_sin is None else step.positions, cos_sin,
                               self.k, self.v, step.slots, k_scale=self.k_scale,
                               v_scale=self.v_scale, q_weight=q_weight, k_weight=k_weight, eps=eps,
                               interleaved=interleaved, unit_offset=unit_offset)

    def attend(self, q: torch.Tensor, step: Step, scale: float | None = None,
               window: int | None = None) -> torch.Tensor:
        """Causal attention of the step's queries over the cache (ops.paged_attention)."""
        return ops.paged_attention(q, self.k, self.v, step.block_tables, step.context_lens,
                                   step.cu_seqlens, step.max_seqlen, k_scale=self.k_scale,
                                   v_scale=self.v_scale, scale=scale, window=window)

    def read(self, slots: torch.Tensor):
        """Keys and values at `slots`, as the numbers they stand for: fp32 [n, heads, head_dim],
        NaN for a slot outside the cache."""
        slots = slots.long()
        row = slots.clamp(0, self.num_pages * self.page_size - 1)
        page, at, outside = row // self.page_size, row % self.page_size, (row != slots)[:, None, None]
        out = []
        for x, s in ((self.k, self.k_scale), (self.v, self.v_scale)):
            rows = x[page, :, at].float()
            rows = rows if s is None else rows * s[page, :, at].unsqueeze(-1)
            out.append(rows.masked_fill(outside, math.nan))
        return out[0], out[1]
