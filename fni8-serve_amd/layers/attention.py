"""GQAAttention over the paged cache (fni8serve/layers/gqa_attention.py:29-157).

    GQAAttention(qkv, o, num_heads, num_kv_heads, head_dim, rotary, ...)
    .qkv_proj .o_proj                            LinearW8A8 (gqa_attention.py:53-54)

forward(x, cache, step) takes the tokens of a step (decoded tokens, drafted tokens, chunks
of prompts, mixed) through the QKV linear; the norm of every query and key head, the
rotation and the append to the cache in one launch; attention over the cache; and the O
linear (gqa_attention.py:62-100, :143-157).  Nothing synchronises, so a decode step can be
captured in a graph with its tensors filled anew between replays.

Where calling a norm or the rotation does more than its class defines (a hook, a forward of
its own, a subclass) or the norms are not of one kind, the modules are called one after the
other; a normed head is then rounded to fp16 before it is rotated.
"""
from __future__ import annotations

import torch
import torch.nn as nn
from torch.nn.modules.module import _has_any_global_hook

from ..kv_cache import PagedKVCache, Step
from ..qtensor import QTensor
from .linear import LinearW8A8
from .mlp import bare
from .norm import RMSNorm
from .rotary import RotaryEmbedding


class GQAAttention(nn.Module):
    def __init__(self, qkv: QTensor, o: QTensor, num_heads: int, num_kv_heads: int, head_dim: int,
                 rotary: RotaryEmbedding | None, *, q_norm: RMSNorm | None = None,
                 k_norm: RMSNorm | None = None, bias_qkv=None, bias_o=None,
                 scale: float | None = None, window: int | None = None):
        super().__init__()
        self.qkv_proj = LinearW8A8(qkv, bias_qkv)
        self.o_proj = LinearW8A8(o, bias_o)
        self.num_heads, self.num_kv_heads, self.head_dim = num_heads, num_kv_heads, head_dim
        self.rotary, self.q_norm, self.k_norm = rotary, q_norm, k_norm
        self.scale, self.window = scale, window
        wide = (num_heads + 2 * num_kv_heads) * head_dim
        if num_heads < 1 or num_kv_heads < 1 or num_heads % num_kv_heads:
            raise ValueError(f"{num_heads} query heads are no multiple of {num_kv_heads} key heads")
        if self.qkv_proj.out_features != wide or self.o_proj.in_features != num_heads * head_dim:
            raise ValueError(f"qkv has {self.qkv_proj.out_features} outputs and o "
                             f"{self.o_proj.in_features} inputs, expected {wide} and "
                             f"{num_heads * head_dim}")
        if rotary is not None and rotary.head_dim != head_dim:
            raise ValueError(f"rotary is for heads of {rotary.head_dim}, not {head_dim}")
        norms = [n for n in (q_norm, k_norm) if n is not None]
        if any(n.weight.numel() != head_dim or n.eps != norms[0].eps
               or n.add_unit_offset != norms[0].add_unit_offset for n in norms):
            raise ValueError("the norms of queries and keys are over head_dim, with one eps and "
                             "one add_unit_offset")

    def forward(self, x: torch.Tensor, cache: PagedKVCache, step: Step) -> torch.Tensor:
        """x fp16 [T, hidden] on the GPU -> [T, hidden]; the step's keys and values are in the
        cache afterwards."""
        D, nq, nk = self.head_dim, self.num_heads * self.head_dim, self.num_kv_heads * self.head_dim
        q, k, v = (t.unflatten(-1, (-1, D)) for t in self.qkv_proj(x).split([nq, nk, nk], -1))
        q_norm, k_norm, rotary = self.q_norm, self.k_norm, self.rotary
        if self._in_one_launch():
            norm = q_norm if q_norm is not None else k_norm
            q = cache.append(q, k, v, step, None if rotary is None else rotary.cos_sin,
                             q_weight=None if q_norm is None else q_norm.weight,
                             k_weight=None if k_norm is None else k_norm.weight,
                             eps=1e-6 if norm is None else norm.eps,
                             interleaved=rotary is not None and rotary.interleaved,
                             unit_offset=norm is not None and norm.add_unit_offset)
        else:
            q = q if q_norm is None else q_norm(q)
            k = k if k_norm is None else k_norm(k)
            if rotary is not None:
                q, k = rotary(q, k, step.positions)
            q = cache.append(q, k, v, step)
        out = cache.attend(q, step, scale=self.scale, window=self.window)
        return self.o_proj(out.flatten(1))

    def _in_one_launch(self) -> bool:
        """Whether the norms and the rotation are what the append computes on its way."""
        norms = [n for n in (self.q_norm, self.k_norm) if n is not None]
        return ((self.rotary is None or bare(self.rotary, RotaryEmbedding))
                and all(bare(n, RMSNorm) and n.weight.dtype == torch.float16
                        and n.eps == norms[0].eps
                        and n.add_unit_offset == norms[0].add_unit_offset for n in norms)
                and not _has_any_global_hook())
