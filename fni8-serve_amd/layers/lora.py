"""Low-rank adapters of many requests beside a LinearW8A8 (the unmerged forward of
fni8serve/training/lora.py:14-170, in serving: every token of a batch has its own adapter).

    batch = AdapterBatch(num_adapters)                 one for the modules that see the same rows
    mlp.down_proj = LoRALinear(mlp.down_proj, batch, rank=16)
    mlp.down_proj.load(3, [(A, B)], scaling=alpha / rank)
    batch.assign(ids)                                  once a step: each row's adapter, -1 none
    y = mlp(x)

A merged projection (QKV, gate and up) has one pair of matrices for each part of its output
(splits).  The module takes the place of the linear that it wraps: GatedMLP, GQAAttention and
LMHead call it as they call that.  While rows have adapters GatedMLP runs its projections one after
the other, since the adapter reads what its fused kernels never write.  SparseMoE's experts are stacked at
construction and take no adapters.
"""
from __future__ import annotations

from collections.abc import Sequence

import torch
import torch.nn as nn
from torch.nn.modules.module import _has_any_global_hook

from .. import ops
from .linear import LinearW8A8
from .mlp import _DEFINED, bare


class AdapterBatch:
    """Which adapter each row of a step has, shared by all LoRALinear modules that see these rows
    (an LMHead that sees the last token of each sequence needs one of its own)."""

    def __init__(self, num_adapters: int):
        if not 0 < num_adapters <= 65534:
            raise ValueError(f"num_adapters {num_adapters} must be from 1 to 65534")
        self.num_adapters = num_adapters
        self.ids: torch.Tensor | None = None
        self.plan: ops.LoraPlan | None = None
        self._kept: dict[tuple[torch.device, int], ops.LoraPlan] = {}
        self._assigned: set[tuple[torch.device, int]] = set()  # since the last clear

    def assign(self, ids: torch.Tensor) -> None:
        """ids int [rows]: each row's adapter, any number outside [0, num_adapters) for none.
        Nothing waits for the GPU.  The plan lies in memory that is kept, its own for every number
        of rows (4 bytes a row and an adapter): a captured graph of so many rows reads what the
        last assign of that many left there, so assign before a replay, on its stream."""
        if ids.dim() != 1 or ids.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"ids must be int32 or int64 [rows] (got {ids.dtype}, "
                             f"{tuple(ids.shape)})")
        self.ids, self.plan = ids, None
        if ids.is_cuda:
            self.plan = self._keep(ops.lora_plan(ids, self.num_adapters))

    def _keep(self, plan: ops.LoraPlan) -> ops.LoraPlan:
        """The plan, copied to the memory of its number of rows."""
        key = plan.rows.device, plan.rows.numel()
        kept = self._kept.get(key)
        if kept is None:
            with torch.inference_mode(False):  # a later assign outside it writes these too
                kept = self._kept[key] = ops.LoraPlan(*(torch.empty_like(t) for t in plan))
        for to, t in zip(kept, plan):
            to.copy_(t)
        self._assigned.add(key)
        return kept

    def clear(self) -> None:
        """No row has an adapter: the modules are the linears that they wrap, and a captured graph
        adds nothing until the next assign of its number of rows."""
        self.ids = self.plan = None
        for key in self._assigned:
            seg_off, rows = self._kept[key]
            seg_off.zero_()[-1:].fill_(rows.numel())      # all rows in the last segment
        self._assigned.clear()


class LoRALinear(nn.Module):
    def __init__(self, base: LinearW8A8, batch: AdapterBatch, rank: int,
                 splits: Sequence[int] | None = None):
        """rank: the largest of any adapter; kept as the next multiple of 8, smaller ones are
        filled with zeros.  splits: the widths of a merged projection's parts."""
        super().__init__()
        self.base, self.batch = base, batch
        self.in_features, self.out_features = base.in_features, base.out_features
        self.splits = [self.out_features] if splits is None else [int(n) for n in splits]
        if sum(self.splits) != self.out_features or min(self.splits) < 1:
            raise ValueError(f"splits {self.splits} do not add up to {self.out_features} outputs")
        if not 0 < rank <= 256:
            raise ValueError(f"rank {rank} must be from 1 to 256")
        self.rank = -(-rank // 8) * 8
        S, dev = batch.num_adapters, base.weight.data.device
        zeros = lambda *s: torch.zeros(s, dtype=torch.float16, device=dev)  # noqa: E731
        self.register_buffer("a", zeros(S, len(self.splits) * self.rank, self.in_features))
        self.register_buffer("b", zeros(S, self.out_features, self.rank))
        self.register_buffer("scaling", torch.zeros(S, device=dev))
        # of each part: rows that are filled up, and slots that are empty, add nothing
        self.register_buffer("ranks", torch.zeros(S, len(self.splits), dtype=torch.int32, device=dev))

    def _apply(self, fn, *args, **kw):
        had = dict(self._buffers)  # they move with the module and keep their types in half()
        super()._apply(fn, *args, **kw)
        for name, t in had.items():
            if self._buffers[name].dtype != t.dtype:
                self._buffers[name] = t.to(self._buffers[name].device)
        return self

    def _load_from_state_dict(self, state, prefix, *args):
        if prefix + "a" in state and prefix + "ranks" not in state:  # saved without: all rows
            state[prefix + "ranks"] = torch.full_like(self.ranks, self.rank)
        super()._load_from_state_dict(state, prefix, *args)

    # what callers read of the linear (layers/mlp.py, layers/attention.py)
    @property
    def weight(self):
        return self.base.weight

    @property
    def bias(self):
        return self.base.bias

    def _int8_ok(self, x: torch.Tensor) -> bool:
        """Where rows have adapters its input is needed in 16 bits: the fused chains leave it to be
        called, as they do where calling it does more than the classes define."""
        return (self.batch.ids is None and bare(self, LoRALinear) and bare(self.base, LinearW8A8)
                and not _has_any_global_hook() and self.base._int8_ok(x))

    def load(self, slot: int, parts: Sequence[tuple[torch.Tensor, torch.Tensor] | None],
             scaling: float = 1.0) -> None:
        """Adapter `slot`: for each part of the output its (A [r, in], B [width, r]) with r up to
        rank, or None for a part without one."""
        if not 0 <= slot < self.batch.num_adapters:
            raise ValueError(f"slot {slot} is not among {self.batch.num_adapters} adapters")
        if len(parts) != len(self.splits):
            raise ValueError(f"{len(parts)} pairs for {len(self.splits)} parts")
        for pair, wide in zip(parts, self.splits):
            if pair is not None:
                r = pair[0].shape[0]
                if r > self.rank or pair[0].shape != (r, self.in_features) \
                        or pair[1].shape != (wide, r):
                    raise ValueError(f"A {tuple(pair[0].shape)} and B {tuple(pair[1].shape)} do not "
                                     f"fit {self.in_features} inputs, {wide} outputs and rank "
                                     f"{self.rank}")
        self.a[slot].zero_()
        self.b[slot].zero_()
        n = 0
        for p, (pair, wide) in enumerate(zip(parts, self.splits)):
            if pair is not None:
                r = pair[0].shape[0]
                self.a[slot, p * self.rank:p * self.rank + r].copy_(pair[0])
                self.b[slot, n:n + wide, :r].copy_(pair[1])
            n += wide
        self.scaling[slot] = scaling
        for p, pair in enumerate(parts):
            self.ranks[slot, p] = 0 if pair is None else pair[0].shape[0]

    def unload(self, slot: int) -> None:
        """Rows of this adapter get nothing added from now on."""
        self.load(slot, [None] * len(self.splits), 0.0)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        y = self.base(x)
        if self.batch.ids is None:
            return y
        if not x.is_cuda:
            return self._on_host(x, y)
        if self.batch.plan is None:
            raise ValueError(f"the batch's ids are on {self.batch.ids.device}, the rows on "
                             f"{x.device}")
        # in place where nobody else can hold y: no hook, no forward but the linear's own
        fresh = bare(self.base, LinearW8A8) and not _has_any_global_hook()
        return ops.lora_add(y, x, self.a, self.b, self.batch.plan, scaling=self.scaling,
                            splits=self.splits, out=y if fresh else None, ranks=self.ranks)

    def _on_host(self, x: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
        """CPU tensors, beside the linear's own fallback: sums in 32 bits, rounded once."""
        ids = self.batch.ids
        x2, out = x.reshape(-1, self.in_features), y.reshape(-1, self.out_features)
        out = out.to(torch.float32, copy=True)
        if ids.is_cuda or ids.numel() != x2.shape[0]:
            raise ValueError(f"{x2.shape[0]} rows on the host, {ids.numel()} ids on {ids.device}")
        for e in range(self.batch.num_adapters):
            at = (ids == e).nonzero().squeeze(1)
            if at.numel():
                rows, n = x2[at].float(), 0
                for p, wide in enumerate(self.splits):
                    r, j = int(self.ranks[e, p]), p * self.rank
                    low = (rows @ self.a[e, j:j + r].float().t()) * self.scaling[e]
                    out[at, n:n + wide] += low @ self.b[e, n:n + wide, :r].float().t()
                    n += wide
        return out.to(y.dtype).reshape(y.shape)


_DEFINED[LoRALinear] = (LoRALinear.forward, LoRALinear._int8_ok)
