"""Sampler: one token a row of logits (fni8serve/layers/sampler.py:20-87).

    token = Sampler()(head(hidden), temperature, top_k, top_p, min_p)

Settings are numbers, or tensors with one a row (ops.sample).  The random numbers are the
caller's (u), or drawn from torch's generator: a call in a captured graph draws new ones at
every replay.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from .. import ops


class Sampler(nn.Module):
    def __init__(self, return_logprobs: bool = False):
        super().__init__()
        self.return_logprobs = return_logprobs

    def forward(self, logits: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, *,
                u: torch.Tensor | None = None, generator: torch.Generator | None = None):
        """logits fp16 or fp32 [..., V] on the GPU -> int64 [...] (and log-probabilities)."""
        greedy = not torch.is_tensor(temperature) and temperature == 0
        if u is None and not greedy:
            u = torch.rand(logits.shape[:-1], device=logits.device, generator=generator)
        return ops.sample(logits, u, temperature, top_k, top_p, min_p,
                          return_logprobs=self.return_logprobs)
