"""RotaryEmbedding: rotary positions (fni8serve/layers/rotary.py:21-55).

`cos_sin` fp32 [max_position, rotary_dim] holds each position's cosines, then its sines,
computed in 64 bits: an angle of position 131072 has lost 0.01 rad in 32.  `scaling`
stretches the positions for long contexts:

    {"type": "linear", "factor": f}     every angle divided by f
    {"type": "ntk", "factor": f}        base * f^(R / (R - 2)): the fastest pair keeps its
                                        angles, the slowest is stretched by f
    {"type": "yarn", "factor": f, "original_max_position": n, "beta_fast": 32,
     "beta_slow": 1, "attention_factor": 0.1 ln f + 1}
                                        pairs that turn more than beta_fast times in n
                                        positions keep their angles, those that turn less
                                        than beta_slow times are divided by f, a linear ramp
                                        over the pairs between; cosines and sines times
                                        attention_factor (Peng et al., YaRN, 2023)

forward(q, k, positions) rotates [T, heads, head_dim] tensors into new ones: fp16 on the
GPU, of a head_dim that is a multiple of 8 and at most 256, through the kernel (`ops.rope`),
anything else in fp32 by torch, as RMSNorm does.  A position outside the table gives NaN.
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn

from .. import ops


def _frequencies(rotary_dim: int, base: float, scaling: dict | None):
    """Angles a position (fp64 [rotary_dim / 2]) and the factor of cosines and sines."""
    pairs = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    if scaling is None:
        return base ** (-pairs / rotary_dim), 1.0
    kind, factor = scaling.get("type"), float(scaling.get("factor", 0))
    if kind not in ("linear", "ntk", "yarn") or not factor >= 1:
        raise ValueError(f"unsupported rotary scaling {scaling!r} (linear, ntk or yarn, with a "
                         "factor of at least 1)")
    if kind == "ntk":
        if rotary_dim < 4:
            raise ValueError("ntk scaling needs a rotary_dim of at least 4")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    freq = base ** (-pairs / rotary_dim)
    if kind == "linear":
        return freq / factor, 1.0
    if kind == "ntk":
        return freq, 1.0
    n, fast, slow = (scaling.get("original_max_position"), scaling.get("beta_fast", 32),
                     scaling.get("beta_slow", 1))
    if not n or n < 1 or not 0 < slow < fast:
        raise ValueError("yarn scaling needs original_max_position and 0 < beta_slow < beta_fast")

    def pair_of(turns):  # the (real) pair that turns so often in n positions
        return rotary_dim * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(base))

    low = max(math.floor(pair_of(fast)), 0)
    high = min(math.ceil(pair_of(slow)), rotary_dim - 1)
    ramp = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - low)
            / max(high - low, 0.001)).clamp(0, 1)
    if high <= 0:  # the first pair already turns less than `slow` times
        ramp = torch.ones_like(ramp)
    factor_of = scaling.get("attention_factor")
    return (freq / factor * ramp + freq * (1 - ramp),
            0.1 * math.log(factor) + 1.0 if factor_of is None else float(factor_of))


class RotaryEmbedding(nn.Module):
    def __init__(self, head_dim: int, max_position: int, base: float = 10000.0,
                 rotary_dim: int | None = None, *, interleaved: bool = False,
                 scaling: dict | None = None, device=None):
        super().__init__()
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if rotary_dim % 2 or not 0 < rotary_dim <= head_dim or max_position < 1 or not base > 1:
            raise ValueError(f"rotary_dim {rotary_dim} of head_dim {head_dim}, {max_position} "
                             f"positions, base {base}: rotary_dim must be even and at most "
                             "head_dim, with one position at least and a base over 1")
        self.head_dim, self.rotary_dim, self.interleaved = head_dim, rotary_dim, interleaved
        freq, factor = _frequencies(rotary_dim, float(base), scaling)
        angle = torch.arange(max_position, dtype=torch.float64)[:, None] * freq
        table = torch.cat([angle.cos(), angle.sin()], 1) * factor
        self.register_buffer("cos_sin", table.float().to(device), persistent=False)

    def _apply(self, fn, *args, **kw):
        table = self.cos_sin  # moves with the module and stays fp32 in half()
        super()._apply(fn, *args, **kw)
        self.cos_sin = table.to(self.cos_sin.device)
        return self

    def _rotate(self, x: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        pos, last = positions.long(), self.cos_sin.shape[0] - 1
        rows = self.cos_sin[pos.clamp(0, last)]
        rows = rows.masked_fill(((pos < 0) | (pos > last)).unsqueeze(-1), math.nan)
        cos, sin = rows.unsqueeze(1).chunk(2, -1)
        y = x.float()
        turn, rest = y[..., :self.rotary_dim], y[..., self.rotary_dim:]
        a, b = (turn[..., 0::2], turn[..., 1::2]) if self.interleaved else turn.chunk(2, -1)
        a, b = a * cos - b * sin, b * cos + a * sin
        turn = torch.stack([a, b], -1).flatten(-2) if self.interleaved else torch.cat([a, b], -1)
        return torch.cat([turn, rest], -1).to(x.dtype)

    def forward(self, q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor):
        if (q.is_cuda and q.dtype == torch.float16 and k.dtype == torch.float16
                and self.head_dim % 8 == 0 and self.head_dim <= 256):
            return ops.rope(q, k, positions, self.cos_sin, interleaved=self.interleaved)
        return self._rotate(q, positions), self._rotate(k, positions)
