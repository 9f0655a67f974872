"""Yarn scaling at lengths so short that even the fastest pair turns slowly."""
import math

import pytest
import torch


@pytest.mark.parametrize("n,slow,fast", [(4, 1, 32), (1, 1, 32), (64, 16, 32), (50, 8, 9), (6.2, 1, 2)])
@pytest.mark.parametrize("R", [2, 8, 64])
def test_pairs_that_all_turn_slowly_are_all_stretched(pkg, R, n, slow, fast):
    assert n / (2 * math.pi) < slow  # the turns of the fastest pair, one radian a position
    rot = pkg.RotaryEmbedding(R, 2, scaling={
        "type": "yarn", "factor": 8, "original_max_position": n, "beta_slow": slow,
        "beta_fast": fast, "attention_factor": 1})
    want = 1e4 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R) / 8
    got = torch.atan2(rot.cos_sin[1, R // 2:].double(), rot.cos_sin[1, :R // 2].double())
    # cosine and sine are off by half a step of fp32 each
    assert ((got - want).abs() <= 2 * 2.0 ** -24).all()
