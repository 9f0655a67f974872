"""Queries that see keys, but with scores of minus infinity only: the softmax has no value
there and the result is NaN, where a query that sees no key at all gives 0."""
import pytest
import torch

import attention_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new,L,finite", [(1, 1, None), (1, 300, None), (1, 300, 100),
                                          (1, 9000, None), (1, 9000, 4000), (5, 200, 197),
                                          (5, 3, 1), (100, 150, 80), (100, 60, 30),
                                          (200, 4000, None), (200, 4000, 3900)])
def test_scores_of_minus_infinity(pkg, cuda, new, L, finite, D, int8):
    """Every key but `finite` has an element of -inf that every query multiplies by 1: a query
    that sees the finite key gives that key's value (its weight is 1), one that sees only
    others NaN, one before the first key 0."""
    k, v, ks, vs, tables = ref.paged([L], 16, 1, D, new + L, int8)
    q = torch.randn(new, 2, D, generator=torch.Generator().manual_seed(L)).half()
    q[..., 0] = 1.0
    if int8:  # a scale of infinity and one code
        q[..., 1:] = 0.0
        k[..., 0] = -100
        scale = torch.full_like(ks, float("inf"))
    else:
        k[..., 0] = -float("inf")
    if finite is not None:
        page, at = tables[0, finite // 16], finite % 16
        if int8:
            scale[page, 0, at] = 0.01
        else:
            k[page, 0, at, 0] = 1.0
    got = pkg.paged_attention(
        q.cuda(), k.cuda(), v.cuda(), tables.cuda(), torch.tensor([L]).int().cuda(),
        torch.tensor([0, new]).int().cuda(), max_seqlen=new,
        k_scale=scale.cuda() if int8 else None, v_scale=vs.cuda() if int8 else None).cpu()
    p = torch.arange(new) + L - new
    assert (got[p < 0] == 0).all()
    sees = torch.zeros(new, dtype=torch.bool) if finite is None else p >= finite
    assert got[(p >= 0) & ~sees].isnan().all()
    if sees.any():
        want = ref.rows_of(v, vs, tables[0], L)[finite].expand(int(sees.sum()), 2, D)
        # 8 bits: the scale's reciprocal, the quotient and a product beside the rounding
        tol = want.abs() * (ref.H16 + 8 * ref.H32) + ref.SUB16 if int8 else torch.zeros_like(want) + 1e-30
        ref.within(got[sees], want, tol)
