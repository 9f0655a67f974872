"""Sequences that are longer than their block tables reach: the tokens past the table count
as keys of NaN, and the queries before them keep their own positions."""
import math

import pytest
import torch

import attention_ref as ref

pytestmark = pytest.mark.gpu


def _dev(t):
    return None if t is None else t.cuda()


def _check(pkg, cap, new, past, Hq, Hk, D, int8, window, seed):
    """Three sequences: one that ends with its table, one of `past` tokens more, a short one.
    A query at a position in the table sees what a sequence that ends with the table shows
    it; one past it is NaN."""
    lens = [cap, cap, 40]
    starts = [0, new, 2 * new, 2 * new + 3]
    k, v, ks, vs, tables = ref.paged(lens, 16, Hk, D, seed, int8)
    g = torch.Generator().manual_seed(seed + 1)
    q = (torch.randn(starts[-1] + 4, Hq, D, generator=g) * 1.5).half()
    inside = max(new - past, 0)  # queries of the second sequence in the table
    rows = [0, new, new + inside, new + inside + 3]
    kept = torch.cat([q[:new + inside], q[2 * new:starts[-1]]])
    want, tol = ref.attention(kept, k, v, tables, lens, rows, ks, vs, window=window)
    full = torch.full((q.shape[0], Hq, D), math.nan, dtype=torch.float64)
    bound = torch.ones_like(full)
    full[:new + inside], bound[:new + inside] = want[:new + inside], tol[:new + inside]
    full[2 * new:starts[-1]], bound[2 * new:starts[-1]] = want[-3:], tol[-3:]
    full[starts[-1]:] = 0.0  # padding
    got = pkg.paged_attention(
        q.cuda(), k.cuda(), v.cuda(), tables.cuda(),
        torch.tensor([cap, cap + past, 40], dtype=torch.int32).cuda(),
        torch.tensor(starts, dtype=torch.int32).cuda(), max_seqlen=max(new, 3), k_scale=_dev(ks),
        v_scale=_dev(vs), window=window)
    ref.within(got, full, bound, f"cap {cap}, {new} new, {past} past")


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("window", [None, 40])
@pytest.mark.parametrize("new,past", [(1, 1), (5, 1), (5, 3), (5, 30), (100, 1), (100, 30),
                                      (150, 149), (150, 151), (100, 1 << 30),
                                      (5, (1 << 31) - 1 - 1600)])
def test_queries_keep_their_positions(pkg, cuda, new, past, window, int8):
    for cap in (160, 1600):
        _check(pkg, cap, new, past, 8, 2, 128, int8, window, new + cap)


@pytest.mark.parametrize("Hq,Hk,D", [(4, 1, 64), (5, 1, 80), (16, 1, 256), (40, 2, 128)])
def test_every_kernel_form(pkg, cuda, Hq, Hk, D):
    for new, past in ((2, 1), (7, 4), (90, 31)):
        _check(pkg, 1040, new, past, Hq, Hk, D, False, None, D + new)


def test_one_sequence_alone(pkg, cuda):
    """A chunk alone in its call has no workgroups for few rows."""
    q = torch.randn(200, 4, 128, generator=torch.Generator().manual_seed(1)).half()
    k, v, _, _, tables = ref.paged([480], 16, 2, 128, 2)
    want, tol = ref.attention(q[:150], k, v, tables, [480], [0, 150])
    got = pkg.paged_attention(q.cuda(), k.cuda(), v.cuda(), tables.cuda(),
                              torch.tensor([530]).int().cuda(), torch.tensor([0, 200]).int().cuda())
    ref.within(got[:150], want, tol)
    assert got[150:].isnan().all()
