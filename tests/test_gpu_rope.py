"""Norms of queries and keys, rotary positions and the cache append on the GPU, against
their plain form in 64 bits."""
import pytest
import torch

import attention_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(pkg):
    return pkg.ops


def _qkv(T, Hq, Hk, D, seed, dtype=torch.float16):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, (Hq + 2 * Hk) * D, generator=g) * 2).to(dtype)
    w = [(1 + 0.3 * torch.randn(D, generator=g)).half() for _ in range(2)]
    return x, [t.unflatten(1, (-1, D)) for t in x.split([Hq * D, Hk * D, Hk * D], 1)], w, g


CASES = [  # T, Hq, Hk, D, R, pairs, unit
    (1, 16, 8, 128, 128, False, False),
    (7, 5, 1, 64, 32, True, False),
    (33, 32, 8, 128, 64, False, True),
    (65, 3, 3, 80, 80, True, True),
    (50, 10, 2, 96, 48, False, False),
    (12, 2, 1, 256, 256, False, False),
    (300, 8, 2, 256, 96, True, False),
    (19, 4, 4, 72, 70, False, False),   # halves that no chunk of 8 ends with
    (19, 4, 4, 40, 22, True, True),
    (5, 1, 1, 8, 2, False, False),
]


@pytest.mark.parametrize("T,Hq,Hk,D,R,pairs,unit", CASES)
@pytest.mark.parametrize("norm", [True, False])
def test_norm_rope(ops, cuda, T, Hq, Hk, D, R, pairs, unit, norm):
    x, (q, k, _), w, g = _qkv(T, Hq, Hk, D, T + D)
    P = 5000
    pos = torch.randint(0, P, (T,), generator=g)
    pos[0], pos[-1] = P - 1, 0
    tab = ref.table(P, R)
    xg = x.cuda()
    qg, kg, _ = (t.unflatten(1, (-1, D)) for t in xg.split([Hq * D, Hk * D, Hk * D], 1))
    if norm:
        got = ops.qk_norm_rope(qg, kg, w[0].cuda(), w[1].cuda(), pos.cuda(), tab.cuda(), eps=1e-5,
                               interleaved=pairs, unit_offset=unit)
    else:
        got = ops.rope(qg, kg, pos.to(torch.int32).cuda(), tab.cuda(), interleaved=pairs)
    assert torch.equal(xg.cpu(), x)
    for y, t, wt in zip(got, (q, k), w):
        want, tol = ref.norm_rope(t, wt if norm else None, pos, tab, pairs, 1e-5, unit)
        assert y.shape == t.shape and y.is_contiguous()
        ref.within(y, want, tol)


def test_norm_without_rotation_and_one_sided_weights(ops, cuda):
    x, (q, k, _), w, _ = _qkv(9, 4, 2, 128, 3)
    got = ops.qk_norm_rope(q.cuda(), k.cuda(), w[0].cuda(), None, None, None)
    ref.within(got[0], *ref.norm_rope(q, w[0], None, None))
    assert torch.equal(got[1].cpu(), k)


def test_positions_outside_the_table_give_nan(ops, cuda):
    x, (q, k, _), w, _ = _qkv(6, 4, 2, 64, 4)
    pos = torch.tensor([0, -1, 9, 10, 1 << 30, 3])
    got = ops.rope(q.cuda(), k.cuda(), pos.cuda(), ref.table(10, 32).cuda())
    for y, t in zip(got, (q, k)):
        ref.within(y, *ref.norm_rope(t, None, pos, ref.table(10, 32)))


def test_far_positions_and_extreme_rows(ops, cuda):
    """The last positions of a long table; rows of zeros, of the largest and the smallest
    values, of infinities and NaN, each of which stays in its row."""
    x, (q, k, _), w, _ = _qkv(8, 2, 2, 128, 5)
    P = 200000
    pos = torch.arange(P - 8, P)
    q[1, 0], q[2, 0], q[3, 1] = 0.0, 60000.0, 6e-8
    k[4, 1, 5], k[5, 0, 100] = float("inf"), float("nan")
    tab = ref.table(P, 128, 1e6)
    for norm in (False, True):
        ww = w if norm else (None, None)
        got = ops.qk_norm_rope(q.cuda(), k.cuda(), *(None if t is None else t.cuda() for t in ww),
                               pos.cuda(), tab.cuda())
        for n, (y, t) in enumerate(zip(got, (q, k))):
            want, tol = ref.norm_rope(t, ww[n], pos, tab)
            rows = torch.ones(8, 2, dtype=torch.bool)
            if n:
                rows[4, 1] = rows[5, 0] = False
                assert not y[4, 1].isfinite().all() and not y[5, 0].isfinite().all()
            big = want.abs() >= 65520
            assert torch.equal(y.cpu()[rows].isinf(), big[rows])
            keep = rows[..., None] & ~big
            ref.within(torch.where(keep, y.cpu().double(), 0.0), torch.where(keep, want, 0.0),
                       torch.where(keep, tol, 1.0))


def test_strides(ops, cuda):
    """Heads before tokens, rows with a gap, unaligned rows, a single token or head."""
    T, H, D = 11, 4, 64
    pos, tab = torch.arange(T).cuda(), ref.table(64, 64).cuda()
    x = torch.randn(H, T, 2 * D).half().cuda()
    base = x[:, :, :D].transpose(0, 1)
    off = torch.randn(T, H * D + 3).half().cuda()[:, 3:].unflatten(1, (H, D))
    wide = torch.randn(T, H, D, 2).half().cuda()[..., 0]
    for q in (base, off, wide, base[:1], base[:, :1], base.expand(T, H, D)[::2]):
        n = q.shape[0]
        got = ops.rope(q, q, pos[:n], tab)
        plain = q.contiguous()
        same = ops.rope(plain, plain, pos[:n], tab)
        assert torch.equal(got[0], same[0]) and torch.equal(got[1], same[0])


def _slots(T, pages, page, g):
    s = torch.randperm(pages * page, generator=g)[:T]
    return s.to(torch.int32)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("T,Hq,Hk,D,R,page", [(1, 16, 8, 128, 128, 16), (40, 4, 4, 64, 64, 32),
                                              (300, 8, 1, 256, 64, 64), (17, 6, 2, 96, 96, 128),
                                              (70, 8, 8, 80, 80, 16), (5, 2, 1, 16, 6, 1024)])
def test_append(ops, cuda, T, Hq, Hk, D, R, page, int8):
    """Queries and keys are qk_norm_rope's, values as they are; codes and scales are those of
    quantize_rowwise; every other slot keeps its bytes, and a dropped token writes none."""
    x, (q, k, v), w, g = _qkv(T, Hq, Hk, D, 7 * T + D)
    pages = -(-T // page) + 2
    slots = _slots(T, pages, page, g)
    drop = torch.zeros(T, dtype=torch.bool)
    if T > 4:
        drop[[1, 3, 4]] = True
        slots[1], slots[3], slots[4] = -1, pages * page, -(1 << 30)
    tab, pos = ref.table(4096, R).cuda(), torch.randint(0, 4096, (T,), generator=g).cuda()
    dt = torch.int8 if int8 else torch.float16
    cache = [torch.randint(-100, 100, (pages, Hk, page, D), generator=g).to(dt).cuda()
             for _ in range(2)]
    scale = [torch.rand(pages, Hk, page, generator=g).cuda() if int8 else None for _ in range(2)]
    before = [c.clone() for c in cache] + [s.clone() for s in scale if int8]
    args = (pos, tab)
    kw = dict(q_weight=w[0].cuda(), k_weight=w[1].cuda())
    xg = x.cuda()
    qg, kg, vg = (t.unflatten(1, (-1, D)) for t in xg.split([Hq * D, Hk * D, Hk * D], 1))
    got = ops.rope_append(qg, kg, vg, *args, *cache, slots.cuda(), *scale, **kw)
    want_q, want_k = ops.qk_norm_rope(qg, kg, kw["q_weight"], kw["k_weight"], *args)
    assert torch.equal(got, want_q)
    live = slots[~drop].long()
    for n, rows in enumerate((want_k, vg)):
        c = before[n].transpose(1, 2).reshape(pages * page, Hk, D).clone()
        rows = rows[(~drop).cuda()].contiguous()
        if int8:
            codes, s = ops.quantize_rowwise(rows)
            t = before[2 + n].transpose(1, 2).reshape(pages * page, Hk).clone()
            t[live.cuda()] = s.view(-1, Hk)
            assert torch.equal(t, scale[n].transpose(1, 2).reshape(pages * page, Hk))
            rows = codes.view(-1, Hk, D)
        c[live.cuda()] = rows
        assert torch.equal(c, cache[n].transpose(1, 2).reshape(pages * page, Hk, D))


def test_append_without_rotation_keeps_the_rows(ops, cuda):
    x, (q, k, v), _, _ = _qkv(3, 2, 2, 64, 9)
    cache = [torch.zeros(2, 2, 16, 64, dtype=torch.float16, device="cuda") for _ in range(2)]
    got = ops.rope_append(q.cuda(), k.cuda(), v.cuda(), None, None, *cache,
                          torch.tensor([31, 0, 7]).cuda())
    assert torch.equal(got.cpu(), q)
    for c, t in zip(cache, (k, v)):
        flat = c.transpose(1, 2).reshape(32, 2, 64).cpu()
        assert torch.equal(flat[[31, 0, 7]], t)
        assert flat.count_nonzero() == t.count_nonzero()


def test_append_in_a_long_cache(ops, cuda):
    """Byte offsets past 32 bits: 2^25 slots of one head of 128 are 8 GiB a cache."""
    pages, page, D = 1 << 13, 4096, 128
    cache = [torch.zeros(pages, 1, page, D, dtype=torch.float16, device="cuda") for _ in range(2)]
    x, (q, k, v), _, _ = _qkv(4, 1, 1, D, 11)
    slots = torch.tensor([pages * page - 1, 1 << 24, (1 << 24) - 1, 5])
    ops.rope_append(q.cuda(), k.cuda(), v.cuda(), None, None, *cache, slots.cuda())
    for c, t in zip(cache, (k, v)):
        assert torch.equal(c.view(-1, D)[slots.cuda()].cpu(), t[:, 0])


def test_append_rows_that_are_not_finite(ops, cuda):
    """8 bits: a row with an infinity or NaN gets codes 0 under a scale that is not finite."""
    x, (q, k, v), _, _ = _qkv(3, 1, 1, 64, 12)
    v[0, 0, 3], v[1, 0, 60] = float("inf"), float("nan")
    cache = [torch.ones(1, 1, 16, 64, dtype=torch.int8, device="cuda") for _ in range(2)]
    scale = [torch.zeros(1, 1, 16, device="cuda") for _ in range(2)]
    ops.rope_append(q.cuda(), k.cuda(), v.cuda(), None, None, *cache,
                    torch.arange(3, device="cuda"), *scale)
    want, s = ops.quantize_rowwise(v.cuda())
    assert torch.equal(cache[1][0, 0, :3], want)
    assert torch.equal(scale[1][0, 0, :3].isnan(), s.isnan()) and scale[1][0, 0, 0].isinf()


def test_empty_and_refused(ops, cuda):
    q = torch.randn(4, 4, 64).half().cuda()
    tab, pos = ref.table(16, 64).cuda(), torch.arange(4).cuda()
    assert ops.rope(q[:0], q[:0], pos[:0], tab)[0].shape == (0, 4, 64)
    cache = torch.zeros(2, 4, 16, 64, dtype=torch.float16, device="cuda")
    bad = [
        lambda: ops.rope(q.bfloat16(), q, pos, tab),
        lambda: ops.rope(q[0], q, pos, tab),
        lambda: ops.rope(q, q[:3], pos, tab),
        lambda: ops.rope(q, q, pos[:3], tab),
        lambda: ops.rope(q, q, pos.float(), tab),
        lambda: ops.rope(q, q, pos, tab.double()),
        lambda: ops.rope(q, q, pos, ref.table(16, 66).cuda()),
        lambda: ops.rope(q, q, pos, tab[:0]),
        lambda: ops.rope(q, q, None, None),
        lambda: ops.rope(q, q.cpu(), pos, tab),
        lambda: ops.rope(q[..., :60], q[..., :60], pos, tab[:, :32].contiguous()),
        lambda: ops.qk_norm_rope(q, q, tab[0], None, pos, tab),
        lambda: ops.qk_norm_rope(q, q, None, None, pos, None),
        lambda: ops.qk_norm_rope(q, q, None, None, pos, tab, eps=float("nan")),
        lambda: ops.rope_append(q, q, q[:, :2], pos, tab, cache, cache, pos),
        lambda: ops.rope_append(q, q, q, pos, tab, cache, cache[:1], pos),
        lambda: ops.rope_append(q, q, q, pos, tab, cache, cache.to(torch.int8), pos),
        lambda: ops.rope_append(q, q, q, pos, tab, cache.transpose(1, 2), cache, pos),
        lambda: ops.rope_append(q, q, q, pos, tab, cache[:, :, :8].contiguous(),
                                cache[:, :, :8].contiguous(), pos),
        lambda: ops.rope_append(q, q, q, pos, tab, cache, cache, pos[:2]),
        lambda: ops.rope_append(q, q, q, pos, tab, cache, cache, pos,
                                k_scale=torch.zeros(2, 4, 16, device="cuda")),
    ]
    for n, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {n} was not refused")
