"""lora_add() against its formula in 64 bits, element by element within a bound derived from the
roundings it may make (bound()): fp32 sums of exact products, the pair of fp16 numbers that
carries a low-rank row, one rounding to fp16."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


def make(T, K, splits, rank, S, seed, ids=None):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, K, generator=g)
    x = torch.where(torch.rand(T, K, generator=g) < 0.01, x * 20, x).half()
    a = (torch.randn(S, len(splits) * rank, K, generator=g) * K ** -0.5).half()
    b = (torch.randn(S, sum(splits), rank, generator=g) * 0.1).half()
    y = (torch.randn(T, sum(splits), generator=g)).half()
    s = torch.rand(S, generator=g) * 2 + 0.25
    if ids is None:
        ids = torch.randint(-1, S, (T,), generator=g)
    return x, y, a, b, s, ids


def exact(x, y, a, b, s, ids, splits):
    """(values, bounds) in 64 bits.

    h_j: K products, exact in fp32, summed in fp32: (K + 16) 2^-23 (|a| |x|)_j at most (a matrix
    instruction may drop what lies below the last place instead of rounding: twice 2^-24).
    As hi + lo: 2^-22 of |h_j|, and the last place of lo, 2^-24 where the largest is 2^8: 2^-32
    of max |h|.  Then 2 rank products and sums, the scaling and the sum with y in fp32, and the
    rounding to fp16: half a step, 2^-11 of the value, 2^-25 among subnormal numbers."""
    T, K, rank = x.shape[0], x.shape[1], b.shape[2]
    out, tol = y.double().clone(), torch.zeros(y.shape, dtype=torch.float64)
    for t in range(T):
        e = int(ids[t])
        if not 0 <= e < a.shape[0]:
            continue
        xt = x[t].double()
        h, habs = a[e].double() @ xt, a[e].double().abs() @ xt.abs()
        scale, n = float(s[e]) if s is not None else 1.0, 0
        for p, wide in enumerate(splits):
            hp, hb = h[p * rank:(p + 1) * rank], habs[p * rank:(p + 1) * rank]
            bp = b[e, n:n + wide].double()
            d = scale * (bp @ hp)
            out[t, n:n + wide] += d
            dh = (K + 16) * 2.0 ** -23 * hb + 2.0 ** -22 * hp.abs() + 2.0 ** -32 * hp.abs().max()
            err = abs(scale) * (bp.abs() @ (dh + (2 * rank + 8) * 2.0 ** -23 * (hp.abs() + dh)))
            tol[t, n:n + wide] = err + 2.0 ** -23 * (y[t, n:n + wide].double().abs() + d.abs())
            n += wide
    return out, tol * 1.001 + 2.0 ** -11 * (out.abs() + tol) + 2.0 ** -25


def check(pkg, x, y, a, b, s, ids, splits, **kw):
    S = a.shape[0]
    dev = [None if t is None else t.cuda() for t in (x, y, a, b, s, ids)]
    x_, y_, a_, b_, s_, ids_ = dev
    plan = pkg.lora_plan(ids_, S)
    got = pkg.lora_add(y_, x_, a_, b_, plan, scaling=s_, splits=splits)
    assert torch.equal(y_.cpu(), y)
    want, tol = exact(x, y, a, b, s, ids, splits)
    err = (got.cpu().double() - want).abs()
    assert (err <= tol).all(), float((err / tol).max())
    bare = (ids < 0) | (ids >= S)
    assert torch.equal(got.cpu()[bare], y[bare])
    place = y_.clone()
    assert pkg.lora_add(place, x_, a_, b_, plan, scaling=s_, splits=splits, out=place) is place
    assert torch.equal(place, got)                       # same bits, in place and run by run
    return got


@pytest.mark.parametrize("T,K,splits,rank,S", [
    (1, 8, [1], 8, 1), (1, 4096, [4096, 1024, 1024], 16, 8), (2, 64, [16, 24], 16, 3),
    (5, 20, [37], 8, 2), (16, 1000, [520, 88], 24, 4), (17, 36, [3, 5, 7], 8, 5),
    (33, 4096, [768], 64, 2), (48, 512, [640, 640], 16, 48), (7, 12288, [264], 128, 3),
    (20, 256, [250], 136, 2), (9, 128, [65], 256, 3), (70, 100, [31], 40, 90),
    (260, 64, [129], 8, 1), (300, 1024, [2048 // 4, 100], 32, 3), (513, 200, [64], 48, 2),
    (700, 72, [513], 72, 4), (400, 48, [96], 256, 2), (1030, 40, [40], 16, 16),
    (2100, 33, [50], 8, 3), (64, 31, [8] * 8, 8, 2), (330, 7, [9], 200, 1)])
def test_shapes(pkg, cuda, T, K, splits, rank, S):
    check(pkg, *make(T, K, splits, rank, S, seed=T + K), splits)


@pytest.mark.parametrize("splits", [[128, 64], [72, 60], [2048 + 64]])
@pytest.mark.parametrize("K,rank", [(8, 8), (136, 32), (264, 40), (130, 72), (512, 136), (96, 256)])
def test_large_batches(pkg, cuda, K, rank, splits):
    """Tiles of 64 tokens: each step of the rank, whole strips and parts of them, chunks of K that
    are whole and not, several parts of K; an adapter with one token, and one with none."""
    g = torch.Generator().manual_seed(rank)
    ids = torch.randint(-1, 3, (1100,), generator=g)
    ids[500] = 3
    check(pkg, *make(1100, K, splits, rank, 5, seed=K + rank, ids=ids), splits)


@pytest.mark.parametrize("T", [3, 70, 600])
def test_ids_of_every_kind(pkg, cuda, T):
    """No token with an adapter, one adapter for all, one of many used, ids outside the range."""
    rng = random.Random(T)
    for ids in ([-1] * T, [0] * T, [4] * T, [rng.choice((-9, 5, 2 ** 31 - 1, 3)) for _ in range(T)],
                [i % 5 for i in range(T)], [-1] * (T - 1) + [2]):
        ids = torch.tensor(ids, dtype=torch.int32)
        check(pkg, *make(T, 136, [48, 16], 16, 5, seed=1, ids=ids), [48, 16])
    ids = torch.tensor([2 ** 40, -2 ** 40, 1] * (T // 3), dtype=torch.int64)
    check(pkg, *make(len(ids), 136, [48, 16], 16, 5, seed=1, ids=ids), [48, 16])


def test_without_scaling_and_with_extreme_values(pkg, cuda):
    x, y, a, b, s, ids = make(40, 64, [72], 16, 3, seed=4)
    check(pkg, x, y, a, b, None, ids, [72])
    # low-rank rows beyond the range of fp16 and far below it
    check(pkg, x * 300, y, (a.float() * 100).half(), (b.float() * 1e-3).half(), s * 1e-4, ids, [72])
    check(pkg, (x.float() * 1e-3).half(), y, (a.float() * 1e-2).half(), b, s * 1e4, ids, [72])
    check(pkg, x, torch.zeros_like(y), a, torch.zeros_like(b), s, ids, [72])
    check(pkg, torch.zeros_like(x), y, a, b, s, ids, [72])


def test_infinite_and_nan_rows_stay_their_own(pkg, cuda):
    x, y, a, b, s, ids = make(20, 64, [72], 16, 3, seed=4)
    ids = torch.arange(20) % 3
    clean = check(pkg, x, y, a, b, s, ids, [72])
    x[3, 5], x[8, 0], x[13, 63] = math.nan, math.inf, -math.inf
    y[6, 1] = math.nan
    got = pkg.lora_add(y.cuda(), x.cuda(), a.cuda(), b.cuda(), pkg.lora_plan(ids.cuda(), 3),
                       scaling=s.cuda())
    sick = torch.zeros(20, dtype=torch.bool)
    sick[[3, 8, 13]] = True
    assert not got.cpu()[sick].isfinite().any() and got[3].isnan().all()
    assert got[6, 1].isnan() and torch.equal(got[6, 2:], clean[6, 2:])
    sick[6] = True
    assert torch.equal(got.cpu()[~sick], clean.cpu()[~sick])


def test_strided_rows(pkg, cuda):
    """Rows of wider tensors, aligned and not, in place and not; what lies around stays."""
    T, K, N, S = 50, 72, 56, 3
    for off in (0, 8, 1, 3):
        x, y, a, b, s, ids = make(T, K, [40, 16], 8, S, seed=off)
        plan = pkg.lora_plan(ids.cuda(), S)
        want = pkg.lora_add(y.cuda(), x.cuda(), a.cuda(), b.cuda(), plan, s.cuda(), [40, 16])
        wx = torch.full((T, K + 16 + off), math.nan, dtype=torch.float16, device="cuda")
        wx[:, off:off + K] = x.cuda()
        wy = torch.full((T, N + 24), 7.0, dtype=torch.float16, device="cuda")
        wy[:, off:off + N] = y.cuda()
        vx, vy = wx[:, off:off + K], wy[:, off:off + N]
        got = pkg.lora_add(vy, vx, a.cuda(), b.cuda(), plan, s.cuda(), [40, 16])
        assert torch.equal(got, want) and got.is_contiguous()
        pkg.lora_add(vy, vx, a.cuda(), b.cuda(), plan, s.cuda(), [40, 16], out=vy)
        assert torch.equal(vy, want)
        rest = torch.ones(N + 24, dtype=torch.bool)
        rest[off:off + N] = False
        assert (wy[:, rest.cuda()] == 7).all()
        three = pkg.lora_add(y.cuda().view(5, 10, N), x.cuda().view(5, 10, K), a.cuda(), b.cuda(),
                             plan, s.cuda(), [40, 16])
        assert torch.equal(three.view(T, N), want)


def test_captured_in_a_graph_with_another_plan_each_time(pkg, cuda):
    T, S = 24, 6
    x, y, a, b, s, ids = (t.cuda() for t in make(T, 512, [256, 128], 16, S, seed=7))
    plan = pkg.lora_plan(ids, S)
    pkg.lora_add(y, x, a, b, plan, s, [256, 128])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = pkg.lora_add(y, x, a, b, plan, s, [256, 128])
    for rep in range(4):
        x.copy_(torch.randn_like(x))
        new = pkg.lora_plan(torch.randint(-1, S, (T,), device="cuda"), S)
        plan.seg_off.copy_(new.seg_off)
        plan.rows.copy_(new.rows)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, pkg.lora_add(y, x, a, b, new, s, [256, 128])), rep


def test_two_streams_at_once(pkg, cuda):
    """Two calls that overlap have workspaces of their own."""
    args = [[t.cuda() for t in make(300, 1024, [512], 16, 4, seed=i)] for i in range(2)]
    plans = [pkg.lora_plan(v[5], 4) for v in args]
    want = [pkg.lora_add(v[1], v[0], v[2], v[3], p, v[4]) for v, p in zip(args, plans)]
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(20):
        for i, st in enumerate(sides):
            with torch.cuda.stream(st):
                v = args[i]
                outs[i].append(pkg.lora_add(v[1], v[0], v[2], v[3], plans[i], v[4]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])


def test_rows_far_apart(pkg, cuda):
    """Offsets past 2^31 elements in x, y and out."""
    ld = 2 ** 30 + 8
    bx, by = (torch.zeros(2 * ld + 256, dtype=torch.float16, device="cuda") for _ in range(2))
    x, y, a, b, s, _ = make(3, 64, [96], 8, 2, seed=3)
    vx, vy = bx.as_strided((3, 64), (ld, 1)), by.as_strided((3, 96), (ld, 1))
    vx.copy_(x)
    vy.copy_(y)
    plan = pkg.lora_plan(torch.tensor([1, 0, 1], device="cuda"), 2)
    want = pkg.lora_add(y.cuda(), x.cuda(), a.cuda(), b.cuda(), plan, s.cuda())
    pkg.lora_add(vy, vx, a.cuda(), b.cuda(), plan, s.cuda(), out=vy)
    assert torch.equal(vy, want)


def test_no_tokens(pkg, cuda):
    x, y, a, b, s, ids = make(0, 64, [96], 8, 2, seed=3)
    plan = pkg.lora_plan(ids.cuda(), 2)
    assert pkg.lora_add(y.cuda(), x.cuda(), a.cuda(), b.cuda(), plan, s.cuda()).shape == (0, 96)


@pytest.mark.parametrize("T,K,splits,rank,S", [
    (1, 64, [72], 8, 2), (40, 136, [48, 16], 16, 5), (70, 100, [31, 8, 9], 40, 6),
    (50, 72, [65], 136, 3), (1100, 136, [128, 64], 32, 5), (1100, 96, [72, 60], 72, 4),
    (1100, 264, [64], 256, 3)])
def test_ranks_of_their_own(pkg, cuda, T, K, splits, rank, S):
    """What a's filled-up rows hold, and what they make of infinities, is not looked at."""
    x, y, a, b, s, ids = make(T, K, splits, rank, S, seed=T + rank)
    rng = random.Random(rank)
    own = torch.tensor([[rng.choice((-3, 0, 1, rng.randint(1, rank), rank - 1, rank, rank + 5))
                         for _ in splits] for _ in range(S)], dtype=torch.int32)
    own[0, 0] = 0                                         # and one with nothing at all
    own[S - 1] = 0
    for e in range(S):
        n = 0
        for p, wide in enumerate(splits):
            r = min(max(int(own[e, p]), 0), rank)
            a[e, p * rank + r:(p + 1) * rank] = 0
            b[e, n:n + wide, r:] = 0
            n += wide
    want = check(pkg, x, y, a, b, s, ids, splits)
    plan = pkg.lora_plan(ids.cuda(), S)
    bad = a.clone()
    for e in range(S):
        for p in range(len(splits)):
            bad[e, p * rank + min(max(int(own[e, p]), 0), rank):(p + 1) * rank] = math.nan
    dev = [t.cuda() for t in (y, x, bad, b)]
    got = pkg.lora_add(*dev, plan, s.cuda(), splits, ranks=own.cuda())
    assert torch.equal(got, want)
    place = y.cuda()
    pkg.lora_add(place, *dev[1:], plan, s.cuda(), splits, out=place, ranks=own.cuda())
    assert torch.equal(place, want)
    x[::3, K // 2] = math.inf
    got = pkg.lora_add(y.cuda(), x.cuda(), a.cuda(), b.cuda(), plan, s.cuda(), splits,
                       ranks=own.cuda()).cpu()
    for t in range(0, T, 3):
        n = 0
        for p, wide in enumerate(splits):
            e = int(ids[t])
            if not 0 <= e < S or own[e, p] <= 0:
                assert torch.equal(got[t, n:n + wide], y[t, n:n + wide]), (t, p)
            else:
                assert not got[t, n:n + wide].isfinite().any(), (t, p)
            n += wide
    clean = torch.arange(T) % 3 != 0
    assert torch.equal(got[clean], want.cpu()[clean])


@pytest.mark.parametrize("T", [5, 1100])
def test_finite_values_beside_an_infinite_one(pkg, cuda, T):
    """A low-rank value that overflows 32 bits, others that are finite but beyond fp16: the row is
    infinite with that one's sign, not the difference of two infinities."""
    h = torch.float16
    x = torch.ones(T, 8, dtype=h)
    a, b = torch.zeros(1, 8, 8, dtype=h), torch.zeros(1, 64, 8, dtype=h)
    a[0, 0, 0], a[0, 1, 0], a[0, 2, 0] = 2.0, 0.5, 2.0 ** -14
    b[0, :, 0] = torch.where(torch.arange(64) % 2 == 0, 1.0, -1.0)
    b[0, :, 1] = -b[0, :, 0]
    b[0, :, 2] = 3.0
    s, y = torch.tensor([3e38]), torch.randn(T, 64).half()
    got = pkg.lora_add(y.cuda(), x.cuda(), a.cuda(), b.cuda(),
                       pkg.lora_plan(torch.zeros(T, dtype=torch.int32, device="cuda"), 1), s.cuda())
    assert torch.equal(got.cpu(), (b[0, :, 0].float() * math.inf).half().expand(T, 64))


@pytest.mark.parametrize("T", [3, 1100])
def test_out_beside_y_in_the_same_rows(pkg, cuda, T):
    """y and out as two column ranges of one tensor are other memory; shifted views are refused."""
    x, y, a, b, s, ids = make(T, 72, [40, 16], 8, 3, seed=T)
    plan = pkg.lora_plan(ids.cuda(), 3)
    want = pkg.lora_add(y.cuda(), x.cuda(), a.cuda(), b.cuda(), plan, s.cuda(), [40, 16])
    wide = torch.zeros(T, 120, dtype=torch.float16, device="cuda")
    vy, vo = wide[:, 4:60], wide[:, 60:116]
    vy.copy_(y)
    assert pkg.lora_add(vy, x.cuda(), a.cuda(), b.cuda(), plan, s.cuda(), [40, 16], out=vo) is vo
    assert torch.equal(vo, want) and torch.equal(vy.cpu(), y)
    for bad in (wide[:, 5:61], wide[:, 59:115], wide.view(-1)[4:4 + T * 56].view(T, 56)):
        with pytest.raises((ValueError, RuntimeError), match="overlaps|other strides"):
            pkg.lora_add(vy, x.cuda(), a.cuda(), b.cuda(), plan, s.cuda(), [40, 16], out=bad)


@pytest.mark.parametrize("splits", [[512], [2048], [4608, 512], [2500, 2500, 130]])
def test_large_batches_of_every_width(pkg, cuda, splits):
    """Tiles of 64 tokens with a workgroup for 256 columns and for 512, whole strips and not."""
    check(pkg, *make(2100, 40, splits, 8, 3, seed=sum(splits)), splits)


@pytest.mark.parametrize("T,S", [(1100, 200), (1024, 1024), (1500, 3000)])
def test_large_batches_of_many_adapters(pkg, cuda, T, S):
    """Tiles of 64 tokens with a few tokens each, slots without any among them."""
    check(pkg, *make(T, 40, [72, 24], 8, S, seed=S), [72, 24])
    g = torch.Generator().manual_seed(S)
    ids = torch.randint(0, 7, (T,), generator=g) * (S // 7)
    check(pkg, *make(T, 136, [64], 16, S, seed=S + 1, ids=ids), [64])
