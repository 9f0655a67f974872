"""sample() against its definition in 64 bits (sample_ref): tokens are equal, log-probabilities
within the rounding of their last step.

Tokens: a running sum is off by less than n * 2^-45 of the largest weight (integer weights,
n <= 151936) and 2^-38 of itself (the weights' polynomial), so a random u picks another token than the 64-bit sums with a chance below
151936 * 2^-27 / 2^17 a row at the worst and about 1e-8 for the rows here; u on a border is
tested where weights are equal, and sums exact on both sides.
Log-probabilities: power and log in 64 bits, one rounding to fp32: 2^-24 relative, and the
kept mass is off by less than 2^-27 of itself: 2^-26 absolute covers that twice over."""
import math
import random

import numpy as np
import pytest
import torch

from sample_ref import sample_row

pytestmark = pytest.mark.gpu

SETTINGS = [dict(temperature=0.0), dict(temperature=1.0), dict(temperature=0.6, top_k=20, top_p=0.95),
            dict(temperature=0.8, top_p=0.9), dict(temperature=1.3, min_p=0.05),
            dict(temperature=0.7, top_k=300), dict(temperature=1.5, top_p=0.99),
            dict(temperature=1.0, top_k=50, top_p=0.7, min_p=0.02), dict(top_k=1), dict(top_p=0.0),
            dict(temperature=1e-6), dict(temperature=20.0, top_p=0.999), dict(min_p=1.0)]


def expected(x, u, **kw):
    x = x.double().cpu().numpy()
    B = x.shape[0]
    u = [0.0] * B if u is None else u.double().cpu().tolist()
    get = lambda n, d: (kw[n].tolist() if torch.is_tensor(kw.get(n)) else  # noqa: E731
                        [float(np.float32(kw.get(n, d))) if n != "top_k" else kw.get(n, d)] * B)
    t, k, p, m = get("temperature", 1.0), get("top_k", 0), get("top_p", 1.0), get("min_p", 0.0)
    return [sample_row(x[i], u[i], t[i], k[i], p[i], m[i]) for i in range(B)]


def check(pkg, x, u, **kw):
    got, logp = pkg.sample(x, u, return_logprobs=True, **kw)
    want = expected(x, u, **kw)
    assert got.dtype == torch.int64 and got.shape == x.shape[:-1]
    assert got.tolist() == [w[0] for w in want]
    lp = np.array([w[1] for w in want])
    g = logp.double().cpu().numpy()
    assert np.array_equal(np.isnan(g), np.isnan(lp))
    ok = ~np.isnan(lp)
    assert (np.abs(g - lp)[ok] <= 2.0 ** -24 * np.abs(lp[ok]) + 2.0 ** -26).all()
    assert torch.equal(pkg.sample(x, u, **kw), got)


def logits(rows, V, seed, fp32=False, spread=2.5, peaks=8):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, V, generator=g) * spread
    at = torch.randint(0, V, (rows, peaks), generator=g)
    x.scatter_add_(1, at, torch.rand(rows, peaks, generator=g) * 8 + 2)
    u = torch.rand(rows, generator=g)
    return (x if fp32 else x.half()).cuda(), u.cuda()


@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("V", [1, 2, 7, 64, 65, 1000, 1024, 1025, 4099, 50257, 151936, 200003])
def test_sizes(pkg, cuda, V, fp32):
    for i, kw in enumerate(SETTINGS):
        x, u = logits(3, V, seed=V + i, fp32=fp32)
        check(pkg, x, u, **kw)


@pytest.mark.parametrize("rows", [1, 2, 17, 100, 300])
def test_rows_with_their_own_settings(pkg, cuda, rows):
    rng = random.Random(rows)
    x, u = logits(rows, 5003, seed=rows)
    pick = [rng.choice(SETTINGS) for _ in range(rows)]
    col = lambda n, d, t: torch.tensor([s.get(n, d) for s in pick], dtype=t, device="cuda")  # noqa: E731
    check(pkg, x, u, temperature=col("temperature", 1.0, torch.float32),
          top_k=col("top_k", 0, torch.int32), top_p=col("top_p", 1.0, torch.float32),
          min_p=col("min_p", 0.0, torch.float32))
    check(pkg, x, u, temperature=0.9, top_k=col("top_k", 0, torch.int64), top_p=0.97)


@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("V", [10, 1000, 40000, 151936])
@pytest.mark.parametrize("levels", [1, 2, 5])
def test_equal_logits(pkg, cuda, V, levels, fp32):
    """Few distinct values: cuts fall among equal logits, and u on the borders between them."""
    g = torch.Generator().manual_seed(V + levels)
    x = torch.randint(0, levels, (6, V), generator=g).float()
    x = (x if fp32 else x.half()).cuda()
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.3, 1 - 2.0 ** -24], device="cuda")
    if levels == 1:  # all weights are 1 and every sum is exact
        for kw in (dict(), dict(top_k=V // 2), dict(top_p=0.5), dict(top_p=0.25, top_k=V // 2),
                   dict(min_p=0.5), dict(top_k=3), dict(temperature=0.0)):
            check(pkg, x, u, **kw)
    for kw in (dict(top_k=V // 3 + 1, temperature=0.7), dict(top_p=0.4), dict(top_k=2, top_p=0.9),
               dict(top_k=max(1, V // levels), top_p=0.6, min_p=0.01)):
        check(pkg, x, torch.rand(6, generator=g).cuda(), **kw)


def test_minus_zero_equals_zero(pkg, cuda):
    for dt in (torch.float16, torch.float32):
        x = torch.tensor([[-0.0, 0.0, -1.0], [0.0, -0.0, -1.0]], dtype=dt, device="cuda")
        u = torch.tensor([0.0, 0.0], device="cuda")
        assert pkg.sample(x, temperature=0.0).tolist() == [0, 0]
        assert pkg.sample(x, u, top_k=1).tolist() == [0, 0]


@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("V", [9, 1300, 70001])
def test_masked_infinite_and_nan_rows(pkg, cuda, V, fp32):
    x, u = logits(9, V, seed=5, fp32=fp32)
    x[0, :] = -math.inf                        # nothing to draw
    x[1, :] = -math.inf
    x[1, V // 2] = -3.0                        # one token left
    x[2, torch.rand(V) < 0.97] = -math.inf     # a grammar's mask
    x[2, V - 1] = 1.0
    x[3, V // 3] = math.nan
    x[4, [1, V - 2]] = math.inf                # two plus infinities share the mass
    x[5, 0] = torch.finfo(x.dtype).max
    x[5, 1:] = torch.finfo(x.dtype).min        # a mask of the type's lowest value
    x[6, :] = torch.finfo(x.dtype).min
    x[7, :] = math.inf
    x[8, 0] = -math.nan
    for kw in SETTINGS:
        check(pkg, x, u, **kw)


def test_random_numbers_and_settings_outside_their_range(pkg, cuda):
    x, _ = logits(8, 1000, seed=11)
    u = torch.tensor([0.0, -1.0, 1.0, 2.0, math.nan, math.inf, -math.inf, 1e-30], device="cuda")
    for kw in (dict(), dict(top_k=10), dict(top_p=0.9), dict(min_p=0.1)):
        check(pkg, x, u, **kw)
    u = torch.rand(8, device="cuda")
    f = lambda *v: torch.tensor(v, device="cuda")  # noqa: E731
    check(pkg, x, u, temperature=f(0.0, -1.0, math.nan, math.inf, 1e-38, 1e-45, 3e38, 1.0))
    check(pkg, x, u, top_p=f(0.0, -1.0, 1.0, 2.0, math.inf, -math.inf, 1e-30, 0.5))
    check(pkg, x, u, min_p=f(0.0, -1.0, 1.0, 2.0, math.inf, -math.inf, 1e-30, 0.5))
    check(pkg, x, u, top_k=torch.tensor([0, -5, 1, 1000, 1001, 2 ** 31 - 1, 999, 2], device="cuda"))


@pytest.mark.parametrize("fp32", [False, True])
def test_strides_shapes_and_streams(pkg, cuda, fp32):
    wide, u = logits(12, 3011, seed=2, fp32=fp32)
    for lo, hi in ((0, 3000), (1, 3001), (3, 3011), (8, 3000)):
        check(pkg, wide[:, lo:hi], u, temperature=0.8, top_p=0.9)
    check(pkg, wide[::3, 5:2000], u[::3], top_k=7)
    x = wide.view(3, 4, 3011)
    got = pkg.sample(x, u.view(3, 4), top_k=40)
    assert got.shape == (3, 4) and torch.equal(got.flatten(), pkg.sample(wide, u, top_k=40))
    turned = wide.t().contiguous().t()                      # columns, not rows, in memory
    assert torch.equal(pkg.sample(turned, u, top_k=40), got.flatten())
    one = pkg.sample(wide[0], u[0], top_k=40)
    assert one.shape == () and one == got[0, 0]
    assert pkg.sample(wide[:0], u[:0]).shape == (0,)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = pkg.sample(wide, u, top_k=40)
    side.synchronize()
    assert torch.equal(other, got.flatten())


def test_captured_in_a_graph(pkg, cuda):
    """Replays read the logits, numbers and settings that their tensors hold then."""
    x, u = logits(20, 30011, seed=3)
    t = torch.full((20,), 0.8, device="cuda")
    k = torch.full((20,), 50, dtype=torch.int32, device="cuda")
    p = torch.full((20,), 0.9, device="cuda")
    pkg.sample(x, u, t, k, p)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, logp = pkg.sample(x, u, t, k, p, return_logprobs=True)
    for rep in range(4):
        x2, u2 = logits(20, 30011, seed=30 + rep)
        x.copy_(x2)
        u.copy_(u2)
        k.copy_(torch.randint(0, 60, (20,)))
        p.copy_(torch.rand(20))
        t.copy_(torch.rand(20) * (rep > 0))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        want, wantp = pkg.sample(x, u, t, k, p, return_logprobs=True)
        assert torch.equal(out, want) and torch.equal(logp, wantp), rep
        assert out.tolist() == [w[0] for w in expected(x, u, temperature=t, top_k=k, top_p=p)]


def test_rows_far_apart(pkg, cuda):
    """Row offsets past 2^31 elements."""
    ld = 2 ** 30 + 24
    buf = torch.zeros(2 * ld + 1000, dtype=torch.float16, device="cuda")
    x = buf.as_strided((3, 1000), (ld, 1))
    src, u = logits(3, 1000, seed=9)
    x.copy_(src)
    assert torch.equal(pkg.sample(x, u, top_p=0.9), pkg.sample(src, u, top_p=0.9))


@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("spread,kw", [
    (1.0, dict(temperature=1.5, top_p=0.98)), (0.3, dict(top_p=0.999999)), (1.0, dict(top_k=5000)),
    (2.0, dict(top_k=1500, top_p=0.5)), (1.0, dict(top_k=40000, top_p=0.9, min_p=1e-3)),
    (0.01, dict(top_p=0.5)), (0.01, dict(top_k=77777)), (1.0, dict(min_p=0.03)),
    (3.0, dict(min_p=1e-12)), (1.0, dict(top_p=0.97, min_p=0.2)), (2.0, dict(top_k=700)),
    (2.5, dict(top_k=1000, top_p=0.999, min_p=0.01)), (4.0, dict(temperature=0.3, top_k=100000)),
    (1.0, dict(top_k=600, min_p=0.5)), (1.5, dict(top_k=60, top_p=0.97, min_p=0.6))])
def test_long_prefixes(pkg, cuda, spread, kw, fp32):
    """Kept prefixes from dozens of tokens to most of the vocabulary."""
    for V, peaks in ((151936, 0), (100003, 5)):
        x, u = logits(4, V, seed=V + peaks, fp32=fp32, spread=spread, peaks=max(peaks, 1))
        check(pkg, x, u, **kw)


def test_neighbouring_peaks(pkg, cuda):
    """The tokens that matter side by side, in one group of a thread or in one part."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(6, 60000, generator=g).half()
    x[0, 800:804] = 15.0
    x[1, 800:832] = torch.linspace(14, 15, 32).half()
    x[2, [100, 2148, 4196, 6244]] = 15.0       # the four vectors of one thread
    x[3, 8190:8194] = 15.0                     # across a border of parts
    x[4, 59992:60000] = 15.0                   # the end of the row
    x[5, 0:8] = torch.linspace(15, 12, 8).half()
    for kw in (dict(top_p=0.95), dict(top_k=3), dict(top_k=20, top_p=0.9), dict(min_p=0.3), dict(),
               dict(top_p=0.9999), dict(temperature=0.0)):
        for seed in range(3):
            check(pkg, x.cuda(), torch.rand(6, generator=g).cuda(), **kw)


def test_a_row_is_the_same_in_every_batch(pkg, cuda):
    x, u = logits(300, 20011, seed=8)
    for kw in (dict(), dict(top_p=0.9), dict(top_k=40)):
        got, logp = pkg.sample(x, u, return_logprobs=True, **kw)
        for i in (0, 7, 299):
            one, logp1 = pkg.sample(x[i:i + 1], u[i:i + 1], return_logprobs=True, **kw)
            assert one[0] == got[i] and logp1[0] == logp[i]


def test_the_longest_rows(pkg, cuda):
    """2^22 logits, 512 parts; one more is refused."""
    x, u = logits(2, 2 ** 22, seed=12, spread=1.5, peaks=3)
    x[1, 2 ** 22 - 1] = 20.0
    for kw in (dict(temperature=0.0), dict(), dict(top_p=0.9), dict(top_k=50, top_p=0.9),
               dict(min_p=0.01)):
        check(pkg, x, u, **kw)
    with pytest.raises((ValueError, RuntimeError)):
        pkg.sample(torch.zeros(1, 2 ** 22 + 1, dtype=torch.float16, device="cuda"), u[:1])


@pytest.mark.parametrize("kw", [dict(), dict(top_p=0.9), dict(top_k=5), dict(min_p=0.1)])
def test_many_rows(pkg, cuda, kw):
    x, u = logits(3000, 131, seed=13)
    check(pkg, x, u, **kw)


@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("low", [-30.0, -6.0, 6.0])
def test_rows_with_a_pattern(pkg, cuda, low, fp32):
    """Places in every eight (or every 32) that are all lower, or all higher, than the others: what
    a few of a group's logits tell of the row is wrong."""
    g = torch.Generator().manual_seed(14)
    x = torch.randn(6, 120000, generator=g)
    i = torch.arange(120000)
    for row, at in enumerate(([1], [6], [1, 6], [0, 2, 3, 4, 5, 7])):
        x[row, (i[:, None] % 8 == torch.tensor(at)).any(1)] += low
    x[4, i // 2048 % 4 == 1] += low
    x[5, i % 8192 < 4096] += low
    x = (x if fp32 else x.half()).cuda()
    for kw in (dict(top_p=0.9), dict(top_p=0.5), dict(top_p=0.99, temperature=2.0), dict(min_p=0.02)):
        check(pkg, x, torch.rand(6, generator=g).cuda(), **kw)


def test_two_streams_at_once(pkg, cuda):
    work = [logits(40, 50257, seed=50 + i) for i in range(2)]
    want = [pkg.sample(x, u, temperature=1.2, top_p=0.98) for x, u in work]
    sides = [torch.cuda.Stream() for _ in work]
    torch.cuda.synchronize()
    got = [[], []]
    for rep in range(5):
        for i, s in enumerate(sides):
            with torch.cuda.stream(s):
                got[i].append(pkg.sample(*work[i], temperature=1.2, top_p=0.98))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(t, want[i]) for t in got[i])


def test_more_parts_than_workgroups(pkg, cuda):
    """540000 rows of two parts each: workgroups take more than one part."""
    B, V = 540000, 8200
    x = torch.empty(B, V, dtype=torch.float16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(7))
    u = torch.rand(B, device="cuda", generator=torch.Generator("cuda").manual_seed(8))
    got = pkg.sample(x, temperature=0.0)
    assert torch.equal(x.gather(1, got[:, None])[:, 0], x.amax(1))
    some = torch.cat([torch.arange(0, 4), torch.arange(524286, 524290), torch.arange(B - 4, B)])
    assert got[some.cuda()].tolist() == x[some.cuda()].argmax(1).tolist()
    for kw in (dict(top_p=0.8), dict()):
        got = pkg.sample(x, u, **kw)[some.cuda()].tolist()
        assert got == [w[0] for w in expected(x[some.cuda()], u[some.cuda()], **kw)]
    del x
    torch.cuda.empty_cache()


def test_many_long_prefixes_at_once(pkg, cuda):
    """Flat rows under top-p, for whose prefix no list is tried: more workgroups than the device
    holds, so that their waves run apart.  Every wave has to go the same way."""
    x, u = logits(1500, 20011, seed=15, spread=1.0, peaks=1)
    kw = dict(temperature=1.5, top_p=0.95)
    got, logp = pkg.sample(x, u, return_logprobs=True, **kw)
    some = torch.arange(0, 1500, 53, device="cuda")
    assert got[some].tolist() == [w[0] for w in expected(x[some], u[some], **kw)]
    for _ in range(3):
        again, logp2 = pkg.sample(x, u, return_logprobs=True, **kw)
        assert torch.equal(again, got) and torch.equal(logp2, logp)


@pytest.mark.parametrize("fp32", [False, True])
def test_rows_that_take_turns_in_the_workspace(pkg, cuda, fp32):
    """More rows than 1 GiB of workspace holds: each has its own logits, number and settings."""
    B, V = 16500, 8200
    x, u = logits(B, V, seed=16, fp32=fp32)
    rng = random.Random(17)
    pick = [rng.choice(SETTINGS) for _ in range(B)]
    col = lambda n, d, t: torch.tensor([s.get(n, d) for s in pick], dtype=t, device="cuda")  # noqa: E731
    kw = dict(temperature=col("temperature", 1.0, torch.float32), top_k=col("top_k", 0, torch.int32),
              top_p=col("top_p", 1.0, torch.float32), min_p=col("min_p", 0.0, torch.float32))
    got, logp = pkg.sample(x, u, return_logprobs=True, **kw)
    at = torch.cat([torch.arange(0, B, 211), torch.arange(15000, 15400, 7), torch.arange(B - 5, B)]).cuda()
    some = {n: t[at] for n, t in kw.items()}
    assert got[at].tolist() == [w[0] for w in expected(x[at], u[at], **some)]
    for lo, hi in ((0, 300), (15100, 15400), (B - 300, B)):
        part, logp2 = pkg.sample(x[lo:hi], u[lo:hi], return_logprobs=True,
                                 **{n: t[lo:hi] for n, t in kw.items()})
        assert torch.equal(part, got[lo:hi]) and torch.equal(logp2, logp[lo:hi])
    assert torch.equal(pkg.sample(x, temperature=0.0), x.argmax(-1))
