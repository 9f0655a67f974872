"""Attention of new tokens over the paged cache on the GPU, against its plain form in 64
bits."""
import math

import pytest
import torch

import attention_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(pkg):
    return pkg.ops


def _starts(new):
    s = [0]
    for n in new:
        s.append(s[-1] + n)
    return s


def _q(T, Hq, D, seed, size=1.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, Hq, D, generator=g) * size).half()


def _run(ops, q, cache, lens, starts, most=None, cu=True, **kw):
    k, v, ks, vs, tables = cache
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    return ops.paged_attention(
        q.cuda(), dev(k), dev(v), dev(tables), torch.tensor(lens, dtype=torch.int32).cuda(),
        torch.tensor(starts, dtype=torch.int32).cuda() if cu else None, max_seqlen=most,
        k_scale=dev(ks), v_scale=dev(vs), **kw)


def _check(ops, new, lens, Hq, Hk, D, page, int8=False, most="max", seed=0, cu=True, **kw):
    q, starts = _q(sum(new), Hq, D, seed + 1), _starts(new)
    cache = ref.paged(lens, page, Hk, D, seed, int8)
    got = _run(ops, q, cache, lens, starts, max(new) if most == "max" else most, cu, **kw)
    k, v, ks, vs, tables = cache
    want, tol = ref.attention(q, k, v, tables, lens, starts, ks, vs, **kw)
    ref.within(got, want, tol)
    return got


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("Hq,Hk,D,page", [(16, 8, 128, 16), (32, 4, 128, 64), (4, 1, 64, 32),
                                          (5, 1, 80, 16), (3, 3, 96, 128), (16, 1, 256, 16),
                                          (8, 8, 16, 16), (40, 2, 128, 1024)])
def test_decode(ops, cuda, Hq, Hk, D, page, int8):
    """One token a sequence, lengths around the edges of pages and tiles, one token long too."""
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 700, 1025]
    _check(ops, [1] * len(lens), lens, Hq, Hk, D, page, int8, seed=D + page, cu=page != 64)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("lens", [[9000], [1], [4097, 3, 2500], [300] * 40])
def test_decode_long_and_few(ops, cuda, lens, int8):
    _check(ops, [1] * len(lens), lens, 8, 2, 128, 16, int8, seed=len(lens))


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("new,Hq,Hk,D", [([2] * 5, 8, 2, 128), ([5] * 4, 32, 8, 128),
                                         ([8, 1, 3, 7, 2], 4, 4, 64), ([3, 3], 20, 1, 96),
                                         ([4] * 3, 16, 1, 256), ([17, 16, 15], 4, 1, 128)])
def test_few_new_tokens(ops, cuda, new, Hq, Hk, D, int8):
    lens = [n + old for n, old in zip(new, (0, 700, 61, 64, 1))]
    _check(ops, new, lens, Hq, Hk, D, 16, int8, seed=Hq)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("new,old,Hq,Hk,D,page", [
    ([200], [0], 4, 2, 128, 16), ([333], [900], 8, 2, 128, 64), ([130, 64, 1, 257], [0, 64, 500, 3],
                                                                 4, 1, 64, 32),
    ([100, 77], [31, 0], 5, 1, 80, 16), ([129], [127], 2, 2, 256, 128), ([90], [10], 16, 1, 96, 16),
    ([64, 128, 256], [0, 0, 0], 2, 1, 16, 16)])
def test_chunks(ops, cuda, new, old, Hq, Hk, D, page, int8):
    _check(ops, new, [a + b for a, b in zip(new, old)], Hq, Hk, D, page, int8, seed=D + len(new))


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("new,old,window", [([300], [277], None), ([130, 1, 200, 3], [0, 500, 65, 9], None),
                                            ([260, 40], [100, 0], 70)])
def test_chunks_of_many_heads(ops, cuda, new, old, window, int8):
    """Rows for more workgroups than the CUs hold at once."""
    _check(ops, new, [a + b for a, b in zip(new, old)], 256, 32, 128, 32, int8, seed=len(new),
           window=window)


@pytest.mark.parametrize("window", [1, 2, 17, 64, 100, 5000])
def test_window(ops, cuda, window):
    _check(ops, [1, 1, 1], [5, 300, 1200], 4, 2, 128, 16, window=window)
    _check(ops, [200, 3, 1, 70], [200, 400, 513, 1000], 4, 2, 64, 32, window=window)
    _check(ops, [4, 4], [4, 999], 8, 2, 128, 16, int8=True, window=window)


@pytest.mark.parametrize("most", [None, 0, 1, 3, 10000])
def test_any_bound_of_new_tokens_gives_the_result(ops, cuda, most):
    _check(ops, [1, 150, 0, 4, 1, 33], [77, 150, 20, 4, 900, 50], 8, 2, 128, 16, most=most)


def test_sequences_without_tokens_and_padding(ops, cuda):
    """Sequences of no new or no tokens at all, queries before the first key (0), and tokens
    past the last sequence (0)."""
    new, lens = [0, 3, 0, 2, 5, 0], [0, 3, 40, 0, 2, 1]
    starts = _starts(new)
    q = _q(sum(new) + 7, 4, 64, 5)
    cache = ref.paged(lens, 16, 2, 64, 6)
    k, v, _, _, tables = cache
    want, tol = ref.attention(q, k, v, tables, lens, starts)
    for most in (5, None):
        got = _run(ops, q, cache, lens, starts, most)
        ref.within(got, want, tol)
        assert got[starts[-1]:].count_nonzero() == 0
        assert got[3:5].count_nonzero() == 0 and got[5:8].count_nonzero() == 0
    big = _q(300, 4, 64, 5)
    assert _run(ops, big, cache, lens, starts)[10:].count_nonzero() == 0


@pytest.mark.parametrize("new", [[1, 1], [2, 3], [100, 70]])
@pytest.mark.parametrize("int8", [False, True])
def test_what_lies_behind_a_sequence_is_not_seen(ops, cuda, new, int8):
    """NaN and infinities in the cache past a sequence's end, on pages it does not own and
    behind its window change nothing."""
    lens = [150, 333]
    q, starts = _q(sum(new), 4, 128, 8), _starts(new)
    k, v, ks, vs, tables = ref.paged(lens, 64, 2, 128, 9, int8)
    plain = _run(ops, q, (k, v, ks, vs, tables), lens, starts, window=90)
    own = torch.zeros(k.shape[0], 64, dtype=torch.bool)
    for s, L in enumerate(lens):
        for j in range(max(0, L - new[s] - 90 + 1), L):
            own[tables[s, j // 64], j % 64] = True
    other = ~own[:, None, :].expand(-1, 2, -1)
    if int8:
        ks, vs = ks.clone(), vs.clone()
        ks[other], vs[other] = math.nan, math.inf
    else:
        k, v = k.clone(), v.clone()
        k[other], v[other] = math.nan, math.inf
    tables = torch.cat([tables, torch.full((2, 3), 1 << 30, dtype=torch.int32)], 1)
    tables[:, 0] = torch.tensor([tables[0, 0], -7])  # the second one's window is past page 0
    assert torch.equal(_run(ops, q, (k, v, ks, vs, tables), lens, starts, window=90), plain)


@pytest.mark.parametrize("new", [3, 40, 150])
def test_values_of_later_tokens_stay_hidden(ops, cuda, new):
    """Infinities and NaN in a new token's own key and value reach it and the tokens after it,
    none before."""
    lens, starts = [new + 20], [0, new]
    q = _q(new, 4, 128, 3)
    k, v, _, _, tables = ref.paged(lens, 16, 2, 128, 4)
    clean = _run(ops, q, (k, v, None, None, tables), lens, starts)
    for cache, value in ((v, math.nan), (v, math.inf), (v, -math.inf), (k, math.nan)):
        at = 20 + new // 2
        kept = cache[tables[0, at // 16], 1, at % 16, 5].clone()
        cache[tables[0, at // 16], 1, at % 16, 5] = value
        got = _run(ops, q, (k, v, None, None, tables), lens, starts)
        cache[tables[0, at // 16], 1, at % 16, 5] = kept
        # equal but for the sign of a zero
        assert torch.equal(got[:new // 2], clean[:new // 2])
        assert torch.equal(got[:, :2], clean[:, :2])  # the other key head
        hit = got[new // 2:, 2:]
        if cache is k:
            assert hit.isnan().all()
        else:
            rest = torch.ones(128, dtype=torch.bool)
            rest[5] = False
            assert torch.equal(hit[..., rest], clean[new // 2:, 2:][..., rest])
            same = hit[..., 5].isnan() if math.isnan(value) else hit[..., 5] == value
            assert same.all()


def test_pages_outside_the_cache_give_nan(ops, cuda):
    lens, new = [100, 100, 40, 70], [1, 1, 1, 1]
    q, starts = _q(4, 4, 64, 1), _starts(new)
    k, v, _, _, tables = ref.paged(lens, 16, 2, 64, 2)
    want, tol = ref.attention(q, k, v, tables, lens, starts)
    tables[1, 3], tables[3, 0] = 1 << 30, -5
    want[1] = want[3] = math.nan
    ref.within(_run(ops, q, (k, v, None, None, tables), lens, starts), want, tol)
    # a length past the block table
    got = _run(ops, q, (k, v, None, None, tables[:, :5]), [80, 1 << 30, 40, 100], starts)
    assert got[1].isnan().all() and got[3].isnan().all() and got[0].isfinite().all()


def test_chunk_with_a_page_outside_the_cache(ops, cuda):
    lens, starts = [300], [0, 200]
    q = _q(200, 4, 128, 1)
    k, v, _, _, tables = ref.paged(lens, 16, 2, 128, 2)
    want, tol = ref.attention(q, k, v, tables, lens, starts)
    tables[0, 10] = k.shape[0]  # the first page past the cache
    want[60:] = math.nan  # tokens from 160 on see page 10
    ref.within(_run(ops, q, (k, v, None, None, tables), lens, starts), want, tol)


@pytest.mark.parametrize("size", [0.0, 30.0])
def test_flat_and_peaked_scores(ops, cuda, size):
    for new, lens in (([1], [3000]), ([100], [900])):
        q, starts = _q(sum(new), 4, 64, 2, size), _starts(new)
        cache = ref.paged(lens, 32, 1, 64, 3)
        want, tol = ref.attention(q, cache[0], cache[1], cache[4], lens, starts)
        ref.within(_run(ops, q, cache, lens, starts), want, tol)


def test_scales_of_very_different_size(ops, cuda):
    """8 bits: rows whose scales span the whole range of the quantization."""
    for new, lens in (([1], [500]), ([90], [200])):
        q, starts = _q(sum(new), 4, 64, 2, 0.5), _starts(new)
        k, v, ks, vs, tables = ref.paged(lens, 16, 2, 64, 3, True)
        g = torch.Generator().manual_seed(4)
        vs = vs * 10.0 ** (-6 * torch.rand(vs.shape, generator=g))
        want, tol = ref.attention(q, k, v, tables, lens, starts, ks, vs)
        ref.within(_run(ops, q, (k, v, ks, vs, tables), lens, starts), want, tol)


def test_scale_argument_and_views(ops, cuda):
    """A scale of one's own; queries as a view of the merged row; block tables as a view."""
    new, lens = [3, 40], [60, 90]
    starts = _starts(new)
    k, v, _, _, tables = ref.paged(lens, 16, 2, 64, 3)
    wide = _q(43, 8, 64, 4)
    q = wide[:, 2:6]
    want, tol = ref.attention(q, k, v, tables, lens, starts, scale=0.3)
    more = torch.full((2, 20), 99, dtype=torch.int32)
    more[:, 1:1 + tables.shape[1]] = tables
    got = ops.paged_attention(wide.cuda()[:, 2:6], k.cuda(), v.cuda(),
                              more.cuda()[:, 1:1 + tables.shape[1]], torch.tensor(lens).cuda(),
                              torch.tensor(starts).cuda(), scale=0.3)
    ref.within(got, want, tol)


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
@pytest.mark.parametrize("int8", [False, True])
def test_any_scale(ops, cuda, scale, int8):
    _check(ops, [1, 2], [300, 70], 4, 2, 128, 16, int8, scale=scale)
    _check(ops, [90, 40], [150, 40], 4, 2, 64, 16, int8, scale=scale)


@pytest.mark.parametrize("shift", [-300.0, 300.0])
def test_scores_far_from_zero(ops, cuda, shift):
    """Every key the same large part along the queries: exponents of hundreds, in one part
    and in several."""
    for new, lens in (([1, 1], [40, 5000]), ([150], [2000])):
        starts = _starts(new)
        q = _q(sum(new), 4, 64, 2)
        k, v, _, _, tables = ref.paged(lens, 16, 2, 64, 3)
        q[..., 0], k[..., 0] = 16.0, shift / 16.0
        want, tol = ref.attention(q, k, v, tables, lens, starts, scale=1.0)
        ref.within(_run(ops, q, (k, v, None, None, tables), lens, starts, scale=1.0), want, tol)


def test_many_sequences(ops, cuda):
    """More sequences than a workgroup has lanes, of every small length."""
    lens = [1 + i % 40 for i in range(700)]
    _check(ops, [1] * 700, lens, 2, 1, 64, 16)
    new = [i % 3 for i in range(600)]
    _check(ops, new, [n + i % 50 for i, n in enumerate(new)], 4, 2, 64, 16, most=None)


@pytest.mark.parametrize("B", [63, 64, 65, 300])
@pytest.mark.parametrize("window", [None, 50])
def test_chunks_and_single_tokens_of_many_sequences(ops, cuda, B, window):
    """Sequences as many as a wave's lanes, one fewer and more, of lengths that repeat."""
    new = [(1, 40, 0, 33, 2, 70)[i % 6] for i in range(B)]
    lens = [n + (0, 100, 7)[i % 3] for i, n in enumerate(new)]
    _check(ops, new, lens, 4, 1, 64, 16, int8=B == 65, seed=B, window=window)


def test_long_cache_offsets(ops, cuda):
    """Pages whose byte offsets pass 32 bits."""
    pages, page, D = 1 << 13, 4096, 128
    k = torch.zeros(pages, 1, page, D, dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    small = ref.paged([700], 4096, 1, D, 3, spare=0)
    for a, b in ((k, small[0]), (v, small[1])):
        a[pages - 1] = b[0].cuda()
    tables = torch.tensor([[pages - 1]], dtype=torch.int32)
    for new in (1, 80):
        q = _q(new, 4, D, 5)
        want, tol = ref.attention(q, small[0], small[1], small[4], [700], [0, new])
        ref.within(_run(ops, q, (k, v, None, None, tables), [700], [0, new]), want, tol)


def test_the_same_call_gives_the_same_bits(ops, cuda):
    for new, lens in (([1] * 6, [5000, 3, 900, 64, 700, 2]), ([300, 1, 5], [900, 400, 64])):
        q, starts = _q(sum(new), 8, 128, 2), _starts(new)
        cache = ref.paged(lens, 16, 2, 128, 3)
        first = _run(ops, q, cache, lens, starts)
        for _ in range(3):
            assert torch.equal(_run(ops, q, cache, lens, starts), first)


def test_refused(ops, cuda):
    q = torch.randn(4, 4, 64).half().cuda()
    k = torch.zeros(3, 2, 16, 64, dtype=torch.float16, device="cuda")
    t = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    n = torch.ones(4, dtype=torch.int32, device="cuda")
    cu = torch.arange(5, dtype=torch.int32, device="cuda")
    ok = ops.paged_attention(q, k, k, t, n, cu)
    assert ok.shape == q.shape
    assert ops.paged_attention(q[:0], k, k, t[:0], n[:0]).shape == (0, 4, 64)
    s = torch.zeros(3, 2, 16, device="cuda")
    bad = [
        lambda: ops.paged_attention(q.float(), k, k, t, n, cu),
        lambda: ops.paged_attention(q[0], k, k, t, n, cu),
        lambda: ops.paged_attention(q[:, :3], k, k, t, n, cu),
        lambda: ops.paged_attention(q[:, :0], k, k, t, n, cu),
        lambda: ops.paged_attention(q[..., :48], k, k, t, n, cu),
        lambda: ops.paged_attention(q, k, k[:2], t, n, cu),
        lambda: ops.paged_attention(q, k.transpose(1, 2), k, t, n, cu),
        lambda: ops.paged_attention(q, k, k, t[0], n, cu),
        lambda: ops.paged_attention(q, k, k, t.float(), n, cu),
        lambda: ops.paged_attention(q, k, k, t[:, :0], n, cu),
        lambda: ops.paged_attention(q, k, k, t, n[:3], cu),
        lambda: ops.paged_attention(q, k, k, t, n, cu[:4]),
        lambda: ops.paged_attention(q, k, k, t[:2], n[:2]),
        lambda: ops.paged_attention(q, k, k, t, n, cu, window=0),
        lambda: ops.paged_attention(q, k, k, t, n, cu, max_seqlen=-1),
        lambda: ops.paged_attention(q, k, k, t, n, cu, scale=float("inf")),
        lambda: ops.paged_attention(q, k, k, t, n, cu, k_scale=s),
        lambda: ops.paged_attention(q, k, k, t, n, cu, k_scale=s, v_scale=s),
        lambda: ops.paged_attention(q, k.cpu(), k, t, n, cu),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
