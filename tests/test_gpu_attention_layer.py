"""A layer's attention as it is served, on the GPU: QKV linear, norms and rotation with the
append, attention over the cache and the O linear in a run; in graphs, on other streams and
through the native host path."""
import ctypes

import pytest
import torch

import attention_ref as ref
from test_gpu_host_path import general, taken  # noqa: F401

pytestmark = pytest.mark.gpu


def _weight(pkg, out, in_, g):
    return pkg.QTensor(torch.randint(-127, 128, (out, in_), generator=g, dtype=torch.int8).cuda(),
                       (torch.rand(out, generator=g) * 2e-4 + 1e-4).cuda(), scheme="per_row_i8")


def _layer(pkg, Hq=8, Hk=2, D=64, hidden=256, pairs=False, norm=True, window=None, P=4096):
    g = torch.Generator().manual_seed(Hq + D)
    norms = [None, None]
    if norm:
        norms = [pkg.RMSNorm(D).cuda().half() for _ in range(2)]
        for n in norms:
            n.weight.data.copy_(torch.rand(D, generator=g) + 0.5)
    rot = pkg.RotaryEmbedding(D, P, rotary_dim=D // 2, interleaved=pairs, device="cuda",
                              scaling={"type": "linear", "factor": 2})
    return pkg.GQAAttention(_weight(pkg, (Hq + 2 * Hk) * D, hidden, g),
                            _weight(pkg, hidden, Hq * D, g), Hq, Hk, D, rot, q_norm=norms[0],
                            k_norm=norms[1], window=window)


def _cache(pkg, layer, lens, page, dtype, seed=0):
    """A cache with room for `lens`, its pages in any order."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    cache = pkg.PagedKVCache(sum(need) + 1, page, layer.num_kv_heads, layer.head_dim, dtype)
    order = torch.randperm(sum(need) + 1, generator=g).int()
    tables = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    for i, n in enumerate(need):
        tables[i, :n], order = order[:n], order[n:]
    return cache, tables.cuda()


def _cpu(t):
    return None if t is None else t.cpu()


@pytest.mark.parametrize("dtype", [torch.float16, torch.int8])
@pytest.mark.parametrize("pairs,norm,window", [(False, True, None), (True, False, 40)])
def test_layer_over_prompts_and_decoding(pkg, cuda, dtype, pairs, norm, window):
    """Prompts in chunks, then decoded and drafted tokens, mixed: every stage of every step
    against its 64-bit form, from the tensors that went into it."""
    layer = _layer(pkg, pairs=pairs, norm=norm, window=window)
    Hq, Hk, D = layer.num_heads, layer.num_kv_heads, layer.head_dim
    cache, tables = _cache(pkg, layer, [200, 150, 40], 16, dtype)
    g = torch.Generator().manual_seed(5)
    total = [0, 0, 0]
    for new in ([130, 0, 7], [60, 64, 1], [1, 80, 1], [1, 1, 1], [4, 4, 4], [1, 0, 1]):
        total = [a + b for a, b in zip(total, new)]
        x = torch.randn(sum(new), 256, generator=g).half().cuda()
        step = cache.step(tables, new, total)
        out = layer(x, cache, step)

        q, k, v = layer.qkv_proj(x).cpu().split([Hq * D, Hk * D, Hk * D], -1)
        q, k, v = (t.unflatten(-1, (-1, D)) for t in (q, k, v))
        tab, pos = layer.rotary.cos_sin.cpu(), step.positions.cpu()
        w = [None if n is None else n.weight.detach().cpu() for n in (layer.q_norm, layer.k_norm)]
        q_want, q_tol = ref.norm_rope(q, w[0], pos, tab, pairs)
        k_want, k_tol = ref.norm_rope(k, w[1], pos, tab, pairs)
        k_got, v_got = cache.read(step.slots)
        if dtype == torch.int8:
            # half a code of a scale that is off by the row's bound, and its own roundings
            for got, want, tol in ((k_got, k_want, k_tol), (v_got, v.double(), torch.zeros(1))):
                code = (want.abs() + tol).amax(-1, keepdim=True) / 127
                ref.within(got, want, tol + code * (0.5 + 2.0 ** -10))
        else:
            ref.within(k_got, k_want, k_tol)
            assert torch.equal(v_got.cpu(), v.float())
        starts = step.cu_seqlens.tolist()
        q_got = pkg.qk_norm_rope(*(t.cuda() for t in (q, k)), *(
            None if t is None else t.cuda() for t in w), step.positions, layer.rotary.cos_sin,
            interleaved=pairs)[0]
        ref.within(q_got, q_want, q_tol)
        got = cache.attend(q_got, step, window=window)
        want, tol = ref.attention(q_got.cpu(), cache.k.cpu(), cache.v.cpu(), tables.cpu(), total,
                                  starts, _cpu(cache.k_scale), _cpu(cache.v_scale), window=window)
        ref.within(got, want, tol)
        assert torch.equal(out, layer.o_proj(got.flatten(1)))


@pytest.mark.parametrize("dtype", [torch.float16, torch.int8])
def test_a_prompt_in_chunks_fills_the_same_cache(pkg, cuda, dtype):
    layer = _layer(pkg)
    x = torch.randn(300, 256, generator=torch.Generator().manual_seed(1)).half().cuda()
    whole, tables = _cache(pkg, layer, [300], 32, dtype)
    parts, _ = _cache(pkg, layer, [300], 32, dtype)
    layer(x, whole, whole.step(tables, [300], [300]))
    at = 0
    for n in (1, 130, 64, 5, 100):
        at += n
        layer(x[at - n:at], parts, parts.step(tables, [n], [at]))
    for a, b in ((whole.k, parts.k), (whole.v, parts.v), (whole.k_scale, parts.k_scale)):
        assert a is None or torch.equal(a, b)


def _steps(cache, tables, lens, new):
    """Steps one after the other, `new` tokens a sequence each."""
    while True:
        lens = [n + new for n in lens]
        yield cache.step(tables, [new] * len(lens), lens)


@pytest.mark.parametrize("new,lens,room", [(1, [300, 17, 4000, 90], 4096), (4, [5, 700], 800),
                                           (70, [0, 300, 33], 768)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.int8])
def test_steps_captured_and_replayed(pkg, cuda, dtype, new, lens, room):
    """The layer's step in a graph, its tensors filled anew for each replay, with eager work
    and allocations between: every replay against the eager step on a cache of its own."""
    layer = _layer(pkg)
    n = len(lens)
    eager, tables = _cache(pkg, layer, [room] * n, 64, dtype)
    g = torch.Generator().manual_seed(3)
    for c in (eager.k, eager.v):
        c.copy_(torch.randint(-100, 100, c.shape, generator=g).to(dtype))
    if dtype == torch.int8:
        for s in (eager.k_scale, eager.v_scale):
            s.copy_(torch.rand(s.shape, generator=g) * 0.01)
    else:
        eager.k.mul_(0.01), eager.v.mul_(0.01)
    played, _ = _cache(pkg, layer, [room] * n, 64, dtype)
    for a, b in zip((played.k, played.v, played.k_scale, played.v_scale),
                    (eager.k, eager.v, eager.k_scale, eager.v_scale)):
        if a is not None:
            a.copy_(b)
    steps = _steps(eager, tables, lens, new)
    first = next(steps)
    static = pkg.Step(*(getattr(first, f).clone() for f in
                        ("positions", "slots", "block_tables", "context_lens", "cu_seqlens")), new)
    x = torch.randn(n * new, 256, generator=g).half().cuda()
    layer(x, eager, first)
    layer(x, played, static)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(x, played, static)
    for i in range(5):
        step = next(steps)
        x.copy_(torch.randn(x.shape, generator=g).half())
        for f in ("positions", "slots", "context_lens"):
            getattr(static, f).copy_(getattr(step, f))
        graph.replay()
        want = layer(x, eager, step)
        junk = torch.full((1 << 20,), float("nan"), device="cuda")
        torch.cuda.synchronize()
        del junk
        assert torch.equal(out, want), i
        assert torch.equal(played.k, eager.k) and torch.equal(played.v, eager.v)


def test_two_graphs_and_two_streams_at_once(pkg, cuda):
    """Two captured calls, replayed on two streams at once, and two eager calls on two streams:
    no workspace is shared."""
    made = []
    for seed, (new, lens) in enumerate((([1] * 6, [9000, 1, 300, 5000, 64, 700]),
                                        ([100, 200], [4000, 2500]))):
        q = torch.randn(sum(new), 8, 128, generator=torch.Generator().manual_seed(seed)).half()
        k, v, _, _, tables = ref.paged(lens, 64, 2, 128, seed)
        starts = torch.tensor([0] + new).cumsum(0).int()
        args = [t.cuda() for t in (q, k, v, tables, torch.tensor(lens, dtype=torch.int32), starts)]
        made.append((args, max(new)))
    want = [pkg.paged_attention(*a, max_seqlen=m) for a, m in made]
    streams = [torch.cuda.Stream() for _ in made]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for a, m in made:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(pkg.paged_attention(*a, max_seqlen=m))
    for _ in range(4):
        for out in outs:
            out.fill_(7.0)
        torch.cuda.synchronize()
        eager = [[], []]
        for _ in range(3):
            for s, g in zip(streams, graphs):
                with torch.cuda.stream(s):
                    g.replay()
            for s, (a, m), got in zip(streams, made, eager):
                with torch.cuda.stream(s):
                    got.append(pkg.paged_attention(*a, max_seqlen=m))
        torch.cuda.synchronize()
        for out, got, w in zip(outs, eager, want):
            assert torch.equal(out, w) and all(torch.equal(t, w) for t in got)


def test_block_tables_on_the_host(pkg, cuda):
    layer = _layer(pkg)
    cache, tables = _cache(pkg, layer, [40, 20], 16, torch.float16)
    a, b = cache.step(tables, [3, 1], [33, 20]), cache.step(tables.cpu(), [3, 1], [33, 20])
    assert all(torch.equal(getattr(a, f), getattr(b, f)) for f in
               ("positions", "slots", "block_tables", "context_lens", "cu_seqlens"))


def test_the_current_stream_orders_the_calls(pkg, cuda):
    """Inputs made on a side stream behind slow work: the calls run on that stream."""
    layer = _layer(pkg)
    x0 = torch.randn(3, 256, generator=torch.Generator().manual_seed(2)).half().cuda()
    a, tables = _cache(pkg, layer, [64] * 3, 16, torch.float16)
    b, _ = _cache(pkg, layer, [64] * 3, 16, torch.float16)
    want = layer(x0, a, a.step(tables, [1] * 3, [1] * 3))
    slow = torch.randn(4096, 4096, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(10):
            slow = slow @ slow * 1e-3
        x = x0 + (slow[0, 0] * 0).nan_to_num().half()
        got = layer(x, b, b.step(tables, [1] * 3, [1] * 3))
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(a.k, b.k)


# ---- the native host path -------------------------------------------------------------

def _args(pkg, int8):
    T, Hq, Hk, D, page = 6, 4, 2, 64, 16
    g = torch.Generator().manual_seed(9)
    qkv = torch.randn(T, (Hq + 2 * Hk) * D, generator=g).half().cuda()
    q, k, v = (t.unflatten(-1, (-1, D)) for t in qkv.split([Hq * D, Hk * D, Hk * D], -1))
    kc, vc, ks, vs, tables = (None if t is None else t.cuda() for t in
                              ref.paged([70, 5, 33, 16, 64, 1], page, Hk, D, 1, int8))
    pos = torch.tensor([69, 4, 32, 15, 63, 0], dtype=torch.int32).cuda()
    slots = (tables[torch.arange(T), (pos // page).long()] * page + pos % page).int()
    return (q, k, v, pos, ref.table(100, D).cuda(), kc, vc, ks, vs, slots, tables, pos + 1,
            torch.rand(D, generator=g).half().cuda())


@pytest.mark.parametrize("int8", [False, True])
def test_native_path_gives_the_general_results(pkg, cuda, general, taken, int8):  # noqa: F811
    q, k, v, pos, tab, kc, vc, ks, vs, slots, tables, lens, w = _args(pkg, int8)
    cu = torch.arange(7, dtype=torch.int32).cuda()
    for kw in (dict(), dict(interleaved=True), dict(unit_offset=True, eps=1e-5)):
        call = lambda: pkg.qk_norm_rope(q, k, w, None, pos, tab, **kw)  # noqa: E731, B023
        assert taken(call) == [("norm_rope", True)]
        a = call()
        with general():
            b = call()
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert taken(lambda: pkg.rope(q, k, pos, tab)) == [("norm_rope", True)]
    caches = [[None if t is None else t.clone() for t in (kc, vc, ks, vs)] for _ in range(2)]

    def append(c):
        return pkg.rope_append(q, k, v, pos, tab, c[0], c[1], slots, c[2], c[3], w, w)
    a = append(caches[0])
    with general():
        b = append(caches[1])
    assert torch.equal(a, b)
    assert all(x is None or torch.equal(x, y) for x, y in zip(*caches))
    assert taken(lambda: append(caches[0])) == [("rope_append", True)]
    for args, kw in (((tables, lens), dict(max_seqlen=1)), ((tables, lens, cu), dict(max_seqlen=1)),
                     ((tables, lens, cu), dict()), ((tables, lens, cu), dict(window=20, scale=0.3))):
        call = lambda: pkg.paged_attention(q, kc, vc, *args, k_scale=ks, v_scale=vs, **kw)  # noqa: E731, B023
        assert taken(call) == [("paged_attention", True)]
        a = call()
        with general():
            b = call()
        assert torch.equal(a, b)


def test_forms_left_to_the_general_way(pkg, cuda, taken):  # noqa: F811
    """64-bit indices, tensors that have to be copied, and refused arguments."""
    q, k, v, pos, tab, kc, vc, ks, vs, slots, tables, lens, w = _args(pkg, False)
    want = pkg.qk_norm_rope(q, k, w, w, pos, tab)
    for form in (dict(pos=pos.long()), dict(q=q.transpose(0, 1).contiguous().transpose(0, 1)
                                            .repeat_interleave(2, 2)[..., ::2]),
                 dict(w=torch.stack([w, w], 1)[:, 0])):
        f = dict(q=q, pos=pos, w=w)
        f.update(form)
        call = lambda: pkg.qk_norm_rope(f["q"], k, f["w"], w, f["pos"], tab)  # noqa: E731, B023
        assert taken(call) == [("norm_rope", False)]
        assert all(torch.equal(a, b) for a, b in zip(call(), want))
    want = pkg.paged_attention(q, kc, vc, tables, lens)
    for args in ((tables.long(), lens), (tables, lens.long()), (tables.t().contiguous().t(), lens)):
        call = lambda: pkg.paged_attention(q, kc, vc, *args)  # noqa: E731, B023
        assert taken(call) == [("paged_attention", False)]
        assert torch.equal(call(), want)
    a, b = kc.clone(), vc.clone()
    assert taken(lambda: pkg.rope_append(q, k, v, pos, tab, a, b, slots.long())) \
        == [("rope_append", False)]
    pkg.rope_append(q, k, v, pos, tab, kc, vc, slots)
    assert torch.equal(a, kc) and torch.equal(b, vc)


def test_indices_beyond_32_bits_lie_outside(pkg, cuda):
    """64-bit positions, slots and pages that would wrap to valid ones do not."""
    q, k, v, pos, tab, kc, vc, ks, vs, slots, tables, lens, w = _args(pkg, False)
    a, b = kc.clone(), vc.clone()
    far = slots.long() + (1 << 32)
    pkg.rope_append(q, k, v, pos, tab, a, b, far)
    pkg.rope_append(q, k, v, pos, tab, a, b, far - (1 << 33))
    assert torch.equal(a, kc) and torch.equal(b, vc)
    assert pkg.rope(q, k, pos.long() + (1 << 32), tab)[0].isnan().all()
    assert pkg.paged_attention(q, kc, vc, tables.long() + (1 << 32), lens).isnan().all()


def test_alignment_of_scales(pkg, cuda):
    """Scales that are a view off a 16-byte boundary are refused, on either path."""
    q, k, v, pos, tab, kc, vc, ks, vs, slots, tables, lens, w = _args(pkg, True)
    off = torch.empty(ks.numel() + 1, device="cuda")[1:].view(ks.shape)
    with pytest.raises(ValueError, match="align"):
        pkg.paged_attention(q, kc, vc, tables, lens, k_scale=off, v_scale=vs)


def test_too_many_workgroups_are_refused(pkg, cuda):
    """Items of both kinds whose sum has no grid, though each kind alone has one."""
    from importlib import import_module
    lib = import_module("fni8serve_amd._lib").load()
    f, B, T, Hk = ctypes.c_void_p(0x1000), 65536, 65536, 130  # nothing is read
    rc = lib.fni8_paged_attention_f16(f, Hk * 16, 16, T, Hk, Hk, 16, f, f, None, None, 8, 16, f, 1,
                                      1, f, f, B, 40, ctypes.c_float(1.0), 0, f, None, 0, None)
    assert rc == -2 and b"too many" in lib.fni8_last_error()


@pytest.mark.parametrize("new,lens", [([1] * 4, [900, 3, 0, 5000]), ([3, 5], [700, 5]),
                                      ([90, 1], [700, 300])])
def test_c_entry_without_a_workspace(pkg, cuda, new, lens):
    """The C entry splits no sequence without a workspace, and gives what the formula gives."""
    from importlib import import_module
    lib = import_module("fni8serve_amd._lib").load()
    T, Hq, Hk, D, page = sum(new), 8, 2, 64, 16
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = torch.randn(T, Hq, D, generator=torch.Generator().manual_seed(T)).half()
    k, v, _, _, tables = ref.paged(lens, page, Hk, D, T)
    d = [t.cuda() for t in (q, k, v, tables, torch.tensor(lens, dtype=torch.int32),
                            torch.tensor(starts, dtype=torch.int32))]
    out = torch.empty_like(d[0])
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    rc = lib.fni8_paged_attention_f16(
        p(d[0]), Hq * D, D, T, Hq, Hk, D, p(d[1]), p(d[2]), None, None, k.shape[0], page, p(d[3]),
        tables.shape[1], tables.shape[1], p(d[4]), p(d[5]), len(lens), max(new),
        ctypes.c_float(D ** -0.5), 0, p(out), None, 0,
        ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == 0
    want, tol = ref.attention(q, k, v, tables, lens, starts)
    ref.within(out, want, tol)
