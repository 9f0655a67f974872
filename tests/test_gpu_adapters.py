"""Adapters on the linears of an MLP, an attention layer and a head, and the draw from its logits,
as a serving step runs them together."""
import pytest
import torch

import attention_ref as ref

pytestmark = pytest.mark.gpu

HIDDEN, INTER, HEADS, KV, DIM, VOCAB, RANK, SLOTS = 512, 1280, 8, 2, 64, 5003, 12, 6


def qtensor(pkg, wl, out, inner, seed):
    q, s = wl.weight_i8(out, inner, seed=seed)
    return pkg.QTensor(q.cuda(), (s * 0.1).cuda(), scheme="per_row_i8")


def fill(m, seed):
    """Adapters in every slot but the last, of different ranks, one with a part left out."""
    g = torch.Generator().manual_seed(seed)
    for slot in range(SLOTS - 1):
        r, parts = RANK - 2 * slot, []
        for i, wide in enumerate(m.splits):
            a = torch.randn(r, m.in_features, generator=g) * m.in_features ** -0.5
            b = torch.randn(wide, r, generator=g) * 0.2
            parts.append(None if slot == 1 and i == 0 else (a.half().cuda(), b.half().cuda()))
        m.load(slot, parts, scaling=0.5 + 0.3 * slot)


def wrap(pkg, linear, batch, seed, splits=None):
    m = pkg.LoRALinear(linear, batch, RANK, splits=splits)
    fill(m, seed)
    return m


def by_row(pkg, m, x, ids):
    """The module's rows one by one, from its base and its matrices in 32 bits."""
    y = m.base(x)
    want = y.clone()
    for t, e in enumerate(ids.tolist()):
        if 0 <= e < SLOTS:
            low, n = (m.a[e].float() @ x[t].float()) * m.scaling[e], 0
            for p, wide in enumerate(m.splits):
                up = m.b[e, n:n + wide].float() @ low[p * m.rank:(p + 1) * m.rank]
                want[t, n:n + wide] = (y[t, n:n + wide].float() + up).half()
                n += wide
    return want


def close(got, want):
    """Two sums in 32 bits in different orders, each rounded to fp16: a step of fp16 apart at most
    (twice half a step, 2^-10 of the value), and 2^-12 for sums of terms of a few units that
    cancel (1e3 products of 2^-24 each)."""
    return bool(((got.float() - want.float()).abs() <= 2.0 ** -10 * want.float().abs() + 2.0 ** -12).all())


def test_modules_match_their_parts(pkg, wl, cuda):
    batch = pkg.AdapterBatch(SLOTS)
    for rows in (1, 7, 70):
        ids = torch.arange(rows) % (SLOTS + 1) - 1
        batch.assign(ids.cuda())
        x = wl.activations(rows, HIDDEN, seed=rows).cuda()
        m = wrap(pkg, pkg.LinearW8A8(qtensor(pkg, wl, 768, HIDDEN, 1)), batch, 2, [512, 128, 128])
        got = m(x)
        assert close(got, by_row(pkg, m, x, ids))
        assert torch.equal(got[ids < 0], m.base(x)[ids < 0])
        host = pkg.LoRALinear(pkg.LinearW8A8(m.weight), pkg.AdapterBatch(SLOTS), RANK)
        assert host.a.is_cuda
        mlp = pkg.GatedMLP(qtensor(pkg, wl, 2 * INTER, HIDDEN, 3), qtensor(pkg, wl, HIDDEN, INTER, 4))
        mlp.gate_up_proj = wrap(pkg, mlp.gate_up_proj, batch, 5, [INTER, INTER])
        mlp.down_proj = wrap(pkg, mlp.down_proj, batch, 6)
        h = mlp.act_fn(mlp.gate_up_proj(x))
        assert torch.equal(mlp(x), mlp.down_proj(h))
        assert close(mlp.down_proj(h), by_row(pkg, mlp.down_proj, h, ids))
    with pytest.raises(ValueError, match="rows"):
        m(wl.activations(3, HIDDEN, seed=1).cuda())
    batch.clear()
    assert torch.equal(m(x), m.base(x))


class Layer:
    """Attention, MLP, head and sampler over one decoded token a sequence."""

    def __init__(self, pkg, wl, batch):
        rot = pkg.RotaryEmbedding(DIM, 256, device="cuda")
        self.attn = pkg.GQAAttention(qtensor(pkg, wl, (HEADS + 2 * KV) * DIM, HIDDEN, 1),
                                     qtensor(pkg, wl, HIDDEN, HEADS * DIM, 2), HEADS, KV, DIM, rot)
        self.attn.qkv_proj = wrap(pkg, self.attn.qkv_proj, batch, 3,
                                  [HEADS * DIM, KV * DIM, KV * DIM])
        self.attn.o_proj = wrap(pkg, self.attn.o_proj, batch, 4)
        self.mlp = pkg.GatedMLP(qtensor(pkg, wl, 2 * INTER, HIDDEN, 5),
                                qtensor(pkg, wl, HIDDEN, INTER, 6))
        self.mlp.gate_up_proj = wrap(pkg, self.mlp.gate_up_proj, batch, 7, [INTER, INTER])
        self.mlp.down_proj = wrap(pkg, self.mlp.down_proj, batch, 8)
        self.head = pkg.LMHead(qtensor(pkg, wl, VOCAB, HIDDEN, 9))
        self.head.proj = wrap(pkg, self.head.proj, batch, 10)
        self.sampler = pkg.Sampler(return_logprobs=True)

    def __call__(self, x, cache, step, settings, u):
        h = x + self.attn(x, cache, step)
        h = h + self.mlp(h)
        return self.sampler(self.head(h), *settings, u=u)


@pytest.mark.parametrize("seqs", [1, 5, 24])
def test_a_decode_step_in_a_graph(pkg, wl, cuda, seqs):
    """Replays with new tokens, adapters, settings and random numbers, each against the eager
    step."""
    batch = pkg.AdapterBatch(SLOTS)
    layer = Layer(pkg, wl, batch)
    cache = pkg.PagedKVCache(2 * seqs, 16, KV, DIM)
    tables = torch.arange(2 * seqs, dtype=torch.int32).view(seqs, 2)
    steps = [cache.step(tables, new=[1] * seqs, total=[n] * seqs) for n in range(1, 8)]
    step = cache.step(tables, new=[1] * seqs, total=[1] * seqs)
    g = torch.Generator().manual_seed(seqs)
    x = wl.activations(seqs, HIDDEN, seed=3).cuda()
    u = torch.rand(seqs, device="cuda")
    kinds = (torch.float32, torch.int32, torch.float32, torch.float32)
    settings = [torch.zeros(seqs, dtype=t, device="cuda") for t in kinds]
    batch.assign(torch.zeros(seqs, dtype=torch.int32, device="cuda"))

    def renew(n):
        x.copy_(wl.activations(seqs, HIDDEN, seed=50 + n))
        u.copy_(torch.rand(seqs, generator=g))
        batch.assign(torch.randint(-1, SLOTS, (seqs,), generator=g).cuda())
        for t, v in zip(settings, ((0.0, 0.7, 1.0, 1.4), (0, 5, 40, 0), (1.0, 0.9, 0.5, 1.0),
                                   (0.0, 0.0, 0.1, 0.02))):
            pick = torch.randint(0, 4, (seqs,), generator=g)
            t.copy_(torch.tensor(v)[pick].to(t.dtype))
        for f in ("positions", "slots", "block_tables", "context_lens", "cu_seqlens"):
            old, new = getattr(step, f), getattr(steps[n], f)
            if old is not None:
                old.copy_(new)

    renew(0)
    layer(x, cache, step, settings, u)                   # first calls outside the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        token, logp = layer(x, cache, step, settings, u)
    for n in range(6):
        renew(n)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = (token.clone(), logp.clone())
        want = layer(x, cache, step, settings, u)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), n
        assert ((got[0] >= 0) & (got[0] < VOCAB)).all()


def test_adapters_change_what_is_drawn(pkg, wl, cuda):
    batch = pkg.AdapterBatch(SLOTS)
    head = pkg.LMHead(qtensor(pkg, wl, VOCAB, HIDDEN, 9), logit_softcap=30.0)
    head.proj = wrap(pkg, head.proj, batch, 10)
    x = wl.activations(32, HIDDEN, seed=1).cuda()
    greedy = pkg.Sampler()
    plain = greedy(head(x), temperature=0.0)             # soft-capped logits are fp32
    assert torch.equal(plain, head(x).argmax(-1))
    batch.assign(torch.tensor([-1, 0] * 16, device="cuda"))
    drawn = greedy(head(x), temperature=0.0)
    assert torch.equal(drawn[::2], plain[::2]) and not torch.equal(drawn[1::2], plain[1::2])
    torch.manual_seed(0)
    one = greedy(head(x), top_k=50)
    torch.manual_seed(0)
    assert torch.equal(one, greedy(head(x), top_k=50))


def test_graphs_of_several_batch_sizes_share_a_batch(pkg, wl, cuda):
    """One captured graph for each number of rows, as a server keeps them: each follows what is
    assigned before its replay, whatever was assigned, and freed, in between."""
    batch = pkg.AdapterBatch(SLOTS)
    m = wrap(pkg, pkg.LinearW8A8(qtensor(pkg, wl, 640, HIDDEN, 81)), batch, 82, splits=[512, 128])
    g = torch.Generator().manual_seed(83)
    ids_of = lambda n: torch.randint(-1, SLOTS, (n,), generator=g)  # noqa: E731
    graphs = {}
    for n in (4, 7, 16, 200):
        x = wl.activations(n, HIDDEN, seed=n).cuda()
        batch.assign(ids_of(n).cuda())
        m(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = m(x)
        graphs[n] = graph, x, y
    for n in (16, 4, 200, 7, 4, 16, 7, 200):
        ids, (graph, x, y) = ids_of(n), graphs[n]
        batch.assign(ids_of(33).cuda())                    # an eager step of another size
        other = [torch.full((64,), 1 << 20, dtype=torch.int32, device="cuda") for _ in range(8)]
        batch.assign(ids.cuda())
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, m(x)) and close(y, by_row(pkg, m, x, ids)), n
        del other


def test_ids_on_the_host_beside_rows_on_the_gpu_are_refused(pkg, wl, cuda):
    batch = pkg.AdapterBatch(SLOTS)
    m = wrap(pkg, pkg.LinearW8A8(qtensor(pkg, wl, 640, HIDDEN, 84)), batch, 85)
    batch.assign(torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ValueError):
        m(wl.activations(4, HIDDEN, seed=86).cuda())


def test_graphs_of_neighbouring_sizes_keep_their_plans(pkg, wl, cuda):
    """Every size assigned first, then all replayed: each graph has the plan of its own rows."""
    batch = pkg.AdapterBatch(SLOTS)
    m = wrap(pkg, pkg.LinearW8A8(qtensor(pkg, wl, 640, HIDDEN, 91)), batch, 92, splits=[512, 128])
    g = torch.Generator().manual_seed(93)
    graphs = {}
    for n in (4, 5, 6, 7):
        x = wl.activations(n, HIDDEN, seed=n).cuda()
        batch.assign(torch.zeros(n, dtype=torch.int32, device="cuda"))
        m(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = m(x)
        graphs[n] = graph, x, y
    for order in ((4, 5, 6, 7), (7, 6, 5, 4), (5, 7, 4, 6)):
        ids = {n: torch.randint(-1, SLOTS, (n,), generator=g) for n in graphs}
        for n in order:
            batch.assign(ids[n].cuda())
        for graph, _, _ in graphs.values():
            graph.replay()
        torch.cuda.synchronize()
        for n, (_, x, y) in graphs.items():
            assert close(y, by_row(pkg, m, x, ids[n])), (order, n)


def test_clear_reaches_captured_steps(pkg, wl, cuda):
    batch = pkg.AdapterBatch(SLOTS)
    m = wrap(pkg, pkg.LinearW8A8(qtensor(pkg, wl, 640, HIDDEN, 94)), batch, 95)
    graphs = []
    for n in (6, 70):
        x = wl.activations(n, HIDDEN, seed=n).cuda()
        batch.assign((torch.arange(n) % SLOTS).cuda())
        m(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = m(x)
        graphs.append((graph, x, y))
    for rep in range(3):
        batch.clear()
        for graph, x, y in graphs:
            graph.replay()
            assert torch.equal(y, m.base(x)), rep
        for graph, x, y in graphs:                        # and back
            ids = (torch.arange(len(x)) + rep) % SLOTS
            batch.assign(ids.cuda())
            graph.replay()
            assert close(y, by_row(pkg, m, x, ids)), rep


class Keeps:
    """A linear's forward of its own that hands out the same tensor again."""

    def __init__(self, base):
        self.inner, self.kept = base.forward, None

    def __call__(self, x):
        if self.kept is None:
            self.kept = self.inner(x)
        return self.kept


def test_what_the_base_returned_stays(pkg, wl, cuda):
    batch = pkg.AdapterBatch(SLOTS)
    m = wrap(pkg, pkg.LinearW8A8(qtensor(pkg, wl, 640, HIDDEN, 96)), batch, 97)
    x, ids = wl.activations(9, HIDDEN, seed=98).cuda(), torch.arange(9) % SLOTS - 1
    batch.assign(ids.cuda())
    plain, want, seen = m.base(x).clone(), m(x), []
    keep = lambda mod, args, y: seen.append(y)  # noqa: E731
    for register in (m.base.register_forward_hook, torch.nn.modules.module.register_module_forward_hook):
        seen.clear()
        handle = register(keep)
        y = m(x)
        handle.remove()
        assert torch.equal(seen[0], plain) and torch.equal(y, want)
    m.base.forward = Keeps(m.base)
    for _ in range(3):
        assert torch.equal(m(x), want)
    assert torch.equal(m.base.forward.kept, plain)


def test_nothing_is_added_where_a_slot_has_nothing(pkg, wl, cuda):
    """Rows with infinities keep what the base makes of them in empty and unloaded slots and in
    parts without an adapter."""
    g = torch.Generator().manual_seed(99)
    codes = torch.randint(0, 7, (768, HIDDEN), generator=g, dtype=torch.uint8)   # all below 0
    data = codes[:, ::2] | codes[:, 1::2] << 4
    base = pkg.LinearW8A8(pkg.QTensor(data.cuda(), torch.full((768, HIDDEN // 64), 0.02, device="cuda"),
                                      scheme="per_group_i4", group_size=64, codebook="nf4"))
    batch = pkg.AdapterBatch(SLOTS)
    m = wrap(pkg, base, batch, 100, splits=[512, 256])   # slot 1 has no first part
    m.unload(3)
    for rows in (6, 1200):
        x = wl.activations(rows, HIDDEN, seed=rows).cuda()
        ids = torch.arange(rows) % (SLOTS + 1) - 1
        batch.assign(ids.cuda())
        clean = m(x)
        assert close(clean, by_row(pkg, m, x, ids))
        x[:, 7] = torch.inf
        plain, y = base(x), m(x)
        assert plain.isinf().all()
        bare = (ids < 0) | (ids == 3) | (ids == SLOTS - 1)
        assert torch.equal(y[bare], plain[bare])
        assert torch.equal(y[ids == 1, :512], plain[ids == 1, :512])
        assert not y.isfinite().any()


def test_the_mlp_fuses_again_without_adapters(pkg, wl, cuda, monkeypatch):
    batch = pkg.AdapterBatch(SLOTS)
    up, down = qtensor(pkg, wl, 2 * INTER, HIDDEN, 3), qtensor(pkg, wl, HIDDEN, INTER, 4)
    plain, mlp = pkg.GatedMLP(up, down), pkg.GatedMLP(up, down)
    mlp.gate_up_proj = wrap(pkg, mlp.gate_up_proj, batch, 5, [INTER, INTER])
    mlp.down_proj = wrap(pkg, mlp.down_proj, batch, 6)
    calls, fused = [], pkg.ops.act_and_mul_quant
    monkeypatch.setattr(pkg.ops, "act_and_mul_quant", lambda *a: calls.append(1) or fused(*a))
    for rows in (1, 4, 5, 70):
        x = wl.activations(rows, HIDDEN, seed=rows).cuda()
        calls.clear()
        assert torch.equal(mlp(x), plain(x)) and len(calls) == (rows >= 5)
        batch.assign(torch.zeros(rows, dtype=torch.int32, device="cuda"))
        calls.clear()
        assert not torch.equal(mlp(x), plain(x)) and not calls
        batch.clear()
        assert torch.equal(mlp(x), plain(x))
        seen = []
        handle = mlp.down_proj.register_forward_hook(lambda *a: seen.append(1))
        assert torch.equal(mlp(x), plain(x)) and seen
        handle.remove()


def test_attention_reaches_its_output_through_adapters(pkg, wl, cuda):
    """Every stage of an attention layer with both projections adapted, over prompts and decoded
    tokens, against its plain form from the tensors that went into it."""
    batch = pkg.AdapterBatch(SLOTS)
    attn = Layer(pkg, wl, batch).attn
    cache = pkg.PagedKVCache(6, 16, KV, DIM)
    tables = torch.arange(6, dtype=torch.int32).view(2, 3).cuda()
    total, tab = [0, 0], attn.rotary.cos_sin.cpu()
    for new in ([30, 7], [1, 1], [4, 1]):
        total = [a + b for a, b in zip(total, new)]
        T = sum(new)
        x, ids = wl.activations(T, HIDDEN, seed=T).cuda(), torch.arange(T) % (SLOTS + 1) - 1
        batch.assign(ids.cuda())
        step = cache.step(tables, new, total)
        out = attn(x, cache, step)
        qkv = attn.qkv_proj(x)
        assert close(qkv, by_row(pkg, attn.qkv_proj, x, ids))
        has = (ids >= 0) & (ids < SLOTS - 1)
        for part, base in zip(qkv[has].split(attn.qkv_proj.splits, -1),
                              attn.qkv_proj.base(x)[has].split(attn.qkv_proj.splits, -1)):
            assert not torch.equal(part, base)
        q, k, v = (t.unflatten(-1, (-1, DIM)) for t in qkv.split(attn.qkv_proj.splits, -1))
        k_got, v_got = cache.read(step.slots)
        ref.within(k_got, *ref.norm_rope(k.cpu(), None, step.positions.cpu(), tab))
        assert torch.equal(v_got, v.float())
        q_got = pkg.rope(q, k, step.positions, attn.rotary.cos_sin)[0]
        ref.within(q_got, *ref.norm_rope(q.cpu(), None, step.positions.cpu(), tab))
        got = cache.attend(q_got, step)
        ref.within(got, *ref.attention(q_got.cpu(), cache.k.cpu(), cache.v.cpu(), tables.cpu(), total,
                                       [0, new[0], T], None, None))
        low = got.flatten(1)
        assert torch.equal(out, attn.o_proj(low)) and close(out, by_row(pkg, attn.o_proj, low, ids))
        assert not torch.equal(out, attn.o_proj.base(low))
