"""AdapterBatch and LoRALinear on the CPU, and what they and Sampler refuse."""
from types import SimpleNamespace

import pytest
import torch


def linear(pkg, out, inner, seed):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-127, 128, (out, inner), generator=g, dtype=torch.int8)
    return pkg.LinearW8A8(pkg.QTensor(q, torch.rand(out, generator=g) * 0.01, scheme="per_row_i8"))


def pair(rank, inner, wide, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rank, inner, generator=g).half(),
            (torch.randn(wide, rank, generator=g) * 0.1).half())


def test_rows_get_their_own_adapter(pkg):
    base, batch = linear(pkg, 40, 32, 1), pkg.AdapterBatch(4)
    m = pkg.LoRALinear(base, batch, rank=6, splits=[24, 16])
    assert (m.rank, m.in_features, m.out_features) == (8, 32, 40)
    assert m.weight is base.weight and m.bias is base.bias
    p0, p1 = pair(6, 32, 24, 2), pair(3, 32, 16, 3)
    m.load(2, [p0, p1], scaling=0.5)
    m.load(0, [None, pair(5, 32, 16, 4)], scaling=2.0)
    x = torch.randn(5, 32).half()
    plain = base(x)
    assert torch.equal(m(x), plain)                      # no ids yet
    batch.assign(torch.tensor([2, -1, 0, 4, 1]))
    y = m(x)
    assert torch.equal(y[[1, 3, 4]], plain[[1, 3, 4]])   # none, outside, an empty slot
    want = plain[0].float() + 0.5 * torch.cat([(p0[1].float() @ (p0[0].float() @ x[0].float())),
                                               (p1[1].float() @ (p1[0].float() @ x[0].float()))])
    # sums of 32 products of a few units in 32 bits, then half a step of fp16
    assert torch.allclose(y[0].float(), want, rtol=2.0 ** -11, atol=1e-4)
    assert torch.equal(y[2, :24], plain[2, :24]) and not torch.equal(y[2, 24:], plain[2, 24:])
    assert torch.equal(m(x.view(5, 1, 32)).view(5, 40), y)
    m.unload(2)
    assert torch.equal(m(x)[0], plain[0])
    batch.clear()
    assert torch.equal(m(x), plain)


def test_refusals(pkg):
    base, batch = linear(pkg, 40, 32, 1), pkg.AdapterBatch(4)
    for n in (0, -1, 65535):
        with pytest.raises(ValueError, match="num_adapters"):
            pkg.AdapterBatch(n)
    for kw in (dict(rank=0), dict(rank=257), dict(rank=8, splits=[20, 16]),
               dict(rank=8, splits=[40, 0])):
        with pytest.raises(ValueError):
            pkg.LoRALinear(base, batch, **kw)
    m = pkg.LoRALinear(base, batch, rank=8, splits=[24, 16])
    good = [pair(8, 32, 24, 1), pair(8, 32, 16, 2)]
    for slot, parts in ((4, good), (-1, good), (0, good[:1]), (0, [good[1], good[0]]),
                        (0, [pair(9, 32, 24, 1), None]), (0, [pair(8, 31, 24, 1), None]),
                        (0, [(good[0][0], good[0][1][:, :7]), None])):
        with pytest.raises(ValueError):
            m.load(slot, parts)
    for ids in (torch.zeros(2, 2, dtype=torch.int32), torch.zeros(3)):
        with pytest.raises(ValueError, match="ids"):
            batch.assign(ids)
    batch.assign(torch.tensor([0, 1]))
    with pytest.raises(ValueError, match="rows"):
        m(torch.zeros(3, 32).half())
    with pytest.raises(ValueError, match="GPU"):
        pkg.Sampler()(torch.zeros(3, 32).half())


def test_the_mlp_calls_an_adapted_linear(pkg):
    """GatedMLP on the CPU with both projections wrapped: the sum of its parts."""
    up, down = linear(pkg, 48, 32, 1).weight, linear(pkg, 32, 24, 2).weight
    mlp, batch = pkg.GatedMLP(up, down), pkg.AdapterBatch(2)
    x = torch.randn(3, 32).half()
    plain = mlp(x)
    mlp.gate_up_proj = pkg.LoRALinear(mlp.gate_up_proj, batch, 8, splits=[24, 24])
    mlp.down_proj = pkg.LoRALinear(mlp.down_proj, batch, 8)
    assert torch.equal(mlp(x), plain)
    mlp.gate_up_proj.load(1, [pair(8, 32, 24, 3), pair(4, 32, 24, 4)])
    mlp.down_proj.load(1, [pair(8, 24, 32, 5)])
    batch.assign(torch.tensor([1, -1, 0]))
    y = mlp(x)
    assert torch.equal(y[1:], plain[1:]) and not torch.equal(y[0], plain[0])
    h = mlp.gate_up_proj(x)
    assert torch.equal(mlp.down_proj(mlp.act_fn(h)), y)


def plan_of(pkg, ids, slots):
    """ops.lora_plan's result, made on the host."""
    e = torch.where((ids < 0) | (ids >= slots), slots, ids)
    off = torch.cat([torch.zeros(1, dtype=torch.long), torch.bincount(e, minlength=slots + 1).cumsum(0)])
    return pkg.LoraPlan(off.int(), torch.argsort(e, stable=True).int())


def test_every_number_of_rows_has_its_own_plan(pkg):
    batch = pkg.AdapterBatch(3)
    g = torch.Generator().manual_seed(1)
    ids = {n: torch.randint(-1, 3, (n,), generator=g) for n in (1, 2, 3, 4, 5, 6, 7, 8)}
    kept = {n: batch._keep(plan_of(pkg, v, 3)) for n, v in ids.items()}
    for n, v in ids.items():
        assert all(torch.equal(a, b) for a, b in zip(kept[n], plan_of(pkg, v, 3))), n
    new = plan_of(pkg, torch.tensor([2, -1, 0, 1, 2]), 3)
    again = batch._keep(new)                              # the memory of five rows, written anew
    assert all(a.data_ptr() == b.data_ptr() for a, b in zip(again, kept[5]))
    assert all(torch.equal(a, b) for a, b in zip(kept[5], new))
    assert all(torch.equal(a, b) for a, b in zip(kept[6], plan_of(pkg, ids[6], 3)))


def test_clear_empties_the_kept_plans(pkg):
    batch = pkg.AdapterBatch(3)
    kept = [batch._keep(plan_of(pkg, torch.tensor([2, -1, 0, 1, 2])[:n], 3)) for n in (5, 3, 0)]
    batch.clear()
    for plan, n in zip(kept, (5, 3, 0)):
        assert plan.seg_off.tolist() == [0, 0, 0, 0, n]
        assert sorted(plan.rows.tolist()) == list(range(n))
    new = plan_of(pkg, torch.tensor([0, 1, 1]), 3)
    batch._keep(new)
    assert all(torch.equal(a, b) for a, b in zip(kept[1], new))


def test_plans_made_in_inference_mode_are_written_outside_it(pkg):
    batch = pkg.AdapterBatch(3)
    ids = torch.tensor([2, -1, 0, 1, 2])
    with torch.inference_mode():
        kept = batch._keep(plan_of(pkg, ids, 3))
    new = plan_of(pkg, ids.flip(0), 3)
    batch._keep(new)
    assert all(torch.equal(a, b) for a, b in zip(kept, new))
    batch.clear()
    with torch.inference_mode():
        batch._keep(plan_of(pkg, ids, 3))
    assert all(torch.equal(a, b) for a, b in zip(kept, plan_of(pkg, ids, 3)))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_what_the_base_returned_stays(pkg, dtype):
    """A hook on the base, or a base that keeps its output, sees it as the base made it."""
    base, batch = linear(pkg, 40, 32, 1), pkg.AdapterBatch(2)
    m = pkg.LoRALinear(base, batch, rank=8)
    m.load(0, [pair(8, 32, 40, 2)])
    batch.assign(torch.tensor([0, -1, 0]))
    x = torch.randn(3, 32).to(dtype)
    plain, seen = base(x).clone(), []
    handle = base.register_forward_hook(lambda mod, args, y: seen.append(y))
    y = m(x)
    handle.remove()
    assert torch.equal(seen[0], plain) and not torch.equal(y[0], plain[0])
    assert torch.equal(m(x), y)


def test_matrices_keep_their_types(pkg):
    """half(), float() and the like on a model that holds one: what the kernel reads stays."""
    base, batch = linear(pkg, 40, 32, 1), pkg.AdapterBatch(2)
    m = pkg.LoRALinear(base, batch, rank=8)
    m.load(0, [pair(8, 32, 40, 2)], scaling=1 / 3)
    batch.assign(torch.tensor([0, -1, 0]))
    x = torch.randn(3, 32).half()
    y, model = m(x), torch.nn.Sequential(m)
    for to in (model.half, model.float, model.double, model.bfloat16, lambda: model.to(torch.float16)):
        to()
        assert (m.a.dtype, m.b.dtype, m.scaling.dtype) == (torch.float16, torch.float16, torch.float32)
        assert torch.equal(m(x), y)
    model.to("meta")
    assert m.a.device.type == m.scaling.device.type == "meta" and m.scaling.dtype == torch.float32


def test_nothing_is_added_where_a_slot_has_nothing(pkg):
    """Rows with infinities keep what the base makes of them in empty and unloaded slots and in
    parts without an adapter; a rank that is filled up changes nothing."""
    g = torch.Generator().manual_seed(6)
    q = torch.randint(1, 128, (40, 32), generator=g, dtype=torch.int8)   # no 0: no NaN from inf
    base = pkg.LinearW8A8(pkg.QTensor(q, torch.rand(40, generator=g) * 0.01 + 0.01, scheme="per_row_i8"))
    batch = pkg.AdapterBatch(4)
    m = pkg.LoRALinear(base, batch, rank=16, splits=[24, 16])
    one, two = pair(1, 32, 24, 7), pair(1, 32, 16, 8)
    m.load(0, [None, two])
    m.load(1, [one, two])
    m.load(2, [one, two])
    m.unload(2)
    x = torch.randn(4, 32, generator=g).half()
    x[:, 5] = torch.inf
    plain = base(x)
    assert plain.isinf().all()
    batch.assign(torch.tensor([0, 1, 2, 3]))
    y = m(x)
    assert torch.equal(y[2:], plain[2:]) and torch.equal(y[0, :24], plain[0, :24])
    # one rank: an infinity of either sign times B, added to the base's plus infinity
    for p, (n, w, (a, b)) in enumerate(((0, 24, one), (24, 16, two))):
        up = torch.inf * torch.sign(a[0, 5].float()) * b[:, 0].float()
        assert torch.equal(y[1, n:n + w].isinf(), up > 0) and torch.equal(y[1, n:n + w].isnan(), up < 0)


def test_matrices_saved_without_ranks(pkg):
    """A state without them has all rows."""
    base = linear(pkg, 40, 32, 1)
    m, n = (pkg.LoRALinear(base, pkg.AdapterBatch(2), rank=8) for _ in range(2))
    m.load(1, [pair(8, 32, 40, 2)], scaling=0.5)
    state = m.state_dict()
    n.load_state_dict(state)
    assert torch.equal(n.ranks, m.ranks) and n.ranks.tolist() == [[0], [8]]
    del state["ranks"]
    k = pkg.LoRALinear(base, pkg.AdapterBatch(2), rank=8)
    k.load_state_dict(state)
    x, ids = torch.randn(3, 32).half(), torch.tensor([1, -1, 0])
    for t in (m, n, k):
        t.batch.assign(ids)
    assert torch.equal(n(x), m(x)) and torch.equal(k(x), m(x))
    assert k.ranks.tolist() == [[8], [8]]


def test_without_ids_it_has_the_rule_of_its_base(pkg):
    """The fused chains take it as they take its base, unless calling it does more."""
    gpu = SimpleNamespace(is_cuda=True)
    batch = pkg.AdapterBatch(2)
    m = pkg.LoRALinear(linear(pkg, 40, 32, 1), batch, rank=8)
    assert m._int8_ok(gpu) and not m._int8_ok(torch.zeros(1, 32))
    batch.assign(torch.tensor([0]))
    assert not m._int8_ok(gpu)
    batch.clear()
    assert m._int8_ok(gpu)
    for module in (m, m.base):
        handle = module.register_forward_hook(lambda *a: None)
        assert not m._int8_ok(gpu)
        handle.remove()
        assert m._int8_ok(gpu)
    handle = torch.nn.modules.module.register_module_forward_hook(lambda *a: None)
    assert not m._int8_ok(gpu)
    handle.remove()
    m.base.forward = m.base.forward
    assert not m._int8_ok(gpu)
    class Other(pkg.LoRALinear):
        pass
    assert not Other(linear(pkg, 40, 32, 1), batch, rank=8)._int8_ok(gpu)
