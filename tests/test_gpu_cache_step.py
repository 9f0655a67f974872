"""PagedKVCache.step and the slots on the GPU: no wait for the GPU, wherever the block tables
lie."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture
def no_sync():
    """A wait for the GPU by torch raises."""
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    yield
    torch.cuda.set_sync_debug_mode("default")


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("where", ["cpu", "cuda"])
@pytest.mark.parametrize("view", [False, True])
def test_a_step_does_not_wait(pkg, cuda, no_sync, where, dtype, view):
    host = torch.tensor([[7, 2, 0], [5, 9, 1], [3, 0, 1 << 28]], dtype=dtype)
    wide = torch.full((3, 5), -1, dtype=dtype)
    wide[:, 1:4] = host
    pinned = (wide if view else host).pin_memory()
    tables = pinned.to(where, non_blocking=True) if where == "cuda" else (wide if view else host)
    if view:
        tables = tables[:, 1:4]
    cache = pkg.PagedKVCache(10, 16, 2, 64)
    step = cache.step(tables, new=[3, 1, 2], total=[18, 33, 33])
    slots = cache.slots(step.block_tables, torch.zeros_like(step.positions), step.positions)
    torch.cuda.set_sync_debug_mode("default")
    assert step.positions.tolist() == [15, 16, 17, 32, 31, 32]
    assert step.slots.tolist()[:5] == [7 * 16 + 15, 2 * 16, 2 * 16 + 1, 1 * 16, 15]
    assert not 0 <= step.slots[5].item() < 160
    assert step.cu_seqlens.tolist() == [0, 3, 4, 6] and step.context_lens.tolist() == [18, 33, 33]
    assert step.block_tables.tolist() == host.tolist()
    assert step.block_tables.is_cuda and step.block_tables.dtype == torch.int32
    assert slots.tolist() == [7 * 16 + 15, 2 * 16, 2 * 16 + 1, 0, 2 * 16 + 15, 0]


def test_positions_outside_the_table_are_dropped(pkg, cuda):
    """Padding and far positions write nothing and stop nothing."""
    cache = pkg.PagedKVCache(4, 16, 1, 64)
    tables = torch.tensor([[3, 1 << 28], [0, 2]], dtype=torch.int32, device="cuda")
    seq = torch.tensor([0, 0, 1, 1, 5, -1, 1], device="cuda")
    pos = torch.tensor([2, 16, -1, 32, 3, 3, 16], device="cuda")
    slots = cache.slots(tables, seq, pos)
    k = torch.ones(7, 1, 64, dtype=torch.float16, device="cuda")
    pkg.rope_append(k, k, k, None, None, cache.k, cache.v, slots)
    want = torch.zeros(4, 16)
    want[3, 2] = want[2, 0] = 1
    for c in (cache.k, cache.v):
        assert torch.equal(c[:, 0].float().cpu(), want[..., None].expand(4, 16, 64))
    got, _ = cache.read(slots)
    assert (got[[0, 6]] == 1).all() and got[1:6].isnan().all()
