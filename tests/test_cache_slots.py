"""Slots of the paged cache, on the CPU: what lies outside the table or the cache has none."""
import pytest
import torch


def _known(cache, slots):
    """Slots, with -1 for every one outside the cache."""
    assert slots.dtype == torch.int32
    inside = (slots >= 0) & (slots < cache.num_pages * cache.page_size)
    return torch.where(inside, slots, -1)


@pytest.mark.parametrize("page_size", [16, 64, 65536])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_pages_outside_the_cache(pkg, page_size, dtype):
    """Page numbers whose slots would wrap to valid ones in 32 bits."""
    cache = pkg.PagedKVCache(4, page_size, 1, 16, device="meta")
    bad = [1 << 28, 1 << 30, (1 << 31) - 1, 1 << 16, 4, -1, -7]
    if dtype == torch.int64:
        bad += [1 << 32, 1 << 60, (1 << 62) + 1, -(1 << 60)]
    tables = torch.tensor([[3, b] for b in bad], dtype=dtype)
    seq = torch.arange(len(bad)).repeat_interleave(3)
    pos = torch.tensor([page_size - 1, page_size, 2 * page_size - 1]).repeat(len(bad))
    want = torch.tensor([4 * page_size - 1, -1, -1]).repeat(len(bad)).int()
    assert torch.equal(_known(cache, cache.slots(tables, seq, pos)), want)
    assert torch.equal(_known(cache, cache.slots(tables, seq.int(), pos.int())), want)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_positions_outside_the_table(pkg, dtype):
    cache = pkg.PagedKVCache(10, 16, 1, 16, device="meta")
    tables = torch.tensor([[7, 2], [5, 9]])
    pos = torch.tensor([-1, -16, -17, 31, 32, (1 << 31) - 1, 0], dtype=dtype)
    seq = torch.tensor([0, 1, 0, 1, 0, 1, 1])
    got = _known(cache, cache.slots(tables, seq, pos))
    assert got.tolist() == [-1, -1, -1, 9 * 16 + 15, -1, -1, 5 * 16]
    for none in (tables[:, :0], tables[:0]):
        assert _known(cache, cache.slots(none, seq, pos)).tolist() == [-1] * 7
    row = torch.tensor([-1, 2, 1 << 40, 1])
    got = _known(cache, cache.slots(tables, row, torch.tensor([3, 3, 3, 3])))
    assert got.tolist() == [-1, -1, -1, 5 * 16 + 3]


def test_the_last_slot_of_the_largest_cache(pkg):
    cache = pkg.PagedKVCache((1 << 15) - 1, 65536, 1, 16, device="meta")
    tables = torch.tensor([[0, (1 << 15) - 2, (1 << 15) - 1]])
    got = cache.slots(tables, torch.tensor([0, 0, 0]), torch.tensor([65536, 131071, 3 * 65536 - 1]))
    end = ((1 << 15) - 1) * 65536
    assert _known(cache, got).tolist() == [end - 65536, end - 1, -1]


def test_a_step_with_a_page_outside_the_cache(pkg):
    """step() gives such tokens no slot, whatever the table's type."""
    cache = pkg.PagedKVCache(10, 16, 1, 16, device="cpu")
    for dtype in (torch.int32, torch.int64):
        tables = torch.tensor([[7, 1 << 28], [1 << 30, 3], [-1, 10]], dtype=dtype)
        step = cache.step(tables, [2, 3, 2], [17, 18, 17])
        assert _known(cache, step.slots).tolist() == [7 * 16 + 15, -1, -1, 3 * 16, 3 * 16 + 1, -1, -1]
