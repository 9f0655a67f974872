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


@pytest.mark.parametrize("dtype", [torch.float16, torch.int8])
def test_reading_outside_the_cache(pkg, dtype):
    """Slots of padding and past the cache read as NaN, beside those that are there."""
    cache = pkg.PagedKVCache(3, 16, 2, 32, dtype, device="cpu")
    for x in (cache.k, cache.v):
        x.copy_(torch.randint(-9, 9, x.shape, generator=torch.Generator().manual_seed(1)))
    if dtype == torch.int8:
        cache.k_scale.fill_(0.5), cache.v_scale.fill_(0.25)
    slots = torch.tensor([-1, 47, 48, -(1 << 31), (1 << 31) - 1, 5], dtype=torch.int32)
    for got, x, s in zip(cache.read(slots), (cache.k, cache.v), (0.5, 0.25)):
        s = s if dtype == torch.int8 else 1.0
        assert got[[0, 2, 3, 4]].isnan().all()
        assert torch.equal(got[1], x[2, :, 15].float() * s)
        assert torch.equal(got[5], x[0, :, 5].float() * s)
    assert cache.read(slots[:0])[0].shape == (0, 2, 32)
    assert cache.read(torch.tensor([1 << 40]))[1].isnan().all()
