"""Decoded tokens without `cu_seqlens` and `max_seqlen`: the call takes the workspace, and
the split of the keys, of one token a sequence."""
import pytest
import torch

from test_gpu_host_path import general  # noqa: F401

pytestmark = pytest.mark.gpu


def _bytes(call):
    """What `call` takes from the allocator, and its result."""
    before = torch.cuda.memory_stats()["allocated_bytes.all.allocated"]
    out = call()
    return torch.cuda.memory_stats()["allocated_bytes.all.allocated"] - before, out


@pytest.mark.parametrize("B,Hq,Hk,pages", [(2, 32, 8, 64), (5, 32, 8, 40), (16, 16, 2, 26),
                                           (64, 32, 8, 128), (256, 32, 8, 128), (512, 32, 4, 64)])
def test_one_token_a_sequence_is_known(pkg, cuda, general, B, Hq, Hk, pages):  # noqa: F811
    D, page = 128, 16
    g = torch.Generator(device="cuda").manual_seed(B)
    cache = torch.randn(2, pages, Hk, page, D, device="cuda", generator=g).half()
    tables = torch.arange(pages, device="cuda").int().expand(B, pages).contiguous()
    lens = torch.randint(1, 200, (B,), device="cuda", generator=g).int()
    lens[B // 2] = pages * page
    q = torch.randn(B, Hq, D, device="cuda", generator=g).half()
    cu = torch.arange(B + 1, device="cuda").int()
    args = (q, cache[0], cache[1], tables, lens)
    calls = [lambda: pkg.paged_attention(*args, cu, max_seqlen=1),
             lambda: pkg.paged_attention(*args), lambda: pkg.paged_attention(*args, max_seqlen=7)]
    (n, want), *others = [_bytes(c) for c in calls]
    with general():
        others += [_bytes(c) for c in calls]
    for m, got in others:
        assert m == n
        # the same cut of the keys: the same bits
        assert torch.equal(got, want)
