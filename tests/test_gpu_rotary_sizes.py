"""RotaryEmbedding on the GPU at head sizes that the kernel does not take."""
import pytest
import torch

import attention_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,rotary,pairs", [(20, 20, False), (36, 10, True), (320, 320, False),
                                              (264, 64, True), (2, 2, False)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_any_even_head(pkg, cuda, dim, rotary, pairs, dtype):
    rot = pkg.RotaryEmbedding(dim, 300, rotary_dim=rotary, interleaved=pairs, device="cuda")
    g = torch.Generator().manual_seed(dim)
    q, k = (torch.randn(9, h, dim, generator=g).to(dtype) for h in (4, 2))
    pos = torch.randint(0, 300, (9,), generator=g)
    for y, x in zip(rot(q.cuda(), k.cuda(), pos.cuda()), (q, k)):
        want, tol = ref.norm_rope(x, None, pos, ref.table(300, rotary), pairs)
        assert y.dtype == dtype
        ref.within(y, want, tol)
