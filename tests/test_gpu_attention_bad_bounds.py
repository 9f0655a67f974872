"""Bounds of sequences that are none (not rising, not from 0, past the tokens): the call ends
and writes nothing outside its result."""
import ctypes
from importlib import import_module

import pytest
import torch

import attention_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("most", [1, 5, 300])
@pytest.mark.parametrize("starts", [[0, 60, 10, 60, 20], [-5, 3, 4, 5, 6], [7, 8, 9, 10, 11],
                                    [0, 1, 2, 3, 1 << 30], [60, 40, 30, 2, 0],
                                    [0, 60, 0, 60, 0], [-(1 << 31), (1 << 31) - 1, 0, 0, 60]])
def test_nothing_outside_the_result(pkg, cuda, starts, most, int8):
    T, Hq, Hk, D, page, lens = 60, 8, 2, 128, 16, [900, 70, 3000, 64]
    lib = import_module("fni8serve_amd._lib").load()
    q = torch.randn(T, Hq, D, generator=torch.Generator().manual_seed(1)).half().cuda()
    k, v, ks, vs, tables = (None if t is None else t.cuda() for t in
                            ref.paged(lens, page, Hk, D, 2, int8))
    n = lib.fni8_paged_attention_workspace_bytes(T, Hq, Hk, D, 4, most, tables.shape[1] * page)
    assert n > 0 and n % 256 == 0
    # the result and the workspace with 4 KB of marks on both sides
    out = torch.full((2048 + T * Hq * D + 2048,), 7.0, dtype=torch.float16, device="cuda")
    work = torch.full((4096 + n + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
    lengths = torch.tensor(lens, dtype=torch.int32).cuda()
    p = lambda t, at=0: None if t is None else ctypes.c_void_p(t.data_ptr() + at)  # noqa: E731

    def call(cu):
        cu = torch.tensor(cu, dtype=torch.int32).cuda()
        rc = lib.fni8_paged_attention_f16(
            p(q), Hq * D, D, T, Hq, Hk, D, p(k), p(v), p(ks), p(vs), k.shape[0], page, p(tables),
            tables.shape[1], tables.shape[1], p(lengths), p(cu), 4, most, ctypes.c_float(D ** -0.5),
            0, p(out, 4096), p(work, 4096), n,
            ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        assert rc == 0
        torch.cuda.synchronize()
        assert (out[:2048] == 7).all() and (out[-2048:] == 7).all()
        assert (work[:4096] == 0x5A).all() and (work[-4096:] == 0x5A).all()
        return out[2048:-2048].view(T, Hq, D).clone()

    good = call([0, 1, 40, 41, 60])
    call(starts)
    assert torch.equal(call([0, 1, 40, 41, 60]), good)
