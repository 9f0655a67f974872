"""RotaryEmbedding, the cache's bookkeeping and the attention entry points' refusals, on the
CPU."""
import ctypes
import math

import pytest
import torch

import attention_ref as ref


@pytest.mark.parametrize("dim,rotary,pairs", [(64, None, False), (64, 32, True), (80, 20, False)])
def test_rotation_on_the_cpu(pkg, dim, rotary, pairs):
    rot = pkg.RotaryEmbedding(dim, 300, base=1e4, rotary_dim=rotary, interleaved=pairs)
    g = torch.Generator().manual_seed(dim)
    q, k = torch.randn(9, 4, dim, generator=g), torch.randn(9, 2, dim, generator=g).half()
    pos = torch.randint(0, 300, (9,), generator=g)
    for y, x in zip(rot(q, k, pos), (q, k)):
        want, tol = ref.norm_rope(x, None, pos, ref.table(300, rotary or dim), pairs)
        assert y.dtype == x.dtype
        ref.within(y, want, tol)


def test_table_is_exact_at_far_positions(pkg):
    """The last position of a long table: fp32 of the 64-bit cosine and sine."""
    P, R = 200000, 64
    rot = pkg.RotaryEmbedding(R, P, base=1e6)
    for i in range(R // 2):
        a = (P - 1) * 1e6 ** (-2 * i / R)
        # pow and the product round the angle by a few steps of 2^-52
        tol = 2.0 ** -24 + a * 2.0 ** -50
        assert abs(rot.cos_sin[P - 1, i].item() - math.cos(a)) <= tol
        assert abs(rot.cos_sin[P - 1, R // 2 + i].item() - math.sin(a)) <= tol


def test_scaling(pkg):
    def angles(scaling, base=1e4, R=64):
        rot = pkg.RotaryEmbedding(R, 2, base=base, scaling=scaling)
        return torch.atan2(rot.cos_sin[1, R // 2:].double(), rot.cos_sin[1, :R // 2].double())

    plain = angles(None)
    assert torch.allclose(angles({"type": "linear", "factor": 4}), plain / 4, rtol=1e-5)
    ntk = angles({"type": "ntk", "factor": 4})
    assert torch.allclose(ntk[0], plain[0]) and torch.allclose(ntk[-1], plain[-1] / 4, rtol=1e-4)
    n = 4096
    yarn = angles({"type": "yarn", "factor": 8, "original_max_position": n})
    turns = n * plain / (2 * math.pi)
    fast, slow = turns > 2 * 32, turns < 1 / 2  # away from the ramp's rounded ends
    assert fast.any() and slow.any()
    assert torch.allclose(yarn[fast], plain[fast], rtol=1e-5)
    assert torch.allclose(yarn[slow], plain[slow] / 8, rtol=1e-4)
    assert ((yarn <= plain * (1 + 1e-5)) & (yarn >= plain / 8 * (1 - 1e-4))).all()
    rot = pkg.RotaryEmbedding(64, 2, scaling={"type": "yarn", "factor": 8,
                                              "original_max_position": n})
    assert torch.allclose(rot.cos_sin[0, :32], torch.full((32,), 0.1 * math.log(8) + 1))


def test_rotary_refusals(pkg):
    for kw in (dict(rotary_dim=66), dict(rotary_dim=3), dict(rotary_dim=0), dict(max_position=0),
               dict(base=1.0), dict(scaling={"type": "cubic", "factor": 2}),
               dict(scaling={"type": "linear", "factor": 0.5}), dict(scaling={"type": "linear"}),
               dict(scaling={"type": "yarn", "factor": 2}),
               dict(scaling={"type": "yarn", "factor": 2, "original_max_position": 64,
                             "beta_slow": 0})):
        args = dict(head_dim=64, max_position=8)
        args.update(kw)
        with pytest.raises(ValueError):
            pkg.RotaryEmbedding(**args)


def test_positions_outside_the_table_on_the_cpu(pkg):
    rot = pkg.RotaryEmbedding(16, 8, rotary_dim=8)
    q, _ = rot(torch.ones(4, 2, 16), torch.ones(4, 1, 16), torch.tensor([0, -1, 8, 1 << 40]))
    assert q[0].isfinite().all() and q[1:, :, :8].isnan().all()
    assert (q[..., 8:] == 1).all()


def test_table_stays_fp32(pkg):
    rot = pkg.RotaryEmbedding(64, 8)
    kept = rot.cos_sin.clone()
    rot.half()
    assert rot.cos_sin.dtype == torch.float32 and torch.equal(rot.cos_sin, kept)
    assert rot.to("meta").cos_sin.is_meta


def test_step_positions_and_slots(pkg):
    cache = pkg.PagedKVCache(10, 16, 2, 64, device="cpu")
    tables = torch.tensor([[7, 2, 0], [5, 9, 1], [3, 0, 0]])
    step = cache.step(tables, new=[3, 1, 0], total=[18, 33, 4])
    assert step.positions.tolist() == [15, 16, 17, 32]
    assert step.slots.tolist() == [7 * 16 + 15, 2 * 16, 2 * 16 + 1, 1 * 16]
    assert step.cu_seqlens.tolist() == [0, 3, 4, 4] and step.context_lens.tolist() == [18, 33, 4]
    assert step.max_seqlen == 3 and step.slots.dtype == torch.int32
    assert cache.step(tables[:0], [], []).max_seqlen == 0
    for new, total in (([1], [1]), ([1, 1, 5], [1, 1, 4]), ([-1, 1, 1], [1, 1, 1]),
                       ([1, 1, 1], [49, 1, 1])):
        with pytest.raises(ValueError):
            cache.step(tables, new, total)


def test_cache_read_and_refusals(pkg):
    cache = pkg.PagedKVCache(3, 16, 2, 32, torch.int8, device="cpu")
    cache.k[1, 1, 5], cache.k_scale[1, 1, 5] = 3, 0.5
    k, v = cache.read(torch.tensor([16 + 5, 0]))
    assert k.shape == (2, 2, 32) and (k[0, 1] == 1.5).all() and k[1].count_nonzero() == 0
    for args in ((0, 16, 1, 64), (4, 24, 1, 64), (4, 8, 1, 64), (4, 16, 0, 64), (4, 16, 1, 24),
                 (4, 16, 1, 272), (1 << 20, 4096, 1, 16)):
        with pytest.raises(ValueError):
            pkg.PagedKVCache(*args, device="meta")
    with pytest.raises(ValueError):
        pkg.PagedKVCache(4, 16, 1, 64, torch.bfloat16, device="cpu")


def _w(pkg, out, in_):
    return pkg.QTensor(torch.ones(out, in_, dtype=torch.int8), torch.ones(out), scheme="per_row_i8")


def test_layer_shapes_are_checked(pkg):
    rot = pkg.RotaryEmbedding(64, 8)
    ok = (_w(pkg, 8 * 64, 128), _w(pkg, 128, 4 * 64), 4, 2, 64, rot)
    layer = pkg.GQAAttention(*ok, q_norm=pkg.RMSNorm(64), k_norm=pkg.RMSNorm(64))
    assert layer.qkv_proj.out_features == 512
    for i, bad in ((0, _w(pkg, 7 * 64, 128)), (1, _w(pkg, 128, 3 * 64)), (3, 3),
                   (5, pkg.RotaryEmbedding(32, 8))):
        args = list(ok)
        args[i] = bad
        with pytest.raises(ValueError):
            pkg.GQAAttention(*args)
    with pytest.raises(ValueError):
        pkg.GQAAttention(*ok, q_norm=pkg.RMSNorm(64), k_norm=pkg.RMSNorm(64, eps=1e-5))
    with pytest.raises(ValueError):
        pkg.GQAAttention(*ok, q_norm=pkg.RMSNorm(32))


def test_entry_points_take_gpu_tensors_only(pkg):
    q = torch.zeros(2, 4, 64, dtype=torch.float16)
    c = torch.zeros(2, 4, 16, 64, dtype=torch.float16)
    i = torch.zeros(2, dtype=torch.int32)
    tab = torch.zeros(4, 64)
    for call in (lambda: pkg.rope(q, q, i, tab), lambda: pkg.qk_norm_rope(q, q, None, None, i, tab),
                 lambda: pkg.rope_append(q, q, q, i, tab, c, c, i),
                 lambda: pkg.paged_attention(q, c, c, i[:, None], i)):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_c_argument_errors_return_before_any_launch(pkg):
    from importlib import import_module
    lib = import_module("fni8serve_amd._lib").load()
    P = ctypes.c_void_p
    f = P(0x1000)  # never dereferenced
    e = ctypes.c_float(1e-6)
    NULL, SHAPE, ALIGN, STRIDE = -1, -2, -3, -4

    def rows(**kw):
        a = dict(q=f, ldq=256, hsq=64, Hq=4, k=f, ldk=128, hsk=64, Hk=2, T=3, D=64, qw=None,
                 kw=None, eps=e, unit=0, pos=f, tab=f, P=8, R=64, pairs=0, qo=f, ko=f, st=None)
        a.update(kw)
        return lib.fni8_qk_norm_rope_f16(*a.values())

    assert rows(q=None) == NULL and rows(qo=None) == NULL and rows(ko=None) == NULL
    assert rows(pos=None) == NULL and rows(tab=None) == NULL
    for kw in (dict(T=-1), dict(T=(1 << 23) + 1), dict(D=60), dict(D=264), dict(R=66), dict(R=3),
               dict(P=0), dict(Hq=-1), dict(eps=ctypes.c_float(float("nan")))):
        assert rows(**kw) == SHAPE, kw
    assert rows(hsq=56) == STRIDE and rows(ldk=32) == STRIDE
    assert rows(q=P(0x1008)) == ALIGN and rows(ldq=260) == ALIGN and rows(tab=P(0x1004)) == ALIGN

    def append(**kw):
        a = dict(q=f, ldq=256, hsq=64, Hq=4, k=f, ldk=128, hsk=64, Hk=2, v=f, ldv=128, hsv=64, T=3,
                 D=64, qw=None, kw=None, eps=e, unit=0, pos=f, tab=f, P=8, R=64, pairs=0, qo=f,
                 kc=f, vc=f, ks=None, vs=None, pages=4, page=16, slots=f, st=None)
        a.update(kw)
        return lib.fni8_rope_append_f16(*a.values())

    assert append(slots=None) == NULL and append(v=None) == NULL and append(kc=None) == NULL
    assert append(ks=f) == NULL
    for kw in (dict(page=24), dict(page=8), dict(pages=0), dict(pages=1 << 27), dict(D=72, ldq=512,
               hsq=72, ldk=512, hsk=72, ldv=512, hsv=72), dict(Hk=0)):
        assert append(**kw) == SHAPE, kw
    assert append(vc=P(0x1008)) == ALIGN and append(slots=P(0x1002)) == ALIGN

    def attn(**kw):
        a = dict(q=f, ldq=256, hsq=64, T=3, Hq=4, Hk=2, D=64, kc=f, vc=f, ks=None, vs=None, pages=4,
                 page=16, tables=f, ldt=2, width=2, lens=f, cu=None, B=3, most=1,
                 scale=ctypes.c_float(1.0), window=0, out=f, work=None, nw=0, st=None)
        a.update(kw)
        return lib.fni8_paged_attention_f16(*a.values())

    assert attn(out=None) == NULL and attn(tables=None) == NULL and attn(lens=None) == NULL
    for kw in (dict(T=4), dict(B=0), dict(B=65537, T=65537), dict(Hq=5), dict(Hq=0), dict(D=72),
               dict(width=0), dict(width=1 << 27, ldt=1 << 27), dict(window=-1), dict(most=-1),
               dict(scale=ctypes.c_float(float("inf")))):
        assert attn(**kw) == SHAPE, kw
    assert attn(ldt=1) == STRIDE
    assert attn(work=P(0x1010), nw=64) == ALIGN and attn(lens=P(0x1002)) == ALIGN
    n = lib.fni8_paged_attention_workspace_bytes
    assert n(64, 32, 8, 128, 64, 1, 16000) > 0 and n(0, 32, 8, 128, 64, 1, 16000) == 0
    assert n(64, 30, 8, 128, 64, 1, 16000) == 0 and n(64, 32, 8, 128, 64, 1, 0) == 0
