"""GQAAttention calls its norms and its rotation where calling them is more than what their
class defines: hooks, forwards of their own, subclasses, norms that differ."""
import pytest
import torch

from test_gpu_attention_layer import _cache, _layer

pytestmark = pytest.mark.gpu


def _stages(layer, x, cache, step):
    """The layer, every module called."""
    D, nq, nk = layer.head_dim, layer.num_heads * layer.head_dim, layer.num_kv_heads * layer.head_dim
    q, k, v = (t.unflatten(-1, (-1, D)) for t in layer.qkv_proj(x).split([nq, nk, nk], -1))
    q = layer.q_norm(q) if layer.q_norm is not None else q
    k = layer.k_norm(k) if layer.k_norm is not None else k
    if layer.rotary is not None:
        q, k = layer.rotary(q, k, step.positions)
    q = cache.append(q, k, v, step)
    return layer.o_proj(cache.attend(q, step, layer.scale, layer.window).flatten(1))


def _both(pkg, layer, change, dtype=torch.float16):
    """(with `change` made to the layer, its stages called, the layer unchanged): outputs."""
    x = torch.randn(30, 256, generator=torch.Generator().manual_seed(1)).half().cuda()
    caches = [_cache(pkg, layer, [64, 40], 16, dtype)[0] for _ in range(3)]
    tables = _cache(pkg, layer, [64, 40], 16, dtype)[1]
    step = caches[0].step(tables, [29, 1], [29, 1])
    plain = layer(x, caches[2], step)
    change(layer)
    got, want = layer(x, caches[0], step), _stages(layer, x, caches[1], step)
    assert torch.equal(got, want) and torch.equal(caches[0].k, caches[1].k)
    return got, plain


def _hook_q(layer):
    layer.q_norm.register_forward_hook(lambda m, a, out: out * 2)


def _hook_rotary(layer):
    layer.rotary.register_forward_hook(lambda m, a, out: (out[0], out[1] * 0.5))


def _pre_hook_k(layer):
    layer.k_norm.register_forward_pre_hook(lambda m, a: (a[0] + 1,))


def _own_forward(layer):
    old = layer.k_norm.forward
    layer.k_norm.forward = lambda x: old(x) * 3


def _own_rotary_forward(layer):
    layer.rotary.forward = lambda q, k, positions: (q, -k)


def _other_eps(layer):
    layer.k_norm.eps = 0.5


def _other_weights(layer):
    layer.q_norm.weight.data = layer.q_norm.weight.data.float() * 2


@pytest.mark.parametrize("change", [_hook_q, _hook_rotary, _pre_hook_k, _own_forward,
                                    _own_rotary_forward, _other_eps, _other_weights])
def test_parts_are_called(pkg, cuda, change):
    got, plain = _both(pkg, _layer(pkg), change)
    assert not torch.equal(got, plain)


def test_a_subclass_is_called(pkg, cuda):
    class Shifted(pkg.RotaryEmbedding):
        def forward(self, q, k, positions):
            return super().forward(q, k, positions + 7)

    class Doubled(pkg.RMSNorm):
        def forward(self, x, residual=None):
            return super().forward(x, residual) * 2

    def rotary(layer):
        layer.rotary = Shifted(64, 4096, rotary_dim=32, device="cuda")

    def norm(layer):
        layer.q_norm = Doubled(64).cuda()

    for change in (rotary, norm):
        got, plain = _both(pkg, _layer(pkg), change)
        assert not torch.equal(got, plain)


def test_hooks_on_every_module(pkg, cuda):
    """A global hook sees the norms and the rotation."""
    layer, seen = _layer(pkg), []
    cache, tables = _cache(pkg, layer, [64], 16, torch.float16)
    step = cache.step(tables, [3], [3])
    x = torch.randn(3, 256, generator=torch.Generator().manual_seed(1)).half().cuda()
    h = torch.nn.modules.module.register_module_forward_hook(
        lambda m, a, out: seen.append(type(m).__name__))
    try:
        layer(x, cache, step)
    finally:
        h.remove()
    assert sorted(seen) == sorted(["LinearW8A8", "RMSNorm", "RMSNorm", "RotaryEmbedding",
                                   "LinearW8A8", "GQAAttention"])


def test_plain_parts_stay_one_launch(pkg, cuda):
    """Without any of that, norms and rotation go with the append."""
    from importlib import import_module
    layer = _layer(pkg)
    cache, tables = _cache(pkg, layer, [64], 16, torch.float16)
    step = cache.step(tables, [3], [3])
    x = torch.randn(3, 256, generator=torch.Generator().manual_seed(1)).half().cuda()
    ops, calls = import_module("fni8serve_amd.ops"), []
    kept = ops.rope_append
    ops.rope_append = lambda *a, **kw: calls.append((a, kw)) or kept(*a, **kw)
    try:
        layer(x, cache, step)
    finally:
        ops.rope_append = kept
    (a, kw), = calls
    assert a[4] is layer.rotary.cos_sin and kw["q_weight"] is layer.q_norm.weight


def test_a_step_without_tokens(pkg, cuda):
    layer = _layer(pkg)
    cache, tables = _cache(pkg, layer, [64, 64], 16, torch.float16)
    for hook in (False, True):
        if hook:
            _hook_q(layer)
        y = layer(torch.empty(0, 256, dtype=torch.float16, device="cuda"), cache,
                  cache.step(tables, [0, 0], [5, 0]))
        assert y.shape == (0, 256)
    assert cache.k.count_nonzero() == 0
