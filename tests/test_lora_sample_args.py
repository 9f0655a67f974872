"""What lora_plan, lora_add, sample and their C entry points refuse, without a GPU."""
import ctypes
import math
import random
from importlib import import_module

import pytest
import torch


@pytest.fixture(scope="module")
def lib(pkg):
    return import_module("fni8serve_amd._lib").load()


P = ctypes.c_void_p
F = ctypes.c_float
FAKE = P(0x1000)  # never dereferenced: every call below fails its checks


def lora(lib, **kw):
    c = dict(x=FAKE, ldx=64, T=4, K=64, a=FAKE, b=FAKE, S=2, rank=16, splits=[32, 16], scaling=None,
             seg_off=FAKE, rows=FAKE, y=FAKE, ldy=48, out=FAKE, ldo=48, work=FAKE, bytes=1 << 30)
    c.update(kw)
    n = c["splits"]
    n = None if n is None else (ctypes.c_int64 * len(n))(*n)
    return lib.fni8_lora_add_f16(c["x"], c["ldx"], c["T"], c["K"], c["a"], c["b"], c["S"], c["rank"],
                                 n, c.get("parts", 0 if n is None else len(n)), c["scaling"],
                                 c["seg_off"], c["rows"], c["y"], c["ldy"], c["out"], c["ldo"],
                                 c["work"], c["bytes"], None)


def test_lora_entry_refuses(lib):
    for name in ("x", "a", "b", "splits", "seg_off", "rows", "y", "out"):
        assert lora(lib, **{name: None}) == -1, name
    for kw in (dict(T=-1), dict(T=(1 << 23) + 1), dict(K=0), dict(K=1 << 24, ldx=1 << 24), dict(S=0),
               dict(S=65535), dict(rank=0), dict(rank=12), dict(rank=264), dict(rank=-8),
               dict(splits=[48, 0]), dict(splits=[-1, 49]), dict(splits=[4] * 9),
               dict(splits=[48], parts=0), dict(splits=[1 << 23]),
               dict(splits=[(1 << 23) - 1, 2], ldy=1 << 24, ldo=1 << 24), dict(bytes=16)):
        assert lora(lib, **kw) == -2, kw
        assert lib.fni8_last_error()
    for kw in (dict(ldx=63), dict(ldy=47, ldo=47), dict(ldo=47, out=P(0x2000)), dict(ldo=56)):
        assert lora(lib, **kw) == -4, kw
    for kw in (dict(a=P(0x1008)), dict(b=P(0x1002)), dict(x=P(0x1001)), dict(y=P(0x1001)),
               dict(scaling=P(0x1002)), dict(seg_off=P(0x1001)), dict(rows=P(0x1002)),
               dict(work=P(0x1080)), dict(work=None)):
        assert lora(lib, **kw) == -3, kw


def test_lora_workspace(lib):
    size = lib.fni8_lora_workspace_bytes
    assert size(0, 64, 2, 32) == 0 and size(4, 0, 2, 32) == 0 and size(4, 64, 0, 32) == 0
    assert size(4, 64, 2, 0) == 0 and size(4, 64, 2, 4096) == 0 and size(-1, 64, 2, 32) == 0
    for T in (1, 16, 300, 8192, 1 << 20):
        for K in (8, 4096, 12288):
            for R in (8, 48, 768):
                assert size(T, K, 8, R) >= T * R * 4 and size(T, K, 8, R) % (T * R * 4) == 0


def sample(lib, **kw):
    c = dict(x=FAKE, B=2, V=100, ld=100, u=None, tokens=FAKE, logprobs=None, work=FAKE, bytes=1 << 30,
             temperature=None, top_k=None, top_p=None, min_p=None, fp32=0)
    c.update(kw)
    return lib.fni8_sample(c["x"], c["fp32"], c["B"], c["V"], c["ld"], c["u"], c["temperature"], F(1.0),
                           c["top_k"], 0, c["top_p"], F(1.0), c["min_p"], F(0.0), c["tokens"],
                           c["logprobs"], c["work"], c["bytes"], None)


def test_sample_entry_refuses(lib):
    assert sample(lib, x=None) == -1 and sample(lib, tokens=None) == -1
    for kw in (dict(B=-1), dict(B=(1 << 20) + 1), dict(V=0), dict(V=(1 << 22) + 1, ld=1 << 23)):
        assert sample(lib, **kw) == -2, kw
    assert sample(lib, ld=99) == -4
    for kw in (dict(x=P(0x1001)), dict(x=P(0x1002), fp32=1), dict(u=P(0x1002)), dict(tokens=P(0x1004)),
               dict(logprobs=P(0x1002)), dict(temperature=P(0x1002)), dict(top_k=P(0x1001)),
               dict(top_p=P(0x1002)), dict(min_p=P(0x1002))):
        assert sample(lib, **kw) == -3, kw
    size = lib.fni8_sample_workspace_bytes
    assert size(-1, 100) == 0 and size(1, 0) == 0 and size(1, (1 << 22) + 1) == 0


def test_sample_refuses(pkg):
    x, u = torch.zeros(3, 10, dtype=torch.float16), torch.zeros(3)
    for kw in (dict(temperature=-1.0), dict(temperature=math.nan), dict(temperature=math.inf),
               dict(top_k=-1), dict(top_p=1.5), dict(top_p=-0.1), dict(top_p=math.nan),
               dict(min_p=2.0), dict(min_p=-1.0), dict(temperature=torch.ones(2)),
               dict(top_k=torch.ones(3)), dict(top_p=torch.ones(3, dtype=torch.int32)),
               dict(min_p=torch.ones(4)), dict(top_k=torch.ones(3, dtype=torch.bool))):
        with pytest.raises(ValueError, match=next(iter(kw))):
            pkg.sample(x, u, **kw)
    for bad in (x.bfloat16(), x.double(), x[:, :0], torch.zeros((), dtype=torch.float16)):
        with pytest.raises(ValueError, match="logits"):
            pkg.sample(bad, u)
    for bad in (u.double(), u[:2], u.unsqueeze(1), None):
        with pytest.raises(ValueError, match="u "):
            pkg.sample(x, bad)
    with pytest.raises(ValueError, match="u "):
        pkg.sample(x, None, temperature=torch.zeros(3))
    with pytest.raises(ValueError, match="GPU"):
        pkg.sample(x, u)


def test_lora_refuses(pkg):
    h = torch.float16
    y, x = torch.zeros(4, 48, dtype=h), torch.zeros(4, 64, dtype=h)
    a, b = torch.zeros(2, 32, 64, dtype=h), torch.zeros(2, 48, 16, dtype=h)
    plan = pkg.LoraPlan(torch.zeros(4, dtype=torch.int32), torch.zeros(4, dtype=torch.int32))
    ok = dict(y=y, x=x, a=a, b=b, plan=plan, splits=[32, 16])
    for name, bad in (("y", y.float()), ("x", x.bfloat16()), ("a", a.float()), ("b", b[0]),
                      ("a", a.transpose(0, 1)), ("splits", [32, 8]), ("splits", None),
                      ("splits", [16, 16, 16]), ("x", x[:, :60]), ("x", x[:3]), ("y", y[:, :40]),
                      ("plan", pkg.LoraPlan(plan.seg_off[:3], plan.rows)),
                      ("plan", pkg.LoraPlan(plan.seg_off, plan.rows[:3])),
                      ("plan", pkg.LoraPlan(plan.seg_off.long(), plan.rows)),
                      ("scaling", torch.ones(3)), ("scaling", torch.ones(2, dtype=h))):
        with pytest.raises(ValueError):
            pkg.lora_add(**dict(ok, **{name: bad}))
    with pytest.raises(ValueError, match="rank"):
        pkg.lora_add(y, x, torch.zeros(2, 24, 64, dtype=h), torch.zeros(2, 48, 12, dtype=h), plan,
                     splits=[32, 16])
    with pytest.raises(ValueError, match="GPU"):
        pkg.lora_add(**ok)
    for n in (0, -1, 65535):
        with pytest.raises(ValueError, match="num_adapters"):
            pkg.lora_plan(torch.zeros(4, dtype=torch.int32), n)
    with pytest.raises(ValueError, match="GPU"):
        pkg.lora_plan(torch.zeros(4, dtype=torch.int32), 2)


def test_lora_refuses_ranks(pkg, lib):
    h = torch.float16
    y, x = torch.zeros(4, 48, dtype=h), torch.zeros(4, 64, dtype=h)
    a, b = torch.zeros(2, 32, 64, dtype=h), torch.zeros(2, 48, 16, dtype=h)
    plan = pkg.LoraPlan(torch.zeros(4, dtype=torch.int32), torch.zeros(4, dtype=torch.int32))
    i = torch.int32
    for bad in (torch.zeros(2, dtype=i), torch.zeros(2, 1, dtype=i), torch.zeros(3, 2, dtype=i),
                torch.zeros(2, 2), torch.zeros(2, 2, dtype=torch.int64)):
        with pytest.raises(ValueError, match="ranks"):
            pkg.lora_add(y, x, a, b, plan, splits=[32, 16], ranks=bad)
    with pytest.raises(ValueError, match="GPU"):
        pkg.lora_add(y, x, a, b, plan, splits=[32, 16], ranks=torch.zeros(2, 2, dtype=i))
    splits = (ctypes.c_int64 * 2)(32, 16)
    rc = lib.fni8_lora_add_ranks_f16(FAKE, 64, 4, 64, FAKE, FAKE, 2, 16, splits, 2, None, P(0x1002),
                                     FAKE, FAKE, FAKE, 48, FAKE, 48, FAKE, 1 << 30, None)
    assert rc == -3 and lib.fni8_last_error()


def test_lora_refuses_an_out_that_overlaps_y(lib):
    """Every way that rows of two views can lie, against a set of their elements.  No workspace:
    a call that gets past this check fails at that one."""
    rng, seen = random.Random(1), {True: 0, False: 0}
    for _ in range(3000):
        T, N = rng.choice((1, 2, 3, 7)), rng.choice((1, 2, 5))
        ldy, ldo = N + rng.randint(0, 8), N + rng.randint(0, 8)
        if rng.random() < 0.5:
            ldo = ldy
        d = rng.randint(-60, 60)
        if d == 0:
            continue
        y = {t * ldy + n for t in range(T) for n in range(N)}
        out = {d + t * ldo + n for t in range(T) for n in range(N)}
        rc = lora(lib, T=T, splits=[N], y=P(0x1000), ldy=ldy, out=P(0x1000 + 2 * d), ldo=ldo,
                  work=None)
        assert rc == (-4 if y & out else -3), (T, N, ldy, ldo, d)
        seen[bool(y & out)] += 1
    assert min(seen.values()) > 300
    assert lora(lib, work=None) == -3                     # in place
    far = dict(T=1 << 23, ldy=1 << 24, ldo=1 << 24, work=None)
    assert lora(lib, **far, out=P(0x1000 + 2 * 48)) == -3   # two halves of the same rows
    assert lora(lib, **far, out=P(0x1000 + 2 * 47)) == -4
    assert lora(lib, **dict(far, ldo=(1 << 24) - 8), out=P(0x1000 + 2 * 48)) == -4


def test_sample_workspace_is_bounded(lib):
    """Rows beyond what 1 GiB holds take turns in it."""
    size = lib.fni8_sample_workspace_bytes
    for V in (1, 131, 2048, 2049, 8200, 50257, 151936, 1 << 22):
        one = size(1, V)
        assert 0 < one < 1 << 30 and size(2, V) == 2 * one and size(0, V) == 0
        for B in (256, 5000, 540000, 1 << 20):
            assert size(B, V) == one * min(B, (1 << 30) // one), (B, V)
