"""Plain 64-bit forms of the rotation, the cache append and paged attention, with the error
bounds that the kernels' roundings allow.  Used by the attention tests on the CPU and the
GPU; no kernel code is used here.

Bounds count half steps: a rounding to fp16 is off by 2^-11 of the value (2^-25 below the
normal range), one to fp32 by 2^-24.
"""
import math

import torch

H16, SUB16, H32 = 2.0 ** -11, 2.0 ** -25, 2.0 ** -24


def table(P, R, base=10000.0):
    """cos | sin of P positions, fp32 [P, R]."""
    f = base ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    a = torch.arange(P, dtype=torch.float64)[:, None] * f
    return torch.cat([a.cos(), a.sin()], 1).float()


def norm_rope(x, weight, pos, cos_sin, interleaved=False, eps=1e-6, unit=False):
    """Rows x [T, H, D] normed and rotated in 64 bits, and the bound of the kernel's error.

    The normed value carries the sum of squares (D products and sums: at most D half steps of
    fp32, halved by the root), the quotient, root and two products (4); the rotation two
    products and a sum (3): (D/2 + 8) half steps of |a c| + |b s|, then the rounding."""
    y = x.double()
    D = y.shape[-1]
    if weight is not None:
        w = weight.double() + (1.0 if unit else 0.0)
        y = y / (y.square().sum(-1, keepdim=True) / D + eps).sqrt() * w
    size = y.abs()
    if cos_sin is not None:
        R = cos_sin.shape[1]
        rows = cos_sin.double()[pos.long().clamp(0, cos_sin.shape[0] - 1)]
        bad = (pos < 0) | (pos >= cos_sin.shape[0])
        rows[bad] = math.nan
        c, s = rows[:, None, :R // 2], rows[:, None, R // 2:]
        i = torch.arange(R // 2)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
        ya, yb = y[..., a], y[..., b]
        y, size = y.clone(), size.clone()
        y[..., a], y[..., b] = ya * c - yb * s, yb * c + ya * s
        size[..., a] = (ya * c).abs() + (yb * s).abs()
        size[..., b] = (yb * c).abs() + (ya * s).abs()
    return y, H16 * y.abs() + SUB16 + (D / 2 + 8) * H32 * size * (1 + H16)


def rows_of(cache, scale, table_row, n):
    """The first n tokens of a sequence from its pages: [n, heads, D] in 64 bits."""
    page = cache.shape[2]
    ids = table_row[:-(-n // page)].long()
    x = cache[ids].transpose(1, 2).flatten(0, 1)[:n].double()
    if scale is not None:
        x = x * scale[ids].transpose(1, 2).flatten(0, 1)[:n].double()[..., None]
    return x


def attention(q, k_cache, v_cache, tables, lens, starts, k_scale=None, v_scale=None, scale=None,
              window=None):
    """(out, bound) [T, Hq, D] in 64 bits.

    Bound: the weights' rounding to fp16 is one half step of sum p |v| each (and 2^-25 of the
    largest weight, which is at most 1 of a sum that is at least 1, for every key); a score is
    off by its D products and sums, D half steps of fp32 of scale * sum |q k|, and 8 more for
    the scale, the maximum and the exponential, which moves its weight and the sum alike
    (twice); the sums over L keys and the joins of parts add L + 16 half steps of fp32; the
    result's own rounding."""
    T, Hq, D = q.shape
    Hk = k_cache.shape[1]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(T, Hq, D, dtype=torch.float64)
    tol = torch.full((T, Hq, D), SUB16, dtype=torch.float64)
    for s, L in enumerate(lens):
        a, b = starts[s], starts[s + 1]
        n = b - a
        if n == 0 or L == 0:
            continue
        K = rows_of(k_cache, k_scale, tables[s], L)
        V = rows_of(v_cache, v_scale, tables[s], L)
        p = torch.arange(n) + L - n
        ahead = torch.arange(L)[None] - p[:, None]
        hidden = ahead > 0
        if window:
            hidden |= ahead <= -window
        for h in range(Hq):
            k, v, x = K[:, h * Hk // Hq], V[:, h * Hk // Hq], q[a:b, h].double()
            z = (x @ k.T * scale).masked_fill(hidden, -math.inf)
            top = z.amax(-1, keepdim=True)
            e = torch.where(hidden, 0.0, (z - torch.where(top.isinf(), 0.0, top)).exp())
            l = e.sum(-1, keepdim=True)
            some = (l > 0).squeeze(-1)
            w = torch.where(l > 0, e / l.clamp_min(1e-300), 0.0)
            o = torch.where(hidden[..., None], 0.0, w[..., None] * v[None]).sum(1) \
                if n * L * D <= 1 << 24 else w @ v
            size = w @ v.abs()
            worst = (x.abs() @ k.abs().T * abs(scale)).masked_fill(hidden, 0.0).amax(-1)
            slip = 2 * ((D + 2) * worst + 8 * (1 + worst)) * H32
            bound = H16 * o.abs() + (H16 + slip[:, None] + (L + 16) * H32) * size \
                + SUB16 * ((~hidden).double() @ v.abs()) / l.clamp_min(1.0)
            out[a:b, h] = torch.where(some[:, None], o, 0.0)
            tol[a:b, h] += bound
    return out, tol


def paged(lens, page, Hk, D, seed, int8=False, spare=2, dtype=torch.float16):
    """A cache with each sequence's pages in any order: k, v, k_scale, v_scale, tables."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g).to(torch.int32)
    tables = torch.full((len(lens), max(1, max(need))), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = order[at:at + n]
        at += n
    k, v = (torch.randn(pages, Hk, page, D, generator=g).to(dtype) for _ in range(2))
    if not int8:
        return k, v, None, None, tables
    out = []
    for x in (k, v):
        s = x.float().abs().amax(-1, keepdim=True).clamp_min(1e-6) / 127
        out.append((torch.round(x.float() / s).clamp_(-127, 127).to(torch.int8), s.squeeze(-1)))
    return out[0][0], out[1][0], out[0][1], out[1][1], tables


def within(got, want, tol, what=""):
    """got is within tol of want, NaN where and only where want is."""
    got = got.double().cpu()
    nan = want.isnan()
    assert torch.equal(got.isnan(), nan), f"{what}: NaN in other places"
    off = torch.where(nan, 0.0, (got - want).abs())
    over = off / torch.where(nan, 1.0, tol)
    assert over.max() <= 1, (f"{what}: off by {over.max():.2f} of the bound at "
                             f"{torch.nonzero(over == over.max())[0].tolist()}")
