"""The attention block between a decoder layer's QKV and O projections, as timed cases.

Four operators, in the order in which a serving step calls them:

  rope       rotary positions on queries and keys: adjacent pairs or halves of the
             head, all of it or its first `rotary` elements
  norm_rope  an RMS norm of every query and key head, and the rotation, in one pass
  append     norm and rotation of a step's queries and keys, the keys and values
             appended to the paged cache (16 bits, or 8 bits with one scale a row)
  attention  the step's queries over the paged cache: one token a sequence (decode),
             a few (verification of drafted tokens), or a chunk of a prompt, with
             each sequence's own length, causal, with or without a window

The inputs are views of one merged QKV row, as the projection leaves them.  Head
counts and sizes are those of Qwen3-0.6B (16 + 8 heads of 128), Qwen3-8B (32 + 8)
and Qwen3-30B-A3B (32 + 4), and generic ones.
"""
import importlib.util
import math
import os
import random
import sys

import torch

own = False


def _ops():
    """The tensor-level entry points of the package in `fni8-serve_amd`."""
    name = "fni8serve_amd"
    if name not in sys.modules:
        home = os.path.join(os.getcwd(), "fni8-serve_amd")
        spec = importlib.util.spec_from_file_location(
            name, os.path.join(home, "__init__.py"), submodule_search_locations=[home])
        sys.modules[name] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[name])
    return sys.modules[name].ops


# ---- the cases -----------------------------------------------------------------

def _rows(kind, tokens, heads, kv_heads, dim, rotary, **more):
    c = {"kind": kind, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
         "rotary": rotary, "interleaved": False, "page": 0, "pages": 0, "int8": False,
         "norm": kind != "rope", "far": 40960}
    c.update(more)
    return c


def _attn(seqs, q_min, q_max, old_min, old_max, heads, kv_heads, dim, page, **more):
    c = {"kind": "attention", "seqs": seqs, "q_min": q_min, "q_max": q_max, "old_min": old_min,
         "old_max": old_max, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
         "int8": False, "window": 0, "mix": 1}
    c.update(more)
    return c


def listed():
    cases = [
        # a short prompt; adjacent pairs, half of a small head rotated
        ("rope_7tok_pairs", _rows("rope", 7, 16, 8, 64, 32, interleaved=True, far=8192)),
        # a large prefill batch of a model without query and key norms
        ("rope_8192tok", _rows("rope", 8192, 32, 8, 128, 128)),
        # single-stream decode of the smallest model: the smallest call
        ("norm_rope_1tok", _rows("norm_rope", 1, 16, 8, 128, 128)),
        # a ragged prefill chunk
        ("norm_rope_4097tok", _rows("norm_rope", 4097, 32, 4, 128, 128)),
        # a decode batch, one new token in each of 48 sequences, into 8 bits
        ("append_int8_48tok", _rows("append", 48, 32, 8, 128, 128, page=16, pages=64, int8=True)),
        # a prefill chunk into 16 bits
        ("append_4096tok", _rows("append", 4096, 32, 8, 128, 128, page=64, pages=80)),
        # single-stream decode early in a conversation: latency counts
        ("decode_1seq", _attn(1, 1, 1, 776, 776, 16, 8, 128, 16)),
        # a decode batch of conversations of very different length
        ("decode_64seq_ragged", _attn(64, 1, 1, 200, 16000, 32, 8, 128, 16)),
        # four long documents, the cache in 8 bits
        ("decode_int8_4seq_long", _attn(4, 1, 1, 30000, 65000, 32, 4, 128, 64, int8=True)),
        # five drafted tokens verified in each of 16 sequences
        ("verify_int8_16seq", _attn(16, 5, 5, 500, 6000, 32, 8, 128, 16, int8=True)),
        # the next chunk of one long prompt: the largest work
        ("chunk_2048_over_14k", _attn(1, 2048, 2048, 14336, 14336, 32, 8, 128, 64)),
        # chunks of several prompts beside decoding sequences, small heads, a window
        ("mixed_12seq_window", _attn(12, 1, 600, 0, 5000, 16, 4, 64, 32, window=1024)),
    ]
    return [dict(c, name=n) for n, c in cases]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# the largest listed attention case, in (query, key) pairs of one element of one head, and
# in padded scores; the largest cache that a decode case reads, in elements
_MOST_PAIRS = 2048 * 15000 * 32 * 128
_MOST_SCORES = 2048 * 16384 * 32
_MOST_CACHE = 64 * 16000 * 8 * 128


def draw(rng):
    kind = rng.choice(("rope", "norm_rope", "append", "attention", "attention", "attention"))
    dim = rng.choice((64, 80, 96, 128, 128, 256))
    kv_heads = rng.choice((1, 2, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 4, 4, 5, 8))
    if kind != "attention":
        rotary = rng.choice((dim, dim, dim // 2, 2 * rng.randint(4, dim // 2)))
        # at most the bytes of the largest listed case of rows
        most = 8192 * 40 * 128 // ((heads + 2 * kv_heads) * dim)
        c = _rows(kind, _log_int(rng, 1, min(8192, most)), heads, kv_heads, dim, rotary,
                  interleaved=rng.random() < 0.4, far=rng.choice((8192, 40960, 131072)))
        if kind == "append":
            c["page"] = rng.choice((16, 32, 64, 128))
            c["pages"] = -(-c["tokens"] // c["page"]) + rng.randint(1, 16)
            c["int8"] = rng.random() < 0.5
            c["norm"] = rng.random() < 0.7
        return c
    seqs, mix = _log_int(rng, 1, 64), rng.randrange(1 << 20)
    form = rng.choice(("decode", "verify", "chunk", "mixed"))
    lo, hi = {"decode": (1, 1), "verify": (2, 8), "chunk": (64, 2048), "mixed": (0, 700)}[form]
    q_max = hi if form == "decode" else _log_int(rng, max(2, lo), hi)
    q_min = {"decode": 1, "verify": q_max, "chunk": max(1, q_max // 2), "mixed": 0}[form]
    room = min(_MOST_PAIRS // (seqs * q_max * heads * dim), _MOST_SCORES // (seqs * q_max * heads),
               _MOST_CACHE // (seqs * kv_heads * dim), 60000) - q_max
    while room < 16 and seqs > 1:
        seqs = max(1, seqs // 2)
        room = min(_MOST_PAIRS // (seqs * q_max * heads * dim),
                   _MOST_SCORES // (seqs * q_max * heads),
                   _MOST_CACHE // (seqs * kv_heads * dim), 60000) - q_max
    old_max = _log_int(rng, 16, max(17, room))
    return _attn(seqs, q_min, q_max, rng.choice((0, old_max // 8, old_max)), old_max, heads,
                 kv_heads, dim, rng.choice((16, 32, 64, 128)), int8=rng.random() < 0.4,
                 window=rng.choice((0, 0, 0, 100, 1024)), mix=mix)


def _lengths(case):
    """New tokens and tokens in all (the new ones among them) of every sequence."""
    rng = random.Random(case["mix"])
    new = [rng.randint(case["q_min"], case["q_max"]) for _ in range(case["seqs"])]
    new[0] = case["q_max"]
    old = [_log_int(rng, max(1, case["old_min"]), max(1, case["old_max"])) if case["old_max"] else 0
           for _ in new]
    old[0] = case["old_max"]
    return new, [a + b if a else b for a, b in zip(new, old)]


# ---- inputs --------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _quantized(x):
    """Rows of 8 bits and their scales, as the cache holds them."""
    s = x.float().abs().amax(-1, keepdim=True).clamp_min(1e-6) / 127
    return torch.round(x.float() / s).clamp_(-127, 127).to(torch.int8), s.squeeze(-1)


def prepare(case, seed):
    g = _gen(seed)
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "attention":
        new, full = _lengths(case)
        page, tokens = case["page"], sum(new)
        width = max(1, -(-max(full) // page))
        # every sequence's pages lie anywhere in the cache
        need = [-(-n // page) for n in full]
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        tables = torch.zeros(len(full), width, dtype=torch.int32, device="cuda")
        at = 0
        for i, n in enumerate(need):
            tables[i, :n] = order[at:at + n]
            at += n
        # keys and queries as norms with learned weights leave them: scores of a few units
        cache = torch.empty(2, pages, kv, page, dim, dtype=torch.float16, device="cuda")
        cache.normal_(generator=g)
        scale = None
        if case["int8"]:
            cache, scale = _quantized(cache)
        wide = torch.randn(tokens, (heads + 2 * kv) * dim, generator=g, device="cuda",
                           dtype=torch.float16) * 1.5
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        return {"case": case, "q": wide[:, :heads * dim].unflatten(1, (heads, dim)),
                "cache": cache, "scale": scale, "tables": tables, "full": ints(full),
                "starts": ints(starts), "most_new": max(new), "most": max(full)}
    tokens, rotary = case["tokens"], case["rotary"]
    wide = torch.randn(tokens, (heads + 2 * kv) * dim, generator=g, device="cuda",
                       dtype=torch.float16) * 2
    q, k, v = (t.unflatten(1, (-1, dim)) for t in wide.split([heads * dim, kv * dim, kv * dim], 1))
    far = case["far"]
    # a batch of decoded tokens stands anywhere, a prompt's chunk is one run of positions
    if tokens <= 64:
        pos = torch.randint(0, far, (tokens,), generator=g, device="cuda")
    else:
        pos = torch.randint(0, far - tokens + 1, (1,), generator=g, device="cuda") \
            + torch.arange(tokens, device="cuda")
    freq = 1e6 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
    angle = torch.arange(far, dtype=torch.float64, device="cuda")[:, None] * freq
    state = {"case": case, "q": q, "k": k, "v": v, "pos": pos.to(torch.int32),
             "table": torch.cat([angle.cos(), angle.sin()], 1).float()}
    for name in ("q_weight", "k_weight"):
        w = 1 + 0.3 * torch.randn(dim, generator=g, device="cuda")
        state[name] = w.half() if case["norm"] else None
    if case["kind"] == "append":
        page, pages = case["page"], case["pages"]
        # whole pages in any order, tokens in order within a run; old contents stay around them
        order = torch.randperm(pages, generator=g, device="cuda")
        at = torch.arange(tokens, device="cuda")
        if tokens <= 64:
            at = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
        state["slots"] = (order[at // page] * page + at % page).to(torch.int32)
        old = torch.randn(2, pages, kv, page, dim, generator=g, device="cuda", dtype=torch.float16)
        state["cache"], state["scale"] = _quantized(old) if case["int8"] else (old, None)
    return state


# ---- the operators in their plain form -------------------------------------------

def _plain_rows(x, weight, pos, table, interleaved):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight.float()
    r = table.shape[1]
    cos, sin = table[pos.long()].unsqueeze(1).chunk(2, -1)
    turn, rest = x[..., :r], x[..., r:]
    a, b = (turn[..., 0::2], turn[..., 1::2]) if interleaved else turn.chunk(2, -1)
    a, b = a * cos - b * sin, b * cos + a * sin
    turn = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turn, rest], -1).half()


def _plain_append(state, k, v):
    cache, scale, page = state["cache"], state["scale"], state["case"]["page"]
    slots = state["slots"].long()
    at, off = slots // page, slots % page
    rows = torch.stack([k, v])
    if scale is None:
        cache[:, at, :, off] = rows.transpose(0, 1)
        return
    codes, s = _quantized(rows)
    cache[:, at, :, off] = codes.transpose(0, 1)
    scale[:, at, :, off] = s.transpose(0, 1)


def _plain_attention(state):
    case, q, cache, scale = state["case"], state["q"], state["cache"], state["scale"]
    full, starts = state["full"].long(), state["starts"].long()
    heads, kv, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    tokens, most_new, most = q.shape[0], state["most_new"], state["most"]
    group = heads // kv
    dev = q.device
    j = torch.arange(most, device=dev)
    at, off = state["tables"].long()[:, j // page], (j % page).expand(len(full), most)

    def gathered(n):
        rows = cache[n][at, :, off].float()
        if scale is not None:
            rows *= scale[n][at, :, off].unsqueeze(-1)
        return rows.permute(0, 2, 1, 3)                          # [seqs, kv, most, dim]

    new = starts[1:] - starts[:-1]
    i = torch.arange(most_new, device=dev)
    rows = q[(starts[:-1, None] + i).clamp_max(tokens - 1)].float()
    rows = rows.unflatten(2, (kv, group)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    scores = torch.matmul(rows, gathered(0).transpose(2, 3)).mul_(dim ** -0.5)
    pos = (full - new)[:, None] + i                              # [seqs, most_new]
    seen = (j <= pos[..., None]) & (j < full[:, None, None])
    if case["window"]:
        seen &= j > pos[..., None] - case["window"]
    hidden = ~seen[:, None, None]
    scores = scores.unflatten(2, (group, most_new)).masked_fill_(hidden, -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top.isinf(), 0, top)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.flatten(2, 3), gathered(1)).unflatten(2, (group, most_new))
    out = (out / total.clamp_min(1e-30)).permute(0, 3, 1, 2, 4)  # [seqs, most_new, kv, group, dim]
    t = torch.arange(tokens, device=dev)
    seq = torch.bucketize(t, starts[1:], right=True)
    return out[seq, t - starts[seq]].reshape(tokens, heads, dim).half()


def run(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "attention":
        if not own:
            return _plain_attention(state)
        k_scale, v_scale = (None, None) if state["scale"] is None else state["scale"]
        return _ops().paged_attention(
            state["q"], state["cache"][0], state["cache"][1], state["tables"], state["full"],
            state["starts"], max_seqlen=state["most_new"], k_scale=k_scale, v_scale=v_scale,
            window=case["window"] or None)
    q, k, pos, table, pairs = (state["q"], state["k"], state["pos"], state["table"],
                               case["interleaved"])
    if kind != "append":
        if not own:
            return (_plain_rows(q, state["q_weight"], pos, table, pairs),
                    _plain_rows(k, state["k_weight"], pos, table, pairs))
        if kind == "rope":
            return _ops().rope(q, k, pos, table, interleaved=pairs)
        return _ops().qk_norm_rope(q, k, state["q_weight"], state["k_weight"], pos, table,
                                   eps=1e-6, interleaved=pairs)
    if own:
        k_scale, v_scale = (None, None) if state["scale"] is None else state["scale"]
        q = _ops().rope_append(q, k, state["v"], pos, table, state["cache"][0], state["cache"][1],
                               state["slots"], k_scale=k_scale, v_scale=v_scale,
                               q_weight=state["q_weight"], k_weight=state["k_weight"], eps=1e-6,
                               interleaved=pairs)
    else:
        q = _plain_rows(q, state["q_weight"], pos, table, pairs)
        _plain_append(state, _plain_rows(k, state["k_weight"], pos, table, pairs), state["v"])
    if state["scale"] is None:
        return q, state["cache"]
    # the cache's codes as the values that they stand for, rounded to 16 bits
    values = torch.empty_like(state["cache"], dtype=torch.float16)
    return q, torch.mul(state["cache"], state["scale"].unsqueeze(-1), out=values)


# ---- the same in 64 bits ---------------------------------------------------------

def _exact_rows(x, weight, pos, table, interleaved):
    y = x.double().clone()
    if weight is not None:
        y /= ((y * y).sum(-1, keepdim=True) / y.shape[-1] + 1e-6).sqrt()
        y *= weight.double()
    half = table.shape[1] // 2
    angles = table.double()[pos.long()]
    for n in range(half):
        a, b = (2 * n, 2 * n + 1) if interleaved else (n, n + half)
        c, s = angles[:, n, None], angles[:, n + half, None]
        u, w = y[:, :, a].clone(), y[:, :, b].clone()
        y[:, :, a] = u * c - w * s
        y[:, :, b] = u * s + w * c
    return y


def _exact_attention(case, state):
    new, full = _lengths(case)
    heads, kv, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    group, start = heads // kv, 0
    out = torch.zeros(sum(new), heads, dim, dtype=torch.float64, device="cuda")
    for s, (n, length) in enumerate(zip(new, full)):
        if n and length:
            ids = state["tables"][s, :-(-length // page)].long()
            keys, values = (state["cache"][m][ids].transpose(1, 2).flatten(0, 1)[:length].double()
                            for m in (0, 1))                     # [length, kv, dim]
            if state["scale"] is not None:
                ks, vs = (state["scale"][m][ids].transpose(1, 2).flatten(0, 1)[:length].double()
                          for m in (0, 1))
                keys, values = keys * ks[..., None], values * vs[..., None]
            where = torch.arange(length - n, length, device="cuda")[:, None]
            ahead = torch.arange(length, device="cuda")[None] - where
            for h in range(heads):
                z = state["q"][start:start + n, h].double() @ keys[:, h // group].T / math.sqrt(dim)
                z[ahead > 0] = -math.inf
                if case["window"]:
                    z[ahead <= -case["window"]] = -math.inf
                out[start:start + n, h] = torch.softmax(z, -1) @ values[:, h // group]
        start += n
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "attention":
        return _exact_attention(case, state)
    pos, table, pairs = state["pos"], state["table"], case["interleaved"]
    q = _exact_rows(state["q"], state["q_weight"], pos, table, pairs)
    k = _exact_rows(state["k"], state["k_weight"], pos, table, pairs)
    if case["kind"] != "append":
        return q, k
    page, old = case["page"], state["cache"].double()
    if state["scale"] is not None:
        old = old * state["scale"].double()[..., None]
    slots = state["slots"].long()
    for n, rows in enumerate((k, state["v"].double())):
        if case["int8"]:  # rows of 16 bits in codes of 8
            rows = rows.half().double()
            step = rows.abs().amax(-1, keepdim=True).clamp_min(1e-6) / 127
            rows = torch.round(rows / step).clamp(-127, 127) * step
        flat = old[n].transpose(1, 2).flatten(0, 1).clone()      # [slots, kv, dim]
        flat[slots] = rows
        old[n] = flat.unflatten(0, (-1, page)).transpose(1, 2)
    return q, old


def work(case):
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "attention":
        new, full = _lengths(case)
        window, pairs, keys = case["window"] or 1 << 40, 0, 0
        for n, length in zip(new, full):
            pairs += sum(min(p + 1, window) for p in range(length - n, length))
            keys += min(length, n - 1 + window) if n else 0
        row = dim + 4 if case["int8"] else 2 * dim
        moved = 2 * sum(new) * heads * dim * 2 + 2 * keys * kv * row
        return {"bytes": moved + 4 * keys // case["page"] + 8 * len(new),
                "flops": 4 * pairs * heads * dim}
    tokens, rotary = case["tokens"], case["rotary"]
    moved = tokens * (4 + 4 * rotary + heads * dim * 4)          # positions, table rows, queries
    if case["kind"] == "append":
        row = dim + 4 if case["int8"] else 2 * dim
        moved += tokens * (4 + 2 * kv * (2 * dim + row))         # slots, keys and values
    else:
        moved += tokens * kv * dim * 4
    return {"bytes": moved,
            "flops": tokens * (heads + kv) * (3 * rotary + (4 * dim if case["norm"] else 0))}
