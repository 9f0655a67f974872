"""What each request of a batch has of its own around the shared linears, as timed cases.

Two operators, in the order in which a serving step calls them:

  lora    low-rank adapters beside a projection: every token's output row gets the product
          of its own request's adapter added, in one call for all adapters of the batch; the
          parts of a merged projection (Q, K and V; gate and up) have adapters of their own
  sample  one token a row of logits, from given random numbers: temperature, top-k, top-p
          and min-p, the same for every row or each row's own, greedy rows among them

Sizes are those of Qwen3-8B (hidden 4096, intermediate 12288, QKV 4096 + 1024 + 1024,
vocabulary 151936), Qwen3-0.6B (hidden 1024), Qwen3-30B-A3B (hidden 2048) and generic ones.
"""
import importlib.util
import math
import os
import random
import sys

import numpy as np
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

def _sample(rows, vocab, **more):
    c = {"kind": "sample", "rows": rows, "vocab": vocab, "pad": 0, "fp32": False, "mixed": False,
         "temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "spread": 2.5, "peaks": 12,
         "allowed": 1.0, "logprobs": False}
    c.update(more)
    return c


def _lora(tokens, inner, outs, rank, adapters, **more):
    c = {"kind": "lora", "tokens": tokens, "inner": inner, "outs": outs, "rank": rank,
         "adapters": adapters, "run": 1, "bare": 0.0}
    c.update(more)
    return c


def listed():
    cases = [
        # single-stream chat with the usual settings: latency counts
        ("sample_1row_chat", _sample(1, 151936, temperature=0.6, top_k=20, top_p=0.95)),
        # a small vocabulary of odd size, soft-capped logits in 32 bits, log-probabilities asked
        ("sample_5row_fp32", _sample(5, 50257, fp32=True, temperature=0.8, top_p=0.9,
                                     logprobs=True)),
        # a serving batch, each request with settings of its own, a padded vocabulary
        ("sample_64row_mixed", _sample(64, 151936, pad=128, mixed=True)),
        # a large batch whose requests ask for top-p alone, as most interfaces offer it
        ("sample_256row_top_p", _sample(256, 151936, top_p=0.95)),
        # sampling from the whole distribution: rollouts
        ("sample_256row_free", _sample(256, 151936, logprobs=True)),
        # structured output (most of the vocabulary is masked) beside min-p, fairly flat rows
        ("sample_48row_masked", _sample(48, 32000, fp32=True, temperature=1.3, min_p=0.02,
                                        spread=1.5, peaks=0, allowed=0.03)),
        # single-stream decode, merged QKV: latency counts
        ("lora_1tok_qkv", _lora(1, 4096, "4096+1024+1024", 16, 8)),
        # a decode batch in which every request has its own adapter, merged gate and up
        ("lora_48tok_gate_up", _lora(48, 4096, "12288+12288", 16, 48)),
        # a decode batch over a few adapters of high rank, some requests without one
        ("lora_64tok_down", _lora(64, 12288, "4096", 64, 8, bare=0.2)),
        # the vocabulary projection of a small batch
        ("lora_16tok_head", _lora(16, 4096, "151936", 16, 4)),
        # ragged chunks of prompts beside decoding requests, the smallest model
        ("lora_777tok_o", _lora(777, 2048, "1024", 8, 6, run=100, bare=0.1)),
        # a large prefill batch over four adapters
        ("lora_8192tok_qkv", _lora(8192, 4096, "4096+1024+1024", 32, 4, run=1500)),
    ]
    return [dict(c, name=n) for n, c in cases]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# the largest listed cases: logits of a call in bytes; bytes and operations of a call
_MOST_LOGITS = 256 * 151936 * 2
_MOST_BYTES, _MOST_FLOPS = 272000000, 9600000000

_PROJECTIONS = (
    (4096, "4096+1024+1024"), (4096, "4096"), (4096, "12288+12288"), (12288, "4096"),
    (1024, "2048+1024+1024"), (2048, "1024"), (2048, "4096+512+512"), (1536, "1000"),
    (1000, "520+88"), (4096, "32000"), (896, "50257"),
)


def draw(rng):
    if rng.random() < 0.5:
        fp32 = rng.random() < 0.4
        vocab = rng.choice((32000, 50257, 151936, _log_int(rng, 1000, 151936)))
        rows = _log_int(rng, 1, min(256, _MOST_LOGITS // (vocab * (4 if fp32 else 2))))
        c = _sample(rows, vocab, fp32=fp32, pad=rng.choice((0, 0, 64, 7)),
                    spread=rng.uniform(1.0, 4.0), peaks=rng.choice((0, 4, 12, 40)),
                    allowed=rng.choice((1.0, 1.0, 1.0, 0.05)), logprobs=rng.random() < 0.5)
        form = rng.choice(("greedy", "free", "k", "p", "kp", "min", "mixed"))
        c["mixed"] = form == "mixed"
        c["temperature"] = 0.0 if form == "greedy" else rng.uniform(0.3, 1.5)
        if form in ("k", "kp"):
            c["top_k"] = _log_int(rng, 1, 500)
        if form in ("p", "kp"):
            c["top_p"] = rng.uniform(0.5, 0.99)
        if form == "min":
            c["min_p"] = rng.uniform(0.005, 0.2)
        return c
    inner, outs = rng.choice(_PROJECTIONS)
    tokens, bare = _log_int(rng, 1, 8192), rng.choice((0.0, 0.0, 0.1, 0.5))
    c = _lora(tokens, inner, outs, rng.choice((8, 16, 16, 24, 32, 64, 128)),
              _log_int(rng, 1, 64), run=_log_int(rng, 1, max(1, tokens // 2)), bare=bare)
    while (w := work(c))["bytes"] > _MOST_BYTES or w["flops"] > _MOST_FLOPS:
        c["tokens"], c["adapters"] = -(-c["tokens"] * 2 // 3), -(-c["adapters"] * 2 // 3)
        c["run"] = min(c["run"], max(1, c["tokens"] // 2))
    return c


# ---- inputs --------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _settings(case, seed):
    """Each row's own settings, or one for all of them."""
    names = ("temperature", "top_k", "top_p", "min_p")
    if not case["mixed"]:
        return {n: case[n] for n in names}
    rng = random.Random(seed)
    rows = [rng.choice(((0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.0), (0.6, 20, 0.95, 0.0),
                        (0.7, 40, 0.8, 0.0), (rng.uniform(0.3, 1.3), 0, 0.9, 0.0),
                        (1.2, 0, 1.0, 0.05), (rng.uniform(0.5, 1.0), 200, 1.0, 0.0)))
            for _ in range(case["rows"])]
    kinds = (torch.float32, torch.int32, torch.float32, torch.float32)
    return {n: torch.tensor([r[i] for r in rows], dtype=kinds[i], device="cuda")
            for i, n in enumerate(names)}


def _parts(case):
    return [int(n) for n in case["outs"].split("+")]


def prepare(case, seed):
    g = _gen(seed)
    if case["kind"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # a wide bell with some tokens that stand out, one row more than another
        x = torch.randn(rows, vocab + case["pad"], generator=g, device="cuda") * case["spread"]
        if case["peaks"]:
            at = torch.randint(0, vocab, (rows, case["peaks"]), generator=g, device="cuda")
            up = torch.rand(rows, case["peaks"], generator=g, device="cuda") * 8 + 4
            x.scatter_add_(1, at, up)
        if case["allowed"] < 1:
            off = torch.rand(rows, vocab + case["pad"], generator=g, device="cuda") > case["allowed"]
            off[:, vocab // 2] = False
            x.masked_fill_(off, -math.inf)
        x[:, vocab:] = math.nan
        x = x if case["fp32"] else x.half()
        return {"case": case, "logits": x[:, :vocab],
                "u": torch.rand(rows, generator=g, device="cuda"), "set": _settings(case, seed)}
    tokens, inner, rank, count = case["tokens"], case["inner"], case["rank"], case["adapters"]
    parts = _parts(case)
    # requests one after the other, each with an adapter or without
    rng, ids = random.Random(seed), []
    while len(ids) < tokens:
        run = 1 if case["run"] == 1 else _log_int(rng, 1, 2 * case["run"])
        which = -1 if rng.random() < case["bare"] else rng.randrange(count)
        if case["run"] == 1 and count >= tokens and which >= 0:
            which = len(ids)
        ids += [which] * run
    ids = torch.tensor(ids[:tokens], dtype=torch.int32, device="cuda")
    # hidden states: N(0, 1) with 1% outliers of twenty times the size
    x = torch.randn(tokens, inner, generator=g, device="cuda")
    x = torch.where(torch.rand(tokens, inner, generator=g, device="cuda") < 0.01, x * 20, x)
    a = torch.randn(count, len(parts) * rank, inner, generator=g, device="cuda",
                    dtype=torch.float16) * inner ** -0.5
    b = torch.randn(count, sum(parts), rank, generator=g, device="cuda",
                    dtype=torch.float16) * 0.02
    scaling = torch.rand(count, generator=g, device="cuda") * 2 + 0.5
    y = torch.randn(tokens, sum(parts), generator=g, device="cuda", dtype=torch.float16) * 2
    state = {"case": case, "x": x.half(), "y": y, "a": a, "b": b, "scaling": scaling}
    # which tokens belong to which adapter is found once a step, for all of its projections
    if own:
        state["plan"] = _ops().lora_plan(ids, count)
    else:
        state["plan"] = [(e, at) for e in range(count)
                         if (at := (ids == e).nonzero().squeeze(1)).numel()]
    return state


# ---- the operators in their plain form -------------------------------------------

def _column(v, like):
    return v[:, None] if torch.is_tensor(v) else torch.full((like.shape[0], 1), v,
                                                            device=like.device)


def _plain_sample(state):
    x, case = state["logits"].float(), state["case"]
    heat, k, p, least = (_column(state["set"][n], x) for n in ("temperature", "top_k", "top_p",
                                                               "min_p"))
    vocab = x.shape[1]
    x, order = torch.sort(x, dim=1, descending=True, stable=True)
    greedy = heat == 0
    z = (x.double() - x[:, :1].double()) / torch.where(greedy, 1, heat).double()
    w = z.exp()
    rank = torch.arange(vocab, device=x.device)
    keep = (rank < torch.where(k > 0, k, vocab)) & ~(greedy & (rank > 0))
    w = w * keep
    total = w.cumsum(1)
    keep &= (total - w < p.double() * total[:, -1:]) | (p >= 1)
    keep &= w >= least.double()
    keep |= rank == 0
    w = w * keep
    mass = w.sum(1, keepdim=True)
    placed = torch.zeros_like(w).scatter_(1, order, w)           # in vocabulary order again
    passed = placed.cumsum(1) <= state["u"].double()[:, None] * mass
    at = torch.arange(vocab, device=x.device)
    last = torch.where(placed > 0, at, -1).amax(1)
    token = torch.minimum(passed.sum(1), last)
    if not case["logprobs"]:
        return token
    return token, (placed.gather(1, token[:, None]) / mass).log().squeeze(1).float()


def _plain_lora(state):
    case, x, y = state["case"], state["x"], state["y"]
    rank, out = case["rank"], y.clone()
    for e, at in state["plan"]:
        low = torch.matmul(x[at].float(), state["a"][e].float().t()) * state["scaling"][e]
        n = 0
        for i, wide in enumerate(_parts(case)):
            up = torch.matmul(low[:, i * rank:(i + 1) * rank],
                              state["b"][e, n:n + wide].float().t())
            out[at, n:n + wide] = (y[at, n:n + wide].float() + up).half()
            n += wide
    return out


def run(state):
    case = state["case"]
    if case["kind"] == "sample":
        if not own:
            return _plain_sample(state)
        return _ops().sample(state["logits"], state["u"], return_logprobs=case["logprobs"],
                             **state["set"])
    if not own:
        return _plain_lora(state)
    return _ops().lora_add(state["y"], state["x"], state["a"], state["b"], state["plan"],
                           scaling=state["scaling"], splits=_parts(case))


# ---- the same in 64 bits ---------------------------------------------------------

def _exact_row(x, u, heat, k, p, least):
    """Token and log-probability of one row: the kept tokens are a prefix of the order."""
    best = int(np.argmax(x))
    if heat == 0:
        return best, 0.0
    alive = np.flatnonzero(x > -np.inf)
    alive = alive[np.argsort(-x[alive], kind="stable")]
    w = np.exp((x[alive] - x[best]) / heat)
    n = len(alive) if k <= 0 else min(int(k), len(alive))
    if p < 1:
        running = np.cumsum(w[:n])
        n = min(n, 1 + int(np.count_nonzero(running[:-1] < p * running[-1])))
    n = max(1, min(n, int(np.count_nonzero(w >= least))))
    spot = np.argsort(alive[:n])
    running = np.cumsum(w[:n][spot])
    j = min(int(np.searchsorted(running, u * running[-1], side="right")), n - 1)
    return int(alive[spot[j]]), float(np.log(w[spot[j]] / running[-1]))


def _exact_sample(case, state):
    x, u = state["logits"].double().cpu().numpy(), state["u"].double().cpu().numpy()
    values = [state["set"][n] for n in ("temperature", "top_k", "top_p", "min_p")]
    # settings in 32 bits, as the call takes them
    values = [v.tolist() if torch.is_tensor(v) else [float(np.float32(v))] * len(u) for v in values]
    rows = [_exact_row(x[i], u[i], *(v[i] for v in values)) for i in range(len(u))]
    token = torch.tensor([r[0] for r in rows], device="cuda")
    if not case["logprobs"]:
        return token
    return token, torch.tensor([r[1] for r in rows], dtype=torch.float64, device="cuda")


def _exact_lora(case, state):
    out = state["y"].double()
    rank, edges = case["rank"], np.cumsum([0] + _parts(case)).tolist()
    if own:
        seg, rows = state["plan"][0].tolist(), state["plan"][1].long()
        groups = [(e, rows[seg[e]:seg[e + 1]]) for e in range(case["adapters"])]
    else:
        groups = state["plan"]
    for e, at in groups:
        if at.numel():
            a, b = state["a"][e].double(), state["b"][e].double()
            wide = torch.cat([b[lo:hi] @ a[i * rank:(i + 1) * rank] for i, (lo, hi)
                              in enumerate(zip(edges, edges[1:]))])      # the whole update
            out[at] += state["scaling"][e].double() * (state["x"][at].double() @ wide.T)
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return _exact_sample(case, state) if case["kind"] == "sample" else _exact_lora(case, state)


def work(case):
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["fp32"] else 2) + case["rows"] * (4 + 8 + 4),
                "flops": 3 * n}
    tokens, inner, parts = case["tokens"], case["inner"], _parts(case)
    wide, rank = sum(parts), case["rank"]
    carried = tokens * (1 - case["bare"])                        # tokens with an adapter
    requests = max(1.0, tokens / case["run"]) * (1 - case["bare"])
    # a batch over fewer adapters than requests uses nearly all of them
    used = case["adapters"] * (1 - (1 - 1 / case["adapters"]) ** requests) \
        if case["run"] > 1 or case["adapters"] < tokens else carried
    return {"bytes": int(2 * carried * inner + 4 * tokens * wide
                         + 2 * used * rank * (len(parts) * inner + wide)),
            "flops": int(2 * carried * rank * (len(parts) * inner + wide))}
