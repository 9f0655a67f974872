"""One row of sampling from its definition, in 64 bits: the order by a stable sort, masses by
running sums, no histogram and no threshold."""
import numpy as np


def sample_row(x, u, temperature, top_k, top_p, min_p):
    """x float64 [V]; settings as numbers -> (token, logprob)."""
    if np.isnan(x).any() or np.isnan(temperature) or not (x > -np.inf).any():
        return -1, np.nan
    best = int(np.argmax(x))
    if temperature <= 0:
        return best, 0.0
    order = np.argsort(-x, kind="stable")
    with np.errstate(invalid="ignore"):
        z = np.where(x[order] == x[best], 0.0, (x[order] - x[best]) / temperature)
    z = np.where(x[order] == -np.inf, -np.inf, z)
    if x[best] == np.inf:
        z = np.where(x[order] == np.inf, 0.0, -np.inf)
    w = np.exp(z)
    V = len(x)
    n = top_k if 0 < top_k < V else V
    if top_p < 1:
        run = np.cumsum(w[:n])
        before = np.concatenate([[0.0], run[:-1]])
        n = min(n, max(1, int(np.count_nonzero(before < max(top_p, 0.0) * run[-1]))))
    if min_p > 0:
        n = min(n, max(1, int(np.count_nonzero(w >= min(min_p, 1.0)))))
    spot = np.argsort(order[:n])
    tokens, w, z = order[:n][spot], w[:n][spot], z[:n][spot]
    run = np.cumsum(w)
    u = 0.0 if not u > 0 else min(u, 1.0)
    j = int(np.searchsorted(run, u * run[-1], side="right"))
    j = min(j, int(np.flatnonzero(w > 0)[-1]))
    return int(tokens[j]), float(z[j] - np.log(run[-1]))
