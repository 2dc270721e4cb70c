"""CPU definition of the log probabilities (TEST INFRASTRUCTURE ONLY: see oracle/__init__.py), in 64 bits.

Row x, temperature T (0, negative or NaN: 1), z = x / T with NaN logits at -inf and +inf ones at the largest fp32 value:
  log p_i = z_i - ln sum_j e^(z_j), -inf for a logit at -inf; entropy = -sum p_i log p_i, 0 for a row without a candidate;
  rank of i = tokens before it by (larger logit, lower index); alternatives: that order without the logits at -inf.
A given token outside [0, V): log probability 0, rank -1.  No alternative left: id -1, log probability -inf."""
import numpy as np

F32_MAX = float(np.finfo(np.float32).max)


def row(x, tokens=(), top=0, temperature=1.0):
    """x [V] fp32 or fp64 -> (log p of tokens, ranks, entropy, ids [top], their log p), float64 / int."""
    x = np.asarray(x, dtype=np.float64).copy()
    x[np.isnan(x)] = -np.inf
    x = np.minimum(x, F32_MAX) + 0.0
    T = float(temperature) if temperature > 0 else 1.0
    n = len(x)
    m = x.max()
    if m == -np.inf:
        lp, h = np.full(n, -np.inf), 0.0
    else:
        with np.errstate(over="ignore"):
            z = (x - m) / T
        e = np.exp(z)
        lp = z - np.log(e.sum())
        p = e / e.sum()
        h = -float((p[p > 0] * lp[p > 0]).sum())
    order = np.lexsort((np.arange(n), -x))
    place = np.empty(n, dtype=np.int64)
    place[order] = np.arange(n)
    inside = [0 <= t < n for t in tokens]
    of = np.array([lp[t] if ok else 0.0 for t, ok in zip(tokens, inside)], dtype=np.float64)
    ranks = np.array([place[t] if ok else -1 for t, ok in zip(tokens, inside)], dtype=np.int64)
    ids = np.full(top, -1, dtype=np.int64)
    best = [i for i in order[:top] if x[i] > -np.inf]
    ids[:len(best)] = best
    top_lp = np.full(top, -np.inf)
    top_lp[:len(best)] = lp[best]
    return of, ranks, h, ids, top_lp
