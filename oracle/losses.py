"""CPU definitions of the losses over drawn tokens with their gradients (TEST INFRASTRUCTURE ONLY: see oracle/__init__.py), in 64 bits.

Rows and their tokens' log probabilities are oracle/logprobs.py's (NaN logits -inf, +inf ones the largest fp32 value).  A row whose token
lies outside [0, V) is left out; one whose token has log probability -inf adds nothing and has no gradient."""
import numpy as np

F32_MAX = float(np.finfo(np.float32).max)
FAR = 80.0


def log_softmax(x, temperature=1.0):
    """x [V] -> log p, float64 (a row without a candidate: -inf)."""
    x = np.asarray(x, np.float64).copy()
    x[np.isnan(x)] = -np.inf
    x = np.minimum(x, F32_MAX)
    m = x.max()
    if m == -np.inf:
        return np.full(len(x), -np.inf)
    T = float(temperature) if temperature > 0 else 1.0
    with np.errstate(over="ignore"):
        z = (x - m) / T
    return z - np.log(np.exp(z).sum())


def _rows(x, tokens, temperature):
    V = x.shape[1]
    T = np.ones(len(x)) if temperature is None else np.where(np.asarray(temperature, np.float64) > 0, temperature, 1.0)
    table = [log_softmax(r, t) for r, t in zip(x, T)]
    has = np.array([0 <= t < V for t in tokens], bool)
    lp = np.array([l[t] if ok else 0.0 for l, t, ok in zip(table, tokens, has)], np.float64)
    return table, T, has, lp, has & (lp > -np.inf)


def _gradient(table, T, tokens, slope):
    g = np.zeros((len(table), len(table[0]) if len(table) else 0))
    for r, k in enumerate(slope):
        if k != 0:
            g[r] = -k * np.exp(table[r]) / T[r]
            g[r, tokens[r]] += k / T[r]
    return g


def policy(x, tokens, old, adv, clip=(0.2, 0.2), kl=0.0, ref=None, weights=None, temperature=None):
    """-> dict(loss, logprobs, ratio, kl, slope = dloss/dlogprobs, grad)"""
    table, T, has, lp, used = _rows(x, tokens, temperature)
    R = len(tokens)
    ratio, k, term, slope = np.ones(R), np.zeros(R), np.zeros(R), np.zeros(R)
    w = np.full(R, 1.0 / max(1, has.sum())) if weights is None else np.asarray(weights, np.float64)
    for i in np.flatnonzero(used):
        ratio[i] = np.exp(min(lp[i] - float(old[i]), FAR) if old[i] == old[i] else np.nan)
        a = float(adv[i])
        straight, clipped = ratio[i] * a, np.clip(ratio[i], 1 - clip[0], 1 + clip[1]) * a
        term[i] = -min(straight, clipped)
        slope[i] = -straight if straight <= clipped else 0.0
        if ref is not None:
            d = min(float(ref[i]) - lp[i], FAR)
            k[i] = np.expm1(d) - d
            term[i] += kl * k[i]
            slope[i] -= kl * np.expm1(d)
        term[i] *= w[i]
        slope[i] *= w[i]
    return dict(loss=term.sum(), logprobs=lp, ratio=ratio, kl=k, slope=slope, grad=_gradient(table, T, tokens, slope), table=table)


def preference(x, tokens, starts, beta=0.1, margin=0.0, smoothing=0.0, average=False, ref=None, weights=None):
    """-> dict(loss, logprobs [2 P], margins [P], token_logprobs, slope, grad)"""
    table, T, has, lp, used = _rows(x, tokens, None)
    P = len(starts) // 2
    seqs = [slice(starts[i], starts[i + 1]) for i in range(2 * P)]
    count = np.array([max(1, has[s].sum()) if average else 1 for s in seqs], np.float64)
    sums = np.array([lp[s][used[s]].sum() for s in seqs], np.float64) / count
    above = sums - (0.0 if ref is None else np.asarray(ref, np.float64))
    u = beta * (above[0::2] - above[1::2]) - margin
    w = np.full(P, 1.0 / max(1, P)) if weights is None else np.asarray(weights, np.float64)
    soft = lambda v: np.maximum(v, 0) + np.log1p(np.exp(-np.abs(v)))  # noqa: E731
    sigma = lambda v: np.exp(-soft(-v))  # noqa: E731
    loss = (w * ((1 - smoothing) * soft(-u) + smoothing * soft(u))).sum()
    du = w * (smoothing * sigma(u) - (1 - smoothing) * sigma(-u))
    slope = np.zeros(len(tokens))
    for i, s in enumerate(seqs):
        slope[s] = (-1.0 if i % 2 else 1.0) * beta * du[i // 2] / count[i] * used[s]
    return dict(loss=loss, logprobs=sums, margins=u, token_logprobs=lp, slope=slope, grad=_gradient(table, T, tokens, slope), table=table)
