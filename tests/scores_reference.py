"""Plain 64-bit forms of the score-row operators, one row at a time, straight from their definitions."""
import numpy as np


def order(x):
    """Classes of a row that are present, best first, equal scores by ascending class."""
    x = np.asarray(x, np.float64)
    there = np.nonzero(x > -np.inf)[0]                    # NaN compares false
    return there[np.argsort(-x[there], kind="stable")]


def weights(x, o, t):
    """exp((x - best) / t) of the classes ``o`` of a row."""
    x = np.asarray(x, np.float64)[o]
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        return np.where(x == x[0], 1.0, np.exp((x - x[0]) / t))


def top(x, k, t):
    o = order(x)
    values = np.full(k, -np.inf)
    index = np.full(k, -1, np.int64)
    n = min(k, len(o))
    values[:n], index[:n] = np.asarray(x, np.float64)[o[:n]], o[:n]
    if len(o) <= k:
        return values, index, -np.inf
    far, best = o[k:], float(x[o[0]])
    gap = 0.0 if x[far[0]] == best else (float(x[far[0]]) - best) / t
    return values, index, gap + np.log(weights(x, far, t).sum())


def sample(x, u, t, top_k, top_p, min_p):
    o = order(x)
    if len(o) == 0:
        return -1, -np.inf
    if not t > 0:
        return int(o[0]), 0.0
    w = weights(x, o, t)
    if top_k > 0:
        o, w = o[:top_k], w[:top_k]
    if top_p < 1:
        n = 1 + int(np.argmax(np.cumsum(w) >= max(top_p, 0.0) * w.sum()))
        if n < len(o):
            o, w = o[:n], w[:n]
    if min_p > 0:
        xs = np.asarray(x, np.float64)
        n = int(np.sum(xs[o] >= xs[o[0]] + t * np.log(min(min_p, 1.0))))
        o, w = o[:n], w[:n]
    by_class = np.argsort(o)
    run = np.cumsum(w[by_class])
    hit = np.nonzero(run > min(max(u, 0.0), 1.0) * run[-1])[0]
    at = hit[0] if len(hit) else np.nonzero(w[by_class] > 0)[0][-1]
    with np.errstate(divide="ignore"):
        return int(o[by_class][at]), float(np.log(w[by_class][at] / run[-1]))


def _log_softmax(z):
    z = np.asarray(z, np.float64)
    m = z.max()
    if np.isposinf(m):                                    # all weight on the infinite ones
        with np.errstate(divide="ignore"):
            return np.log(np.isposinf(z) / np.isposinf(z).sum())
    with np.errstate(divide="ignore"):
        return z - m - np.log(np.exp(z - m).sum())


def distill(s, values, index, rest, t, weight=1.0):
    """(loss, gradient) of one row."""
    s = np.asarray(s, np.float64)
    n = len(s)
    entries = [(float(v), int(i)) for v, i in zip(values, index) if 0 <= i < n and v > -np.inf]
    if weight == 0 or not entries or np.all(s == -np.inf):
        return 0.0, np.zeros(n)
    if np.isnan(s).any() or np.isposinf(s).any():
        return np.nan, np.full(n, np.nan)
    best = max(v for v, _ in entries)
    z = [0.0 if v == best else (v - best) / t for v, _ in entries]
    log_p = _log_softmax(z + ([float(rest)] if rest is not None else []))
    log_q = _log_softmax(s / t)
    outside = np.ones(n, bool)
    outside[[i for _, i in entries]] = False
    p, loss = np.exp(log_p), 0.0
    for j, (_, i) in enumerate(entries):
        if p[j] > 0:
            loss += p[j] * (log_p[j] - log_q[i])
    grad = np.exp(log_q)
    for j, (_, i) in enumerate(entries):
        grad[i] -= p[j]
    if rest is not None:
        m = s[outside].max() if outside.any() else -np.inf
        if m > -np.inf:
            share = np.exp(np.where(outside, (s - m) / t, -np.inf))
            log_qr = np.log(share.sum()) + (m - s.max()) / t - np.log(np.exp((s - s.max()) / t).sum())
            grad -= p[-1] * share / share.sum()
        else:
            log_qr = -np.inf
        if p[-1] > 0:
            loss += p[-1] * (log_p[-1] - log_qr)
    return weight * t * t * loss, weight * t * grad
