"""The operators over rows of scores from their definitions, in 64 bits, one row at a time (numpy only)."""
import numpy as np


def clean(row, allowed=None):
    row = np.asarray(row, np.float64).copy()
    row[np.isnan(row)] = -np.inf
    if allowed is not None:
        row[~allowed] = -np.inf
    return row


def ranked(row):
    """Indices by falling value, equal values by rising index (lexsort: the last key is the first one)."""
    return np.lexsort((np.arange(row.size), -row))


def log_sum_exp(z):
    m = z.max(initial=-np.inf)
    return -np.inf if m == -np.inf else m + np.log(np.exp(z - m).sum())


def top(row, k, temperature):
    row = clean(row)
    at = ranked(row)[:k]
    value = row[at]
    with np.errstate(invalid="ignore"):
        scaled = row / temperature
    return value, np.where(value > -np.inf, at, -1), log_sum_exp(scaled)


def weights(row, temperature):
    m = row.max()
    if m == -np.inf:
        return np.zeros_like(row)
    with np.errstate(invalid="ignore"):
        below = row - m  # -inf below an infinite maximum: no weight at any temperature
        w = np.exp(below / temperature)
    return np.where(row == m, 1.0, np.where(below > -np.inf, w, 0.0))


def kept(row, temperature, top_k, top_p, min_p):
    """(weights of the kept entries, 0 for the others)"""
    if not temperature > 0:
        temperature, top_k = 1.0, 1
    w = weights(row, temperature)
    at = ranked(row)
    n = row.size if top_k <= 0 else min(top_k, row.size)
    s = w[at[:n]]
    before = np.concatenate([[0.0], np.cumsum(s)[:-1]])
    keep = np.ones(n, bool)
    if top_p < 1:
        keep &= before < top_p * s.sum()
        keep[0] = True
    if min_p > 0:
        keep &= s >= min(min_p, 1.0)
    out = np.zeros_like(w)
    out[at[:n][keep]] = s[keep]
    return out


def sample(row, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, allowed=None):
    """(token, log of its share, distance of the random number from the nearest border between two tokens)"""
    row = clean(row, allowed)
    if row.max() == -np.inf:
        return -1, -np.inf, 1.0
    w = kept(row, float(temperature), int(top_k), float(top_p), float(min_p))
    c = np.cumsum(w)
    share = c / c[-1]
    token = min(int(np.searchsorted(c, float(uniform) * c[-1], side="right")), int(np.nonzero(w)[0][-1]))
    return token, np.log(w[token] / c[-1]), np.abs(share - float(uniform)).min()


def distill(z, teacher, index, teacher_lse, weight, temperature):
    """(loss, gradient of the loss, the sizes of the parts the gradient is the difference of)"""
    z = np.asarray(z, np.float64)
    n = z.size
    teacher = np.asarray(teacher, np.float64)
    valid = (index >= 0) & (index < n) & (teacher > -np.inf)
    if weight == 0 or not valid.any() or (z == -np.inf).all():
        return 0.0, np.zeros(n), np.zeros(n)
    t = teacher[valid] / temperature
    at = index[valid]
    logp = t - (log_sum_exp(t) if teacher_lse is None else float(teacher_lse))
    p = np.exp(logp)
    with np.errstate(invalid="ignore"):
        scaled = z / temperature
        m = scaled.max()
        logq = scaled - m - np.log(np.exp(scaled - m).sum())
    loss = sum(a * (b - logq[j]) for a, b, j in zip(p, logp, at) if a > 0)
    q = np.exp(logq)
    d = p.sum() * q
    parts = d.copy()
    np.subtract.at(d, at, p)
    np.add.at(parts, at, p)
    rest = 0.0 if teacher_lse is None else max(0.0, 1.0 - p.sum())
    others = np.ones(n, bool)
    others[at] = False
    left = log_sum_exp(logq[others]) if others.any() else -np.inf
    if rest > 0 and left > -np.inf:
        loss += rest * (np.log(rest) - left)
        d += rest * q
        d[others] -= q[others] * rest / np.exp(left)
        parts += rest * q
        parts[others] += q[others] * rest / np.exp(left)
    return weight * loss, weight / temperature * d, abs(weight / temperature) * parts
