"""CPU restatement of the training losses on rows of logits in 64 bits (numpy), one row at a time.

Test infrastructure only: nothing in the product path imports it.  The operators are defined in
include/mvsd.h (row_loss, loss_gradient); the reference has none.

Every gradient comes with a scale: the sum of the magnitudes of the terms that it is formed from, which
a relative error of the terms is measured against."""

from __future__ import annotations

import numpy as np

NINF = -np.inf


def log_softmax(x, T=1.0) -> np.ndarray:
    """NaN throughout for a row with a NaN or +inf, or of -inf alone."""
    y = np.asarray(x, np.float64) / T
    top = y.max()
    if not np.isfinite(top):
        return np.full(y.shape, np.nan)
    y = y - top
    others = np.exp(y)
    others[int(np.argmax(y))] = 0.0  # its 1 would take the digits of the rest
    return y - np.log1p(others.sum())


def entropy_of(logp) -> float:
    p = np.exp(logp)
    return float(-(p[p > 0] * logp[p > 0]).sum() if not np.isnan(logp).any() else np.nan)


def token_row(x, token: int, T=1.0):
    """(lp, entropy, logp) of a row; lp is NaN for a token that is none."""
    logp = log_softmax(x, T)
    H = entropy_of(logp)
    if token >= len(logp):
        return np.nan, np.nan, np.full(logp.shape, np.nan)
    return float(logp[token]), H, logp


def token_gradient(logp, token: int, g: float, gH: float, T=1.0):
    """d(g lp + gH H)/dx and its scale."""
    V = len(logp)
    if np.isnan(logp).any():
        return np.full(V, np.nan), np.zeros(V)
    p, H = np.exp(logp), entropy_of(logp)
    live = p > 0
    grad = -g * p
    grad[token] = g * -np.expm1(logp[token])
    scale = abs(g) * p
    scale[token] = abs(grad[token])
    if gH:
        grad[live] -= gH * p[live] * (logp[live] + H)
        scale[live] += abs(gH) * p[live] * (np.abs(logp[live]) + H + 1)
    return grad / T, scale / T


def first_places(ids) -> np.ndarray:
    """Which entries count."""
    seen, use = set(), []
    for i in ids:
        use.append(int(i) >= 0 and int(i) not in seen)
        seen.add(int(i))
    return np.array(use, bool)


def distill_row(x, ids, teacher, divergence="forward", tail=True, T=1.0):
    """(loss, gradient, scale of the loss, scale of the gradient); None for a row without an entry."""
    V = len(x)
    use = first_places(ids)
    if not use.any():
        return None
    ids, v = np.asarray(ids, np.int64)[use], np.asarray(teacher, np.float64)[use]
    if (ids >= V).any():
        return np.nan, np.full(V, np.nan), 0.0, np.zeros(V)
    logp = log_softmax(x, T)
    rest = np.ones(V, bool)
    rest[ids] = False
    lp = logp[ids]
    outcome = np.full(V, len(ids))
    outcome[ids] = np.arange(len(ids))
    if tail and rest.any():
        top = logp[rest].max()
        lt = NINF if top == NINF else top + np.log(np.exp(logp[rest] - top).sum())
        qt = max(1.0 - np.exp(v).sum(), 2.0 ** -24)
        logq, lp = np.append(v, np.log(qt)), np.append(lp, lt)
    elif tail:
        logq = v
    else:
        logq = log_softmax(v, T)
        lp, logq = np.append(lp, NINF), np.append(logq, NINF)  # the rest is no outcome
    q, p = np.exp(logq), np.exp(lp)
    with np.errstate(invalid="ignore", divide="ignore"):
        if divergence == "forward":
            terms = np.where(q > 0, q * (logq - lp), 0.0)
            D = np.where(p > 0, -q / p, 0.0)
            pD = -q
        elif divergence == "reverse":
            terms = np.where(p > 0, p * (lp - logq), 0.0)
            D = np.where(p > 0, lp - logq, 0.0)
            pD = terms
        else:
            m = np.log((p + q) / 2)
            terms = (np.where(q > 0, q * (logq - m), 0.0) + np.where(p > 0, p * (lp - m), 0.0)) / 2
            D = np.where(p > 0, lp - m, 0.0) / 2
            pD = np.where(p > 0, p * (lp - m), 0.0) / 2
    if not tail:
        terms, D, pD = terms[:-1], np.append(D[:-1], 0.0), pD[:-1]
    pD = pD.copy()
    mean = pD.sum()
    P = np.exp(logp)
    if len(D) == len(ids):  # no rest
        D = np.append(D, 0.0)
    grad = P * (D[outcome] - mean)
    grad[ids] = pD[: len(ids)] - P[ids] * mean
    scale = P * (np.abs(D[outcome]) + np.abs(pD).sum())
    scale[ids] = np.abs(pD[: len(ids)]) + P[ids] * np.abs(pD).sum()
    if divergence != "forward":  # errors of the log-probabilities are absolute
        scale += P
        if len(lp) > len(ids):
            scale += P * 2
    finite = np.abs(lp[np.isfinite(lp)])
    size = (q + p).sum() * (1 + np.abs(terms).sum()) + (finite.max() if finite.size else 0.0) * 0.1
    return float(terms.sum()), grad / T, float(size), scale / T


def policy_value(lp, H, old, advantage, ref, low, high, kl_coef, entropy_coef):
    """(loss, dloss/dlp, kl, scale)."""
    r = np.exp(lp - old) if old is not None else (1.0 if lp == lp else np.nan)
    lo, hi = float(np.float32(1.0 - low)), float(np.float32(1.0 + high))
    free, bound = r * advantage, min(max(r, lo), hi) * advantage
    clipped = free > bound
    loss, c = (-bound, 0.0) if clipped else (-free, -free)
    kl, scale = 0.0, abs(free) + abs(bound)
    if ref is not None:
        d = ref - lp
        kl = np.expm1(d) - d
        loss, c = loss + kl_coef * kl, c - kl_coef * np.expm1(d)
        scale += kl_coef * (np.exp(d) + abs(d) + 1)
    if entropy_coef:
        loss -= entropy_coef * H
        scale += entropy_coef * (H + 1)
    return loss, c, kl, scale


def pair_value(m, kind, beta, margin, smoothing):
    """(loss, dloss/dm)."""
    h = beta * m - margin
    if kind == "sigmoid":
        good, bad = np.logaddexp(0, -h), np.logaddexp(0, h)
        return ((1 - smoothing) * good + smoothing * bad,
                beta * (smoothing / (1 + np.exp(-h)) - (1 - smoothing) / (1 + np.exp(h))))
    if kind == "hinge":
        return max(0.0, 1 - h), -beta if h < 1 else 0.0
    off = m - margin - 1 / (2 * beta)
    return off * off, 2 * off


def mean_factor(weights, reduction) -> np.ndarray:
    """What the rows' losses are multiplied by; a row that is left out has weight 0."""
    w = np.asarray(weights, np.float64)
    if reduction != "mean":
        return w
    return w / w.sum() if w.sum() != 0 else np.zeros_like(w)
