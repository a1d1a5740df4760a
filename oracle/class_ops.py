"""Class / vocabulary operators in plain numpy, float64, one row at a time: the definitions that the kernels behind
``ser_amd.vocabulary`` are held to.  Written from the formulas; nothing here is shared with the product."""

from __future__ import annotations

import numpy as np


def sample_row(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, log softmax(x)[token]) for one row of scores (any float dtype) and one uniform number."""
    x = np.asarray(x, dtype=np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if top == -np.inf:
        return -1, -np.inf
    with np.errstate(invalid="ignore", over="ignore"):
        far = np.where(x == top, 0.0, x - top)
    log_all = np.log(np.exp(far).sum())
    if not (temperature > 0 and np.isfinite(temperature)):
        token = int(np.argmax(x))
        return token, far[token] - log_all
    w = np.exp(far / float(temperature))
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if top_k >= 1:
        order = order[: int(top_k)]
    if top_p < 1:
        before = np.concatenate([[0.0], np.cumsum(w[order])[:-1]])
        order = order[: max(1, int(np.count_nonzero(before < max(float(top_p), 0.0) * w[order].sum())))]
    if min_p > 0:
        order = order[w[order] >= min(float(min_p), 1.0)]
    order = np.sort(order)
    upto = np.cumsum(w[order])
    u = float(u) if u > 0 else 0.0
    at = int(np.searchsorted(upto, u * upto[-1], side="right"))
    if at >= len(order):
        at = int(np.flatnonzero(w[order])[-1])
    token = int(order[at])
    return token, far[token] - log_all


def teacher_softmax(index, teacher, n_classes, temperature):
    """float64 probabilities of one row's entries; None where no entry counts."""
    index, teacher = np.asarray(index, np.int64), np.asarray(teacher, np.float64)
    counts = (index >= 0) & (index < n_classes) & (teacher != -np.inf)
    if not counts.any():
        return None
    t = np.where(counts, teacher, -np.inf) / temperature
    e = np.exp(t - t.max())
    return e / e.sum()


def distill_row(x, index, teacher, temperature):
    """(loss, gradient) of one row."""
    x = np.asarray(x, dtype=np.float64)
    p = teacher_softmax(index, teacher, x.size, temperature)
    if p is None:
        return 0.0, np.zeros_like(x)
    if np.isnan(x).any() or (x == np.inf).any():
        return np.nan, np.full_like(x, np.nan)
    z = x / temperature
    top = z.max()
    if top == -np.inf:
        q, logq = np.zeros_like(x), np.full_like(x, -np.inf)
    else:
        with np.errstate(divide="ignore"):
            logq = (z - top) - np.log(np.exp(z - top).sum())
        q = np.exp(logq)
    loss, g = 0.0, temperature * q
    for i, pk in zip(np.asarray(index, np.int64), p):
        if pk > 0:
            loss += pk * (np.log(pk) - logq[i])
            g[i] -= temperature * pk
    return temperature**2 * loss, g


def embedding_gradient(grad, tokens, n_classes, scale):
    """(gradient, sum of |terms|, terms per row): float64."""
    grad, tokens = np.asarray(grad, np.float64), np.asarray(tokens, np.int64)
    out = np.zeros((n_classes, grad.shape[1]))
    size = np.zeros_like(out)
    real = (tokens >= 0) & (tokens < n_classes)
    np.add.at(out, tokens[real], grad[real] * scale)
    np.add.at(size, tokens[real], np.abs(grad[real] * scale))
    return out, size, np.bincount(tokens[real], minlength=n_classes)
