"""Sampling one row at a time in 64 bits on the host: the definition that sample_tokens is checked against."""
from __future__ import annotations

import numpy as np


def token(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """``logits``: one row as float64 numpy values (exact images of the tensor's). Settings are taken as the
    float32 numbers they are for the operator."""
    x = np.where(np.isnan(logits), -np.inf, logits)
    T, p, m, u = (np.float64(np.float32(v)) for v in (temperature, top_p, min_p, u))
    top = x.max()
    if top == -np.inf:
        return -1
    if not T > 0:
        return int(np.flatnonzero(x == top)[0])
    order = np.argsort(-x, kind="stable")
    if 0 < top_k < len(x):
        order = order[:top_k]
    with np.errstate(invalid="ignore", over="ignore"):
        z = np.where(x[order] == top, 0.0, (x[order] - top) / T)
    w = np.where(x[order] == -np.inf, 0.0, np.exp(z))
    run = np.cumsum(w)
    stay = np.ones(len(order), dtype=bool)
    if p < 1:
        stay = run - w < p * run[-1]
        stay[0] = True
    if m > 0:
        stay &= w >= min(m, 1.0)
    weight = np.zeros(len(x))
    weight[order[stay]] = w[stay]
    run = np.cumsum(weight)
    above = np.flatnonzero(run > u * run[-1]) if u >= 0 else np.flatnonzero(weight > 0)
    last = np.flatnonzero(weight > 0)[-1]
    return int(min(above[0], last)) if len(above) else int(last)


def tokens(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """A batch: ``logits`` a CPU tensor [B, V], settings numbers or CPU tensors [B]."""
    x = logits.double().numpy()
    at = lambda v, b: float(v[b]) if hasattr(v, "shape") else v  # noqa: E731
    return [token(x[b], at(u, b), at(temperature, b), int(at(top_k, b)), at(top_p, b), at(min_p, b)) for b in range(x.shape[0])]
