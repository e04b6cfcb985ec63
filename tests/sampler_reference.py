"""Sampling restated in 64 bits, a row at a time."""
import math

import numpy as np


def draw(x, u, t=1.0, k=0, p=1.0, m=0.0):
    """(token, probability, kept) of one row of logits."""
    x = np.asarray(x, np.float64)
    x = np.where(np.isnan(x), -np.inf, x) + 0.0
    n = len(x)
    if x.max() == -np.inf:
        return -1, 0.0, 0
    if not t > 0:
        return int(np.argmax(x)), 1.0, 1
    if x.max() == np.inf:
        w = (x == np.inf).astype(np.float64)
    else:
        w = np.exp((x - x.max()) / t)
        w[x == -np.inf] = 0
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if 0 < k < n:
        order = order[:k]
    if p < 1:
        mass = np.cumsum(w[order])
        order = order[:max(1, int(np.searchsorted(mass, max(p, 0.0) * mass[-1], side="left")) + 1)]
    if m > 0:
        order = order[w[order] >= min(m, 1.0)]
    keep = np.sort(order)
    mass = np.cumsum(w[keep])
    u = min(max(u, 0.0), 1 - 2.0 ** -24) if not math.isnan(u) else 0.0
    i = min(int(np.searchsorted(mass, u * mass[-1], side="right")), len(keep) - 1)
    return int(keep[i]), float(w[keep[i]] / mass[-1]), len(keep)
