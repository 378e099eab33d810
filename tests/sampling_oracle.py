"""The sampler's rule in exact whole numbers and float64, from the weights' definition.

`interval` gives, for one row, every kept token's interval of [0, 1) in real arithmetic; a kernel's
token is right if u lies in its interval widened by what float32 weights may move its ends.
"""
import math

import numpy as np


def row(x, temperature, top_k, top_p, min_p):
    """(kept indices ascending, their float64 probabilities among the kept, log Z, z) of one row."""
    x = np.asarray(x, np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if top == -np.inf:
        return np.array([], int), np.array([]), -math.inf, x
    T = temperature if temperature > 0 else 1.0
    if top == np.inf:
        z = np.where(x == np.inf, 0.0, -np.inf)
    else:
        z = (x - top) / T
    e = np.exp(z)
    order = np.lexsort((np.arange(len(x)), -x))
    keep = np.isfinite(z[order])
    ranks = np.arange(len(x))
    if not temperature > 0:
        keep &= ranks == 0
    if 0 < top_k < len(x):
        keep &= ranks < top_k
    w = np.where(keep, e[order], 0.0)
    before = np.cumsum(w) - w
    if top_p < 1:
        keep &= (before < top_p * w.sum()) | (ranks == 0)
    keep &= (e[order] >= min_p) | (ranks == 0)
    idx = np.sort(order[keep])
    return idx, e[idx] / e[idx].sum(), math.log(e.sum()), z
