"""Sampling by temperature, top-k, top-p and min-p in 64 bits, for the tests."""
import math

import numpy as np


def single(v):
    return float(np.float32(v))


def kept_weights(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Weights of the tokens that stay, 0 for the others; None for a row that takes
    its most probable token."""
    x = x.astype(np.float64)
    temperature, top_p, min_p = single(temperature), single(top_p), single(min_p)
    some = ~np.isnan(x)
    if not some.any() or not temperature >= 2.0 ** -16 or x[some].max() == -math.inf:
        return None
    top = x[some].max()
    weight = np.zeros(len(x))
    if top == math.inf:
        weight[x == top] = 1.0
    elif temperature == math.inf:
        weight[some & (x > -math.inf)] = 1.0
    else:
        weight[some] = np.exp((x[some] - top) / temperature)
    weight[weight < 2.0 ** -44] = 0.0  # never drawn
    rank = np.lexsort((np.arange(len(x)), -np.where(some, x, -math.inf)))
    rank = rank[weight[rank] > 0]
    if top_k > 0:
        rank = rank[:top_k]
    if top_p < 1:
        sums = np.concatenate([[0.0], np.cumsum(weight[rank])])
        rank = rank[:max(1, np.count_nonzero(sums[:-1] < top_p * sums[-1]))]
    if min_p > 0:
        rank = rank[weight[rank] >= min(min_p, 1.0)]
    out = np.zeros(len(x))
    out[rank] = weight[rank]
    return out


def draw(x, u, **settings):
    """(token, probability)."""
    weight = kept_weights(x, **settings)
    if weight is None:
        some = ~np.isnan(x)
        if not some.any():
            return -1, math.nan
        token = int(np.flatnonzero(some & (x == x[some].max()))[0])
        return token, 1.0 if not settings.get("temperature", 1.0) >= 2.0 ** -16 else math.nan
    sums = np.cumsum(weight)
    u = min(max(single(u), 0.0), 1.0) if u == u else 0.0
    token = int(np.searchsorted(sums, u * sums[-1], side="right"))
    token = min(token, int(np.flatnonzero(weight)[-1]))
    return token, weight[token] / sums[-1]
