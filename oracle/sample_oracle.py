"""The choice of a token by its definition (CPU, 64 bits and more).  Test infrastructure only."""
from __future__ import annotations

import math

import numpy as np


def kept(row, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(indices of what is kept, in their order, weights, whether the cut of top_p or min_p is too close to call): row in float64, not-a-numbers
    minus infinity; None where there is nothing.  Too close: within 2^-40 of the weight on either side, which is far above what a
    weight of 2^-44 and the sum of 10^4 of them may be off by, next to a cut at a border."""
    row = np.where(np.isnan(row), -np.inf, row)
    top = row.max()
    if top == -np.inf:
        return None
    if not temperature > 0:
        return np.array([int(np.argmax(row))]), np.ones(1, dtype=np.longdouble), False
    with np.errstate(all="ignore"):
        w = (row == top) * np.longdouble(1) if top == np.inf else np.exp(((row - top) / np.float64(temperature)).astype(np.longdouble))
    w[row == -np.inf] = 0
    order = np.lexsort((np.arange(len(row)), -row))
    close = False
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        sums = np.cumsum(w[order])
        need = np.longdouble(top_p) * sums[-1] if top_p > 0 else np.longdouble(0)
        n = 1 + int((sums[:-1] < need).sum())
        # (sums that are exact are no matter: whole numbers of largest weights)
        near = np.abs(sums[:-1] - need) < need * 2.0 ** -40
        close = bool((near & (sums[:-1] != np.floor(sums[:-1]))).any())
        order = order[:n]
    least = min(max(min_p, 0.0), 1.0)
    close = close or bool((np.abs(w[order] - least) < 2.0 ** -40).any() and 0 < least < 1)
    order = np.sort(order[w[order] >= least])
    return order, w[order], close


def draw(row, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(tokens that the draw may give, log of the probability of each): one token, or two where u meets a border to within 2^-40
    of the whole weight; None where a cut is too close to call."""
    k = kept(row, temperature, top_k, top_p, min_p)
    if k is None:
        return [-1], [-math.inf]
    index, w, close = k
    if close:
        return None
    sums = np.cumsum(w)
    u = min(max(u, 0.0), 1.0) if u == u else 0.0
    target = np.longdouble(u) * sums[-1]
    exact = target == np.floor(target) and (sums == np.floor(sums)).all()
    slack = 0 if exact else sums[-1] * np.longdouble(2.0 ** -40)
    j = [min(int(np.searchsorted(sums, t, side="right")), len(index) - 1) for t in (target - slack, target + slack)]
    tokens, logs = [], []
    for i in range(j[0], j[1] + 1):
        while i == len(index) - 1 and i > 0 and w[i] == 0:
            i -= 1
        if w[i] > 0:
            tokens.append(int(index[i]))
            logs.append(float(np.log(w[i] / sums[-1])))
    return tokens, logs
