"""Rotary positions and the draw of tokens in 64 bits, from their definitions."""
from __future__ import annotations

import numpy as np


def rope(x, positions, frequencies, *, magnitude=1.0, interleaved=False, inverse=False):
    """-> (y float64 [T, H, D], largest |angle| of each row [T], |a| + |b| of each value's pair [T, H, D] (0 where it passes))."""
    x = np.asarray(x, np.float64)
    R = 2 * len(frequencies)
    t = np.asarray(positions, np.float64)[:, None] * np.asarray(frequencies, np.float64)
    c, s = (magnitude * f(t)[:, None] for f in (np.cos, np.sin))
    if inverse:
        s = -s
    y, pair = x.copy(), np.zeros_like(x)
    at = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    a, b = x[..., at[0]], x[..., at[1]]
    y[..., at[0]], y[..., at[1]] = a * c - b * s, b * c + a * s
    pair[..., at[0]] = pair[..., at[1]] = np.abs(a) + np.abs(b)
    return y, np.abs(t).max(1) if t.size else np.zeros(len(x)), pair


def positions(lengths, counts):
    return np.concatenate([np.arange(int(L) - n, int(L)) for L, n in zip(lengths, counts)] or [np.zeros(0)]).astype(np.int64)


def kept(x, temperature, top_k=0, top_p=1.0, min_p=0.0):
    """One row's -> (weights float64 [V], 0 where a token is not kept; how near, relative to the largest weight, a top_p or min_p
    border lies to a sum or weight that decides)."""
    x = np.asarray(x, np.float64).copy()
    x[np.isnan(x)] = -np.inf
    V, near = len(x), np.inf
    order = np.lexsort((np.arange(V), -x))  # descending, the lower index first
    top = x[order[0]]
    if top == -np.inf:
        return np.zeros(V), near
    if not temperature > 0:
        w = np.zeros(V)
        w[order[0]] = 1.0
        return w, near
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.exp((x - top) / temperature)
    w[x == top] = 1.0
    w[np.isnan(w) | (x == -np.inf)] = 0.0
    n = V if top_k <= 0 else min(V, top_k)
    ws = w[order[:n]]
    if top_p < 1:
        run = np.cumsum(ws)
        reach = run >= top_p * run[-1]
        n = int(np.argmax(reach)) + 1
        if len(set(ws[ws > 0])) > 1:  # sums of equal weights are exact
            near = min(near, np.abs(run - top_p * run[-1]).min())
    if min_p > 0:
        m = min(min_p, 1.0)
        if m < 1:
            near = min(near, np.abs(ws - m).min())
        n = min(n, max(1, int((ws >= m).sum())))
    w[order[n:]] = 0.0
    return w, near


def tokens(w, u, slack):
    """The tokens that the number u may draw from the weights w when sums and weights are off by ``slack``."""
    run = np.cumsum(w)
    t = u * run[-1]
    return [int(i) for i in np.nonzero((w > 0) & (run > t - slack) & (run - w <= t + slack))[0]]
