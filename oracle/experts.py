"""An experts' feed-forward block in 64 bits (NumPy): root-mean-square norm, rows in 8 bits, tokens by their experts and back, the experts' products.

The reference has no counterpart; these are the operators' definitions, written out.
"""

import numpy as np

E4M3_MAX = 448.0


def rms_norm(h, weight=None, eps=1e-6):
    """``(y, xhat, rstd)`` of the rows of h."""
    h = np.asarray(h, np.float64)
    rstd = 1 / np.sqrt((h * h).mean(-1, keepdims=True) + eps)
    xhat = h * rstd
    return xhat if weight is None else xhat * np.asarray(weight, np.float64), xhat, rstd


def rms_norm_backward(dy, h, weight=None, dh=None, eps=1e-6):
    """``(dx, dweight)``."""
    _, xhat, rstd = rms_norm(h, None, eps)
    dy = np.asarray(dy, np.float64)
    g = dy if weight is None else dy * np.asarray(weight, np.float64)
    dx = rstd * (g - xhat * (g * xhat).mean(-1, keepdims=True))
    return dx if dh is None else dx + np.asarray(dh, np.float64), (dy * xhat).reshape(-1, dy.shape[-1]).sum(0)


def row_scales(y):
    return np.maximum(np.abs(np.asarray(y, np.float64)).max(-1) / E4M3_MAX, 2.0 ** -126)


def plan(ids, low, high):
    """``(place, offsets)`` of the choices [tokens, chosen] among the experts low .. high - 1."""
    ids = np.asarray(ids)
    flat = ids.reshape(-1)
    key = np.where((flat >= low) & (flat < high), flat - low, high - low)
    order = np.argsort(key, kind="stable")
    place = np.empty(len(flat), np.int64)
    place[order] = np.arange(len(flat))
    counts = np.bincount(key, minlength=high - low + 1)[:high - low]
    return place.reshape(ids.shape), np.concatenate([[0], np.cumsum(counts)])


def sort(x, place, held):
    """Rows in the order of their experts, zeros behind the last held one."""
    x = np.asarray(x)
    out = np.zeros((place.size,) + x.shape[1:], x.dtype)
    for t in range(place.shape[0]):
        for p in place[t]:
            if p < held:
                out[p] = x[t]
    return out


def combine(y, place, held, weights=None):
    y = np.asarray(y, np.float64)
    out = np.zeros((place.shape[0], y.shape[1]))
    for t in range(place.shape[0]):
        for j, p in enumerate(place[t]):
            if p < held:
                out[t] += y[p] * (1.0 if weights is None else float(weights[t, j]))
    return out


def combine_backward(dout, y, place, held, weights):
    """``(dy, dweights)``."""
    dout, y = np.asarray(dout, np.float64), np.asarray(y, np.float64)
    dy, dw = np.zeros((place.size, dout.shape[1])), np.zeros(place.shape)
    for t in range(place.shape[0]):
        for j, p in enumerate(place[t]):
            if p < held:
                dy[p] = float(weights[t, j]) * dout[t]
                dw[t, j] = dout[t] @ y[p]
    return dy, dw


def product(x, w, offsets, dy=None):
    """``y``, or with ``dy`` ``(y, dx, dw)``."""
    x, w = np.asarray(x, np.float64), np.asarray(w, np.float64)
    y = np.zeros((x.shape[0], w.shape[1]))
    dx, dw = np.zeros_like(x), np.zeros_like(w)
    for e in range(w.shape[0]):
        rows = slice(int(offsets[e]), int(offsets[e + 1]))
        y[rows] = x[rows] @ w[e].T
        if dy is not None:
            g = np.asarray(dy, np.float64)[rows]
            dx[rows], dw[e] = g @ w[e], g.T @ x[rows]
    return y if dy is None else (y, dx, dw)
