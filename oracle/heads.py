"""Heads between the projections of an attention block, in 64 bits (NumPy): rotation by positions, head norms, attention.

The reference has no counterpart (it shards the projections by heads, nn/linear_ag.py:46-60, and leaves the rest to its user);
these are the operators' definitions, written out.  Heads are [batch, tokens, heads, head_dim].
"""

import numpy as np


def members(dim, pairs, interleaved):
    """The two members of every pair."""
    p = np.arange(pairs)
    return (2 * p, 2 * p + 1) if interleaved else (p, p + pairs)


def rotate(x, frequencies, positions, interleaved=False, amplitude=1.0, inverse=False):
    """x turned by ``positions`` [tokens] or [batch, tokens]."""
    x = np.asarray(x, np.float64)
    angle = np.broadcast_to(np.asarray(positions, np.float64), x.shape[:2])[:, :, None, None] * np.asarray(frequencies, np.float64)
    c, s = amplitude * np.cos(angle), amplitude * np.sin(angle) * (-1 if inverse else 1)
    a, b = members(x.shape[-1], len(frequencies), interleaved)
    y = x.copy()
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def pair_sum(x, pairs, interleaved, amplitude=1.0):
    """|x| + |x'| with the other member of the pair, times the amplitude: what a rotation's rounding errors scale with."""
    x = np.abs(np.asarray(x, np.float64))
    a, b = members(x.shape[-1], pairs, interleaved)
    y = x.copy()
    y[..., a] = y[..., b] = abs(amplitude) * (x[..., a] + x[..., b])
    return y


def head_norm(x, eps):
    """``(xhat, rstd)``."""
    x = np.asarray(x, np.float64)
    rstd = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    return x * rstd, rstd


def head_norm_rotate_backward(dy, x, weight, eps, frequencies, positions, interleaved=False, amplitude=1.0):
    """``(dx, dweight)``."""
    xhat, rstd = head_norm(x, eps)
    g = rotate(dy, frequencies, positions, interleaved, amplitude, inverse=True)
    wg = g * np.asarray(weight, np.float64)
    return rstd * (wg - xhat * (wg * xhat).mean(-1, keepdims=True)), (g * xhat).sum((0, 1, 2))


def visible(tokens, keys, length, causal):
    """[tokens, keys]: the keys that each query sees."""
    see = np.broadcast_to(np.arange(keys) < length, (tokens, keys))
    if causal:
        see = see & (np.arange(keys) <= np.arange(tokens)[:, None] + keys - tokens)
    return see


def attention(q, k, v, lengths=None, causal=False, scale=None, dy=None):
    """``(out, lse)``, or with ``dy`` ``(out, lse, dq, dk, dv)``; queries that see no key give zeros (lse -inf) and take no gradient."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    (batch, tokens, heads, dim), keys, kv_heads = q.shape, k.shape[1], k.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    out, lse = np.zeros_like(q), np.full((batch, tokens, heads), -np.inf)
    dq, dk, dv = np.zeros_like(q), np.zeros_like(k), np.zeros_like(v)
    for b in range(batch):
        see = visible(tokens, keys, keys if lengths is None else lengths[b], causal)
        some = see.any(-1)
        for h in range(heads):
            j = h * kv_heads // heads
            seen = see.any(0)
            kb, vb = np.where(seen[:, None], k[b, :, j], 0), np.where(seen[:, None], v[b, :, j], 0)
            s = np.where(see, scale * q[b, :, h] @ kb.T, -np.inf)
            top = np.where(some, s.max(-1, initial=-np.inf), 0)
            p = np.exp(s - top[:, None])
            total = p.sum(-1)
            p = p / np.where(some, total, 1)[:, None]
            out[b, :, h] = p @ vb
            lse[b, some, h] = (top + np.log(np.where(some, total, 1)))[some]
            if dy is not None:
                g = np.asarray(dy[b, :, h], np.float64)
                ds = p * (g @ vb.T - (g * out[b, :, h]).sum(-1)[:, None]) * scale
                dq[b, :, h] = ds @ kb
                dk[b, :, j] += ds.T @ q[b, :, h]
                dv[b, :, j] += p.T @ g
    return (out, lse) if dy is None else (out, lse, dq, dk, dv)
