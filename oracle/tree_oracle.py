"""Normalised and rotated heads, attention of drafted trees over a cache, and the accepted path, in float64 from their definitions.

Test infrastructure only.  Heads: y = R(pos) (w * x / sqrt(mean(x^2) + eps)).  Trees: parents[t] < t is the node that node t follows,
-1 the cached tokens; a node sees the cached tokens, its ancestors and itself.
"""
import numpy as np


def frequencies(rotary, theta=10000.0, scaling=1.0, inv_freq=None):
    if inv_freq is not None:
        return np.asarray(inv_freq, np.float32).astype(np.float64)
    return float(np.float32(theta)) ** (-2.0 * np.arange(rotary // 2) / rotary) / float(np.float32(scaling))


def rotate(x, pos, freq, mode, gain=1.0, back=False):
    """x (..., H, D) at positions pos (...): the first 2 * len(freq) elements of a head turned; back: the transposed rotation."""
    x = np.array(x, np.float64)
    n = len(freq)
    if mode == "none" or n == 0:
        return x
    a = np.asarray(pos, np.float64)[..., None] * freq
    c, s = np.cos(a)[..., None, :] * gain, np.sin(a)[..., None, :] * (-gain if back else gain)
    lo, hi = (slice(0, n), slice(n, 2 * n)) if mode == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    u, v = x[..., lo].copy(), x[..., hi].copy()
    x[..., lo], x[..., hi] = u * c - v * s, u * s + v * c
    return x


def norm(x, w, eps):
    x = np.asarray(x, np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    return y if w is None else y * np.asarray(w, np.float64)


def norm_rope(x, w, pos, freq, mode, eps=1e-6, gain=1.0):
    return rotate(norm(x, w, eps), pos, freq, mode, gain)


def norm_rope_grad(x, w, dy, pos, freq, mode, eps=1e-6, gain=1.0):
    """Gradients of sum(norm_rope * dy): of x, and of w summed over every other axis."""
    x = np.asarray(x, np.float64)
    g = rotate(dy, pos, freq, mode, gain, back=True)
    r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    dw = (g * x * r).reshape(-1, x.shape[-1]).sum(0)
    if w is not None:
        g = g * np.asarray(w, np.float64)
    return r * g - x * r ** 3 * (g * x).mean(-1, keepdims=True), dw


def ancestors(parents, n):
    """(n, n): whether node t sees node u; parents None is a chain."""
    seen = np.zeros((n, n), bool)
    for t in range(n):
        p = t - 1 if parents is None else int(parents[t])
        if p >= 0:
            seen[t] = seen[p]
        seen[t, t] = True
    return seen


def depths(parents, n):
    return ancestors(parents, n).sum(1) - 1


def tree_attention(q, k, v, n, parents, scale):
    """q (n, Hq, D) of one sequence, k and v (prefix + n, Hkv, D): out, and sum p |v| (what a relative error of the probabilities moves)."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    hq, hkv, prefix = q.shape[1], k.shape[1], k.shape[0] - n
    see = np.concatenate([np.ones((n, prefix), bool), ancestors(parents, n)], 1)
    out, size = np.zeros_like(q), np.zeros_like(q)
    for h in range(hq):
        kh, vh = k[:, h // (hq // hkv)], v[:, h // (hq // hkv)]
        for t in range(n):
            at = see[t]
            s = kh[at] @ q[t, h] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[t, h], size[t, h] = p @ vh[at], p @ np.abs(vh[at])
    return out, size
