"""RMS norm and rotation of heads and their pullback in Float64 numpy (definition: ``include/nnlib_b200.h``,
``nnlib_b200_norm_rope``; NNlib.jl has no counterpart).  Arrays are ``(heads * d, L, B)``."""
from __future__ import annotations

import numpy as np


def _pairs(d, rot, interleaved):
    p = np.arange(rot // 2)
    return (2 * p, 2 * p + 1) if interleaved else (p, p + rot // 2)


def rotate(n, pos, freqs, interleaved, back=False):
    """``n``: (d, heads, L, B); ``pos``: (L, B)."""
    a, b = _pairs(n.shape[0], 2 * len(freqs), interleaved)
    ang = (pos[None] * np.asarray(freqs, np.float64)[:, None, None])[:, None]
    c, s = np.cos(ang), np.sin(ang) * (-1 if back else 1)
    y = n.copy()
    y[a], y[b] = n[a] * c - n[b] * s, n[a] * s + n[b] * c
    return y


def heads(x, d):
    E, L, B = x.shape
    return np.asarray(x, np.float64).reshape(E // d, d, L, B).transpose(1, 0, 2, 3)


def unheads(y):
    d, H, L, B = y.shape
    return y.transpose(1, 0, 2, 3).reshape(H * d, L, B)


def norm_rope(x, g, pos, freqs, eps, interleaved):
    g = np.asarray(g, np.float64)
    x = heads(x, len(g))
    r = 1 / np.sqrt((x * x).mean(0) + eps)
    return unheads(rotate(x * r * g[:, None, None, None], pos, freqs, interleaved))


def pullback(x, g, pos, freqs, eps, interleaved, dy):
    """``(dx, dg)``."""
    g = np.asarray(g, np.float64)
    d = len(g)
    x, u = heads(x, d), rotate(heads(dy, d), pos, freqs, interleaved, back=True)
    r = 1 / np.sqrt((x * x).mean(0) + eps)
    w = u * g[:, None, None, None]
    dx = r * (w - x * r * r * (w * x).mean(0))
    return unheads(dx), (u * x * r).sum((1, 2, 3))
