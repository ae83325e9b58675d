"""8-bit key / value cache and attention over it, restated in numpy (Float64 where values are compared, Float32 where the
definition rounds: scales and codes are Float32 arithmetic).  NNlib.jl has no counterpart; the definition is that of
``include/nnlib_b200.h``.

Arrays have the library's shapes: codes ``(d*H, page, pages)``, scales ``(H, pages)``, tokens ``(d*H, L, B)``.  Codes are
held as the numbers they are (Float32), whatever their type."""
from __future__ import annotations

import numpy as np
import torch

F32 = np.float32
TINY = F32(2.0 ** -126)


def to_e4m3(x: np.ndarray) -> np.ndarray:
    """To the nearest E4M3 number, ties to even, beyond 448 to 448."""
    t = torch.from_numpy(np.clip(np.ascontiguousarray(x, dtype=F32), -448, 448))
    return t.to(torch.float8_e4m3fn).float().numpy()


def block_scale(amax, code: str):
    if not np.isfinite(amax):
        return F32(np.nan)
    if code == "int8":
        s = F32(F32(amax) * (F32(1) / F32(127)))
    else:
        m, e = np.frexp(F32(amax))
        s = F32(np.ldexp(1.0, int(e) - 9 + int(m > 0.875)))
    return s if amax > 0 and s >= TINY else F32(0)


def to_codes(x, inv, code: str):
    t = np.zeros_like(x, dtype=F32) if inv == 0 else (np.asarray(x, F32) * F32(inv)).astype(F32)
    return np.rint(np.clip(t, -127, 127)).astype(F32) + F32(0) if code == "int8" else to_e4m3(t)


def pages_of(table, rows, pages, b, p):
    n = int(table[p, b]) if table is not None else rows * b + p
    return n if 0 <= n < pages else -1


def write(codes, scale, x, start, code: str, *, count=None, table=None):
    """Writes tokens ``x`` into ``codes`` and ``scale`` in place."""
    E, T, P = codes.shape
    H = scale.shape[0]
    d, (_, L, B) = E // H, x.shape
    rows = table.shape[0] if table is not None else P // B
    for b in range(B):
        s0 = int(start[b])
        end = s0 + (L if count is None else min(max(int(count[b]), 0), L))
        if s0 < 0:
            continue
        for p in range(s0 // T, rows):
            lo, hi = max(s0, p * T), min(end, (p + 1) * T)
            if lo >= hi:
                continue
            page = pages_of(table, rows, P, b, p)
            if page < 0:
                continue
            fill = lo - p * T
            for h in range(H):
                rng = slice(h * d, (h + 1) * d)
                new = x[rng, lo - s0:hi - s0, b].astype(F32)
                amax = np.abs(new).max() if np.isfinite(new).all() else np.inf
                asked = block_scale(amax, code)
                old = scale[h, page] if fill else F32(0)
                s = F32(np.nan) if np.isnan(old) or np.isnan(asked) else max(old, asked)
                inv = F32(1) / s if s > 0 else F32(0)
                if fill and s > old:
                    f = F32(old / s)
                    codes[rng, :fill, page] = to_codes(codes[rng, :fill, page], f, code)
                codes[rng, fill:fill + hi - lo, page] = to_codes(new, inv, code)
                scale[h, page] = s


def read(codes, scale, length, start, B, *, lens=None, table=None):
    """Float32 values, ``(d*H, length, B)``, unrounded."""
    E, T, P = codes.shape
    H = scale.shape[0]
    rows = table.shape[0] if table is not None else (P // B if B else 0)
    out = np.zeros((E, length, B), F32)
    for b in range(B):
        for l in range(length):
            pos = int(start[b]) + l
            if pos < 0 or pos >= rows * T or (lens is not None and pos >= lens[b]):
                continue
            page = pages_of(table, rows, P, b, pos // T)
            with np.errstate(invalid="ignore"):
                out[:, l, b] = np.nan if page < 0 else codes[:, pos % T, page] * np.repeat(scale[:, page], E // H)
    return out


def attention(q, kc, vc, ks, vs, lens, nheads, *, start=None, causal=True, scale=None, table=None):
    """``(x, lse, size, grid)`` in Float64, the last two what errors are measured by: ``size`` is the sum of weights times the
    values' magnitudes (relative errors of the weights), ``grid`` the largest product of a weight and its page's value scale
    times the sum of the codes' magnitudes (errors of such products relative to the largest one)."""
    E, T, P = kc.shape
    H = ks.shape[0]
    d, G = E // H, nheads // H
    _, L, B = q.shape
    rows = table.shape[0] if table is not None else (P // B if B else 0)
    scale = 1.0 / np.sqrt(d) if scale is None else scale
    x, lse = np.full(q.shape, np.nan), np.full((L, nheads, B), -np.inf)
    size, grid = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(B):
        n = int(min(max(int(lens[b]), 0), rows * T))
        s0 = int(start[b]) if start is not None else n - L
        at = np.zeros(B, int)
        vscale = np.array([vs[:, max(pages_of(table, rows, P, b, j // T), 0)] for j in range(n)], np.float64).reshape(n, H)
        k, v = (read(c, s, n, at, B, table=table)[:, :, b].astype(np.float64) if n else np.zeros((E, 0)) for c, s in ((kc, ks), (vc, vs)))
        seen = np.arange(n)[None] <= (s0 + np.arange(L)[:, None] if causal else np.full((L, 1), n))
        some = seen.any(1)
        for h in range(nheads):
            r, c = slice(h * d, (h + 1) * d), slice(h // G * d, (h // G + 1) * d)
            with np.errstate(invalid="ignore"):
                t = np.where(seen, scale * (q[r, :, b].T.astype(np.float64) @ k[c]), -np.inf)
            bad = (np.isnan(t) | (seen & np.isnan(v[c]).any(0)[None])).any(1)       # a NaN among what the query sees
            ok = some & ~bad
            lse[bad, h, b] = np.nan
            if not ok.any():
                continue
            t = t[ok]
            top = t.max(1, keepdims=True)
            w = np.exp(t - top)
            sums = w.sum(1, keepdims=True)
            lse[ok, h, b] = (top + np.log(sums))[:, 0]
            w /= sums
            val = np.where(np.isnan(v[c]), 0.0, v[c])                              # (weight 0 in these rows)
            s = vscale[:, h // G]
            codes = np.abs(val) / np.where(s > 0, s, 1)
            x[r, ok, b], size[r, ok, b] = val @ w.T, np.abs(val) @ w.T
            grid[r, ok, b] = (w * np.where(np.isnan(s), 0, s)).max(1) * (codes @ seen[ok].T)
    return x, lse, size, grid
