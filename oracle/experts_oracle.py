"""Router, products of ragged groups of columns, weighted sums and low-rank adapters from their definitions, in Float64 and
plain loops (test infrastructure)."""
import numpy as np


def softmax(x):
    """Over a vector, with the reference's slow branch: equal shares for +Inf."""
    m = x.max() if x.size else 0.0
    if np.isnan(x).any() or m == -np.inf:
        return np.full_like(x, np.nan)
    e = (x == np.inf).astype(np.float64) if m == np.inf else np.exp(x - m)
    return e / e.sum()


def route(logits, k, bias=None, mask=None, normalize=True):
    """logits (G, N).  -> weights (k, N), experts (k, N), offsets (G + 1), columns (k N), position (k, N)"""
    G, N = logits.shape
    weights, experts = np.zeros((k, N)), np.full((k, N), -1)
    for t in range(N):
        if mask is not None and not mask[t]:
            continue
        x = logits[:, t].astype(np.float64)
        score = logits[:, t].astype(np.float32)
        if bias is not None:
            score = score + bias.astype(np.float32)
        key = [(1 if np.isnan(s) else 0, 0.0 if np.isnan(s) else -float(s), e) for e, s in enumerate(score)]
        top = [e for _, _, e in sorted(key)[:k]]
        experts[:, t] = top
        weights[:, t] = softmax(x[top]) if normalize else softmax(x)[top]
    offsets, columns, position = np.zeros(G + 1, int), np.full(k * N, -1), np.full((k, N), -1)
    at = 0
    for e in range(G):
        for t in range(N):
            for j in range(k):
                if experts[j, t] == e:
                    columns[at], position[j, t] = t, at
                    at += 1
        offsets[e + 1] = at
    return weights, experts, offsets, columns, position


def route_back(logits, experts, dweights, normalize=True):
    """Gradient of the logits for a given choice: the Jacobian of the softmax, written out."""
    G, N = logits.shape
    out = np.zeros((G, N))
    for t in range(N):
        top = experts[:, t]
        if top[0] < 0:
            continue
        among = np.array(sorted(top)) if normalize else np.arange(G)
        p = softmax(logits[among, t].astype(np.float64))
        d = np.zeros(G)
        d[top] = dweights[:, t]
        d = d[among]
        out[among, t] = (np.diag(p) - np.outer(p, p)) @ d
    return out


def runs(offsets, n):
    o = np.clip(np.asarray(offsets, np.int64), 0, n)
    return [(int(o[g]), max(int(o[g]), int(o[g + 1]))) for g in range(len(o) - 1)]


def grouped(A, X, offsets, columns=None, rest=0.0):
    """A (M, K, G), X (K, N) -> (M, R); `rest` fills the columns in no run"""
    R = X.shape[1] if columns is None else len(columns)
    out = np.full((A.shape[0], R), rest)
    for g, (a, b) in enumerate(runs(offsets, R)):
        for i in range(a, b):
            c = i if columns is None else columns[i]
            out[:, i] = A[:, :, g] @ X[:, c] if 0 <= c < X.shape[1] else 0.0
    return out


def grouped_back(A, X, offsets, dC, columns=None):
    dA, dX = np.zeros(A.shape), np.zeros(X.shape)
    for g, (a, b) in enumerate(runs(offsets, dC.shape[1])):
        for i in range(a, b):
            c = i if columns is None else columns[i]
            if 0 <= c < X.shape[1]:
                dA[:, :, g] += np.outer(dC[:, i], X[:, c])
                dX[:, c] += A[:, :, g].T @ dC[:, i]
    return dA, dX


def combine(Y, position, weights):
    k, N = position.shape
    y = np.zeros((Y.shape[0], N))
    for t in range(N):
        for j in range(k):
            if 0 <= position[j, t] < Y.shape[1]:
                y[:, t] += weights[j, t] * Y[:, position[j, t]]
    return y


def combine_back(Y, position, weights, dy):
    k, N = position.shape
    dY, dw = np.zeros(Y.shape), np.zeros((k, N))
    for t in range(N):
        for j in range(k):
            p = position[j, t]
            if 0 <= p < Y.shape[1]:
                dY[:, p] += weights[j, t] * dy[:, t]
                dw[j, t] = dy[:, t] @ Y[:, p]
    return dY, dw


def adapters(W, X, A, B, ids, offsets, scale):
    """scale: one per pair"""
    y = W @ X
    for (a, b), i in zip(runs(offsets, X.shape[1]), ids):
        if 0 <= i < A.shape[2]:
            y[:, a:b] += scale[i] * (B[:, :, i] @ (A[:, :, i] @ X[:, a:b]))
    return y


def adapters_back(W, X, A, B, ids, offsets, scale, dY):
    dX, dA, dB = W.T @ dY, np.zeros(A.shape), np.zeros(B.shape)
    for (a, b), i in zip(runs(offsets, X.shape[1]), ids):
        if 0 <= i < A.shape[2]:
            x, d = X[:, a:b], dY[:, a:b]
            dX[:, a:b] += scale[i] * (A[:, :, i].T @ (B[:, :, i].T @ d))
            dA[:, :, i] += scale[i] * (B[:, :, i].T @ d) @ x.T
            dB[:, :, i] += scale[i] * d @ (A[:, :, i] @ x).T
    return dX, dA, dB
