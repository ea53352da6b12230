"""Plain forms, in binary64 and row by row, of the operators between a policy and a batch (gx_sample, gx_embed)."""
import numpy as np


def sample_row(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """-> (action, log-probability) of one row by its definition; every argument a number read as binary64"""
    x = np.asarray(x, np.float64).copy()
    x[np.isnan(x)] = -np.inf
    n, m = len(x), x.max()
    if m == -np.inf:
        return -1, -np.inf
    u = min(max(u, 0.0), 1.0 - 2.0**-53) if u == u else 0.0
    order = np.argsort(-x, kind="stable")
    if not temperature > 0:
        return int(order[0]), 0.0
    k = n if top_k <= 0 else min(top_k, n)
    with np.errstate(invalid="ignore", over="ignore"):
        z = (x - m) / temperature
    z = np.where(x == m, 0.0, np.where((x == -np.inf) | (m == np.inf), -np.inf, z))
    w = np.exp(z)
    kept = np.zeros(n, bool)
    first = order[:k]
    kept[first] = True
    if top_p < 1:
        s = w[first].sum()
        ahead = np.concatenate([[0.0], np.cumsum(w[first])[:-1]])
        kept[first[1:]] = ahead[1:] < max(top_p, 0.0) * s
    if min_p > 0:
        kept &= w >= min(min_p, 1.0)
    w = np.where(kept, w, 0.0)
    c = np.cumsum(w)
    past = np.nonzero((c > u * c[-1]) & (w > 0))[0]
    action = int(past[0]) if len(past) else int(np.nonzero(w > 0)[0][-1])
    return action, float(z[action] - np.log(c[-1]))


def sample(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """all rows; a parameter is a number (as binary32, as the interface takes it) or one a row"""
    rows = len(x)
    cols = [np.broadcast_to(np.asarray(v, np.float32 if i != 1 else np.int64), rows)
            for i, v in enumerate((temperature, top_k, top_p, min_p))]
    out = [sample_row(x[r], float(u[r]), float(cols[0][r]), int(cols[1][r]), float(cols[2][r]), float(cols[3][r]))
           for r in range(rows)]
    return np.array([a for a, _ in out], np.int32), np.array([b for _, b in out], np.float64)


def embed_grad(grad, ids, n_states, scale=1.0):
    """-> (table, sum of magnitudes, terms) in binary64: what a bound on the sum's rounding needs beside the sum"""
    grad, ids = np.asarray(grad, np.float64), np.asarray(ids)
    inside = (ids >= 0) & (ids < n_states)
    table = np.zeros((n_states, grad.shape[1]))
    size = np.zeros_like(table)
    np.add.at(table, ids[inside], grad[inside])
    np.add.at(size, ids[inside], np.abs(grad[inside]))
    return table * scale, size * abs(scale), np.bincount(ids[inside], minlength=n_states)
