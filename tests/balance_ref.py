"""The balance loss of routed rows and its gradient in 64 bits, from the definition."""
import numpy as np


def scores(z, mode):
    """p [T, E] (scores over their sum; 0 in a row of nothing but -inf) and u'(z)."""
    z = z.astype(np.float64)
    with np.errstate(all="ignore"):
        if mode == 0:
            u, up = z, np.ones_like(z)
        elif mode == 3:
            u = 0.5 * np.where(z < -30, z, np.log(np.logaddexp(0.0, z)))
            up = np.where(z < -30, 0.5, 0.5 / (1 + np.exp(-z)) / np.logaddexp(0.0, z))
        else:
            u, up = -np.logaddexp(0.0, -z), 1 / (1 + np.exp(z))
        m = u.max(1, keepdims=True)
        e = np.exp(u - np.where(np.isinf(m) & (m < 0), 0.0, m))
        s = e.sum(1, keepdims=True)
        return np.where(s == 0, 0.0, e / np.where(s == 0, 1.0, s)), up


def balance(z, idx, keff, mask, off, E, mode, dloss=None, dz=None):
    """loss, counts, rows and (dloss given) dz, the rows of no sequence as `dz` has them."""
    T, K = idx.shape
    n = 1 if off is None else len(off) - 1
    off = [0, T] if off is None else off
    loss, counts, rows = np.zeros(n), np.zeros((n, E), np.int32), np.zeros(n, np.int32)
    p, up = scores(z, mode)
    out = None if dloss is None else dz.astype(np.float64).copy()
    mag = None if dloss is None else np.zeros((T, E))
    for i in range(n):
        at = np.arange(off[i], off[i + 1])
        if out is not None:
            out[at] = 0
        if mask is not None:
            at = at[mask[at] != 0]
        rows[i] = len(at)
        for t in at:
            for k in range(K if keff is None else min(K, max(0, keff[t]))):
                if 0 <= idx[t, k] < E:
                    counts[i, idx[t, k]] += 1
        C = int(counts[i].sum())
        if not C or not len(at):
            continue
        f = counts[i] * (E / C)
        loss[i] = (f * p[at].mean(0)).sum()
        if out is not None:
            w = float(dloss[i]) / len(at) * f
            d = (p[at] * w).sum(1, keepdims=True)
            out[at] = p[at] * (w - d) * up[at]
            mag[at] = p[at] * (np.abs(w) + np.abs(d)) * up[at]
    return loss, counts, rows, out, mag
