"""64-bit references of the sorted-rows and 4-bit operators' tests."""
import numpy as np

from quant_util import E2M1

MIDS = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])   # between neighbouring magnitudes
EVEN = np.array([0, 1, 0, 1, 0, 1, 0], bool)               # whether the upper neighbour's code is even


def mx_quant(x):
    """(codes [rows, cols], scale bytes [rows, ceil(cols / 32)], values) of rows of f64 values: the smallest power of
    two that holds the block's largest magnitude within 6, then the nearest value, ties to the even code."""
    x = np.asarray(x, np.float64)
    rows, cols = x.shape
    nb = (cols + 31) // 32
    v = np.zeros((rows, nb * 32))
    v[:, :cols] = x
    v = v.reshape(rows, nb, 32)
    bad = ~np.isfinite(v).all(2)
    v[bad] = 0
    a = np.abs(v).max(2)
    byte = np.full((rows, nb), 127, np.int64)
    for e in range(253, 0, -1):   # the smallest of 1..253 that holds it
        byte[(a > 0) & (a <= 6 * 2.0 ** (e - 127))] = e
    u = np.abs(v) / 2.0 ** (byte - 127.0)[:, :, None]
    n = ((u[..., None] > MIDS) | ((u[..., None] == MIDS) & EVEN)).sum(-1)
    codes = np.where(np.signbit(v), n + 8, n).reshape(rows, -1)[:, :cols]
    byte[bad] = 255
    vals = E2M1[codes] * np.repeat(2.0 ** (byte - 127.0), 32, 1)[:, :cols]
    vals[np.repeat(bad, 32, 1)[:, :cols]] = np.nan
    return codes, byte.astype(np.uint8), vals


def pack(codes):
    """Codes [rows, cols] as native bytes, low nibble first, a zero nibble behind an odd row."""
    c = np.asarray(codes, np.uint8)
    if c.shape[1] % 2:
        c = np.concatenate([c, np.zeros((len(c), 1), np.uint8)], 1)
    return (c[:, 0::2] | (c[:, 1::2] << 4)).astype(np.uint8)


def plan(idx, keff, mask, E):
    """Offsets [E + 1], live selections in sorted order, places [T, K]."""
    T, K = idx.shape
    by = [[] for _ in range(E)]
    for t in range(T):
        if mask is not None and not mask[t]:
            continue
        for k in range(K if keff is None else min(K, max(0, int(keff[t])))):
            if 0 <= idx[t, k] < E:
                by[idx[t, k]].append(t * K + k)
    off = np.concatenate([[0], np.cumsum([len(b) for b in by])]).astype(np.int32)
    src = np.array([s for b in by for s in b], np.int32)
    pos = np.full(T * K, -1, np.int32)
    pos[src] = np.arange(len(src), dtype=np.int32)
    return off, src, pos.reshape(T, K)


def combine(ys, pos, w, N):
    """(out, magnitudes) of sum_k w ys[pos] over the places within 0..N-1."""
    T, K = pos.shape
    out, mag = np.zeros((T, ys.shape[1])), np.zeros((T, ys.shape[1]))
    for t in range(T):
        for k in range(K):
            if 0 <= pos[t, k] < N:
                r = ys[pos[t, k]] * (1.0 if w is None else float(w[t, k]))
                out[t] += r
                mag[t] += np.abs(r)
    return out, mag


def silu(g):
    return np.where(g >= 0, g / (1 + np.exp(-np.abs(g))), g * np.exp(-np.abs(g)) / (1 + np.exp(-np.abs(g))))
