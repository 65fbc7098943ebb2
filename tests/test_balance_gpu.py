"""Per-expert counts, the balance loss and the gradient of the router's logits
(coli_hip_balance_dev, coli_hip_balance_grad_dev, coli_hip_moe_last_balance_dev)
against the definition in 64 bits."""
import ctypes as C

import numpy as np
import pytest

from balance_ref import balance, scores
from colibri_amd import hiprt
from colibri_amd.backend import ColiHipMoeConfig, f32p, i32p, tensor_array
from moe_ref import Layer, make_router_inputs
from op_util import Bufs

pytestmark = pytest.mark.gpu


def p_tol(z):
    """Relative error of a score over the row's sum: the exponent's argument, up
    to s = max |z| + |max z| of the row, is rounded before it is multiplied with
    log2 e (1.45 s 2^-24, twice for the difference), and about sixteen roundings
    of 2^-23 (exp2, log2, rcp, sqrt and the sums) follow; a sum shares that of
    its largest terms."""
    f = np.where(np.isfinite(z) & (np.abs(z) < 1e30), z, 0.0)
    return (3.0 * float(np.abs(f).max(initial=0.0)) + 32.0) * 2.0 ** -23


def run(session, z, idx, keff, mask, off, mode, dloss, dz0, n):
    b = session.b
    T, E = z.shape
    with Bufs(b) as d:
        pz, pi = d.up(z), d.up(idx)
        pk, pm, po = (None if v is None else d.up(v) for v in (keff, mask, off))
        pl, pc, pr = d.up(np.full(n, 7.0, np.float32)), d.up(np.full((n, E), 7, np.int32)), d.up(np.full(n, 7, np.int32))
        pd, pg = d.up(dloss), d.up(dz0)
        assert b.hip_balance_dev(0, pz, pi, pk, pm, po, n, T, E, idx.shape[1], mode, pl, pc, pr)
        assert b.hip_balance_grad_dev(0, pz, pm, po, n, T, E, mode, pd, pc, pr, pg)
        return d.down(pl, (n,)), d.down(pc, (n, E), np.int32), d.down(pr, (n,), np.int32), d.down(pg, (T, E))


def check(session, z, idx, keff, mask, off, mode, seed=0):
    rng = np.random.default_rng(seed)
    T, E = z.shape
    n = 1 if off is None else len(off) - 1
    dloss = rng.standard_normal(n).astype(np.float32)
    dz0 = np.full((T, E), 7.0, np.float32)
    loss, counts, rows, dz = run(session, z, idx, keff, mask, off, mode, dloss, dz0, n)
    rl, rc, rr, rg, mag = balance(z, idx, keff, mask, off, E, mode, dloss, dz0)
    assert np.array_equal(counts, rc) and np.array_equal(rows, rr)
    t = p_tol(z) + (T / 16 + 96) * 2.0 ** -24
    assert (np.abs(loss - rl) <= t * np.abs(rl) + 1e-30).all(), (np.abs(loss - rl) / rl).max()
    # a row of no sequence: as it was
    inside = np.zeros(T, bool)
    inside[0 if off is None else off[0]: T if off is None else off[-1]] = True
    assert (dz[~inside] == 7.0).all()
    err = np.abs(dz - rg)
    # (2^-126: results below the normal range are flushed)
    bad = inside[:, None] & ~(err <= 2 * p_tol(z) * mag + 2.0 ** -126)
    assert not bad.any(), (int(bad.sum()), float((err[inside] / np.maximum(mag[inside], 1e-30)).max()))
    return loss, dz


def routed(rng, T, E, K, spread=1.0):
    z = (rng.standard_normal((T, E)) * spread).astype(np.float32)
    idx = np.argsort(-z, 1)[:, :K].astype(np.int32)
    return z, np.ascontiguousarray(idx)


SHAPES = [  # T, E, K, offsets
    (1, 1, 1, None), (1, 8, 2, None), (3, 5, 2, [0, 0, 2, 2, 3]), (64, 64, 8, None), (128, 384, 8, [0, 100, 128]),
    (129, 63, 3, None), (200, 130, 4, [5, 60, 60, 61, 180]), (777, 256, 8, [0, 1, 2, 3, 500, 770]),
    (300, 1024, 6, [0, 300]), (1000, 7, 7, [0] + list(range(100, 1000, 3))), (5000, 96, 2, [0, 4990]),
    (40000, 16, 1, None), (700, 512, 64, [0, 350, 700]),
]


@pytest.mark.parametrize("mode", [0, 1, 2, 3])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s[:3])))
def test_matches_definition(session, mode, shape):
    T, E, K, off = shape
    rng = np.random.default_rng(T + E + mode)
    z, idx = routed(rng, T, E, K)
    off = None if off is None else np.asarray(off, np.int32)
    keff = rng.integers(0, K + 1, T).astype(np.int32) if T % 2 else None
    mask = (rng.random(T) < 0.8).astype(np.uint8) if E % 2 == 0 else None
    check(session, z, idx, keff, mask, off, mode, T)


@pytest.mark.parametrize("T", [30, 300])
@pytest.mark.parametrize("E", [1, 2, 3, 4, 5, 65, 127, 129, 257, 258, 385, 386, 513, 515, 769, 1023])
def test_odd_numbers_of_experts(session, E, T):
    """Widths at which the last columns are loaded moved back, one at a time, or not at all."""
    rng = np.random.default_rng(E + T)
    z, idx = routed(rng, T, E, min(E, 3))
    check(session, z, idx, None, (rng.random(T) < 0.7).astype(np.uint8), np.array([1, T // 2, T - 1], np.int32), (0, 1, 3)[E % 3])


@pytest.mark.parametrize("E", [48, 130])
def test_gradient_in_place(session, E):
    """dlogits may be the logits themselves; not a part of them moved by some elements."""
    b = session.b
    rng = np.random.default_rng(E)
    T, off = 500, np.array([0, 7, 200, 490], np.int32)
    z, idx = routed(rng, T, E, 4)
    one = np.ones(3, np.float32)
    loss, counts, rows, dz = run(session, z, idx, None, None, off, 1, one, z, 3)
    with Bufs(b) as d:
        pz, po, pd, pc, pr = d.up(z), d.up(off), d.up(one), d.up(counts), d.up(rows)
        assert not b.hip_balance_grad_dev(0, pz, None, po, 3, T - 1, E, 1, pd, pc, pr, pz + 4 * E)
        assert b.hip_balance_grad_dev(0, pz, None, po, 3, T, E, 1, pd, pc, pr, pz)
        assert np.array_equal(d.down(pz, (T, E)).view(np.uint32), dz.view(np.uint32))


@pytest.mark.parametrize("T", [40, 400])
@pytest.mark.parametrize("mode", [0, 1, 3])
def test_masked_places(session, mode, T):
    """Sequences whose mask leaves no row, rows without selections, indices of no
    expert, logits of -inf and of the type's lowest value, a row of nothing but
    -inf, NaN and infinities in masked rows and behind the last sequence."""
    rng = np.random.default_rng(mode + T)
    E, K = 24, 4
    z, idx = routed(rng, T, E, K, 3.0)
    off = np.array([0, T // 4, T // 2, T // 2, T - 5], np.int32)
    mask = np.ones(T, np.uint8)
    mask[T // 4: T // 2] = 0                   # a sequence of masked rows
    mask[3] = 0
    z[3], z[T // 4], z[T - 1], z[T - 2] = np.nan, np.inf, np.nan, -np.inf
    z[:, 7] = -np.inf
    z[5:9, 2] = np.finfo(np.float32).min
    z[10] = -np.inf
    idx[12] = -1
    idx[13, 1] = E
    keff = np.full(T, K, np.int32)
    keff[14], keff[15] = 0, -3
    check(session, z, idx, keff, mask, off, mode)
    keff[:] = 0                                 # no selection at all: loss and gradients 0
    loss, dz = check(session, z, idx, keff, mask, off, mode)
    assert not loss.any() and not dz[: T - 5].any()


@pytest.mark.parametrize("mode", [0, 1, 3])
def test_far_logits(session, mode):
    """Rows whose scores all underflow in 32 bits (z to -300), rows of large ones."""
    rng = np.random.default_rng(mode)
    z, idx = routed(rng, 96, 40, 4)
    z[:32] -= 200.0
    z[32:48] -= 40.0
    z[48:56] -= 27.5
    z[64:] += 30.0
    check(session, z, idx, None, None, np.array([0, 32, 64, 96], np.int32), mode)


def test_nan_row_reaches_its_sequence_only(session):
    rng = np.random.default_rng(4)
    z, idx = routed(rng, 300, 32, 4)
    z[150, 3] = np.nan
    off = np.array([0, 100, 200, 300], np.int32)
    loss, counts, rows, dz = run(session, z, idx, None, None, off, 0, np.ones(3, np.float32), np.zeros((300, 32), np.float32), 3)
    assert np.isnan(loss[1]) and np.isfinite(loss[[0, 2]]).all()
    assert np.isnan(dz[150]).all() and np.isfinite(np.delete(dz, 150, 0)).all()
    assert (rows == 100).all() and (counts.sum(1) == 400).all()


@pytest.mark.parametrize("mode", [0, 2, 3])
def test_gradient_against_differences(session, mode):
    """Central differences of the forward call's loss, the selections fixed.

    With step h the difference is off by h^2 / 6 of the loss's third derivative
    (a sum of f_e p_e / n, |p'''| <= 1 and the weights at most max f / n, two of
    them) and by the two losses' own error over 2 h."""
    rng = np.random.default_rng(8)
    T, E, K, h = 5, 12, 3, 2.0 ** -5
    z, idx = routed(rng, T, E, K)
    off, one, dz0 = np.array([0, 5], np.int32), np.ones(1, np.float32), np.zeros((T, E), np.float32)
    loss, counts, _, dz = run(session, z, idx, None, None, off, mode, one, dz0, 1)
    f = counts[0] * E / counts.sum()
    tol = h * h / 6 * 2 * f.max() / T + 2 * p_tol(z) * loss[0] / (2 * h)
    for t, e in ((0, 0), (2, 5), (4, 11), (3, int(idx[3, 0]))):
        v = []
        for s in (1, -1):
            zz = z.copy()
            zz[t, e] += np.float32(s * h)
            v.append((float(run(session, zz, idx, None, None, off, mode, one, dz0, 1)[0][0]), float(zz[t, e])))
        assert abs((v[0][0] - v[1][0]) / (v[0][1] - v[1][1]) - dz[t, e]) <= tol


def test_repeats_bitwise_and_unaligned(session):
    b = session.b
    rng = np.random.default_rng(12)
    T, E, K = 3000, 64, 4
    z, idx = routed(rng, T, E, K)
    with Bufs(b) as d:
        pz, pi = d.up(np.concatenate((np.zeros(1, np.float32), z.ravel()))), d.up(idx)
        pa = d.up(z)
        got = []
        for p in (pa, pa, pz + 4):
            pl, pc, pr, pg = (d.up(np.zeros(k, np.float32)) for k in (1, E, 1, T * E + 1))
            pd = d.up(np.ones(1, np.float32))
            g = pg + 4 if p == pz + 4 else pg
            assert b.hip_balance_dev(0, p, pi, None, None, None, 1, T, E, K, 1, pl, pc, pr)
            assert b.hip_balance_grad_dev(0, p, None, None, 1, T, E, 1, pd, pc, pr, g)
            out = d.down(pg, (T * E + 1,))
            got.append((d.down(pl, (1,)), d.down(pc, (E,), np.int32), out[1:] if g != pg else out[:-1]))
        for other in got[1:]:
            for u, v in zip(got[0], other):
                assert np.array_equal(u.view(np.uint32), v.view(np.uint32))


def test_balanced_loads_give_one(session):
    """Every expert selected alike and scored alike: f_e = 1, P_e = 1 / E."""
    T, E, K = 512, 32, 4
    z = np.zeros((T, E), np.float32)
    idx = ((np.arange(T)[:, None] * K + np.arange(K)) % E).astype(np.int32)
    for mode in range(4):
        loss, dz = check(session, z, idx, None, None, None, mode)
        assert abs(float(loss[0]) - 1.0) <= 64 * 2.0 ** -24


@pytest.mark.parametrize("T", [50, 1500])
def test_graph_replays(session, T):
    b = session.b
    rng = np.random.default_rng(T)
    E, K, n = 48, 4, 3
    z, idx = routed(rng, T, E, K)
    z2, idx2 = routed(rng, 9000, 200, 8)
    off = np.array([0, T // 3, T // 2, T - 1], np.int32)
    with Bufs(b) as d:
        pz, pi, po, pd = d.up(z), d.up(idx), d.up(off), d.up(np.ones(n, np.float32))
        qz, qi, ql, qc, qr = d.up(z2), d.up(idx2), d.up(np.zeros(1, np.float32)), d.up(np.zeros(200, np.int32)), d.up(np.zeros(1, np.int32))
        pl, pc, pr, pg = d.up(np.zeros(n, np.float32)), d.up(np.zeros((n, E), np.int32)), d.up(np.zeros(n, np.int32)), d.up(z * 0)

        def step():
            assert b.hip_balance_dev(0, pz, pi, None, None, po, n, T, E, K, 3, pl, pc, pr)
            assert b.hip_balance_grad_dev(0, pz, None, po, n, T, E, 3, pd, pc, pr, pg)

        def got():
            return [d.down(p, s, np.uint32) for p, s in ((pl, (n,)), (pc, (n, E)), (pr, (n,)), (pg, (T - 1, E)))]

        step()
        eager = got()
        with hiprt.Graph(b.hip_stream(0)) as g:
            step()
        for rep in range(3):
            for p, k in ((pl, n), (pc, n * E), (pr, n), (pg, T * E)):
                assert b.hip_fill_random_u8(0, p, k * 4, rep + 1)
            g.launch()
            for u, v in zip(eager, got()):
                assert np.array_equal(u, v), rep
            assert b.hip_balance_dev(0, qz, qi, None, None, None, 1, 9000 - rep, 200, 8, 0, ql, qc, qr)


@pytest.mark.parametrize("mode,S,E,K,D", [(0, 1, 64, 8, 2048), (0, 9, 64, 8, 256), (2, 5, 128, 8, 1536), (1, 70, 33, 4, 640),
                                          (3, 300, 96, 6, 384), (2, 1, 256, 8, 1024), (0, 1, 128, 8, 512),
                                          (3, 1, 40, 4, 384), (0, 64, 64, 8, 256), (1, 65, 64, 8, 256), (0, 2, 16, 2, 256)])
def test_last_forward_of_a_layer(session, mode, S, E, K, D):
    """Counts and loss of the layer's own router after a forward."""
    rng = np.random.default_rng(S + E)
    b = session.b
    layer = Layer(rng, 4, D, 128, E, shared=False)
    x, W, bias = make_router_inputs(rng, S, D, E, K, mode, bias=mode != 0)
    hs = layer.upload(session)
    m = C.c_void_p()
    try:
        (g, _a), (u, _b), (w, _c) = (tensor_array([t[k] for t in hs[:E]]) for k in range(3))
        cfg = ColiHipMoeConfig(D, 128, E, K, mode, 1, 0.0, 1.0, 0)
        assert b.hip_moe_create(C.byref(m), 0, C.byref(cfg), f32p(W), None if bias is None else f32p(bias), g, u, w, None,
                                None, None)
        with Bufs(b) as d:
            pl, pc, pr = d.up(np.zeros(2, np.float32)), d.up(np.zeros((2, E), np.int32)), d.up(np.zeros(2, np.int32))
            assert not b.hip_moe_last_balance_dev(m, None, None, 1, pl, pc, pr)   # no forward yet
            out, idx = np.zeros((S, D), np.float32), np.zeros((S, K), np.int32)
            wt, keff = np.zeros((S, K), np.float32), np.zeros(S, np.int32)
            assert b.hip_moe_forward(m, f32p(x), f32p(out), S, i32p(idx), f32p(wt), i32p(keff))
            off = np.array([0, S // 2, S], np.int32)
            assert b.hip_moe_last_balance_dev(m, None, d.up(off), 2, pl, pc, pr)
            loss, counts, rows = d.down(pl, (2,)), d.down(pc, (2, E), np.int32), d.down(pr, (2,), np.int32)
        z = x.astype(np.float64) @ W.astype(np.float64).T
        rl, rc, rr, _, _ = balance(z, idx, keff, None, off, E, mode)
        assert np.array_equal(counts, rc) and np.array_equal(rows, rr)
        # a logit is an f32 sum of D products: off by (2 D + 16) 2^-24 of their
        # magnitudes, and a score over its sum by twice that, relatively
        dz = ((np.abs(x).astype(np.float64) @ np.abs(W).astype(np.float64).T).max() * (2 * D + 16)) * 2.0 ** -24
        assert (np.abs(loss - rl) <= (p_tol(z) + (S / 16 + 96) * 2.0 ** -24 + 2 * dz) * rl).all()
    finally:
        if m:
            b.hip_moe_free(m)
        for t in hs:
            for h in t:
                session.free(h)


def test_refusals(session):
    b = session.b
    with Bufs(b) as d:
        p = d.up(np.zeros(4096, np.float32))
        ok = (0, p, p, None, None, p, 1, 4, 8, 2, 0, p, p, p)
        for k, bad in ((0, 9), (0, -1), (1, None), (2, None), (6, 0), (6, 16385), (7, 0), (7, (1 << 24) + 1), (8, 0), (8, 1025),
                       (9, 0), (9, 9), (9, 65), (10, -1), (10, 4), (11, None), (12, None), (13, None)):
            assert not b.hip_balance_dev(*(ok[:k] + (bad,) + ok[k + 1:])), (k, bad)
        assert not b.hip_balance_dev(0, p, p, None, None, None, 2, 4, 8, 2, 0, p, p, p)   # sequences without offsets
        ok = (0, p, None, p, 1, 4, 8, 0, p, p, p, p)
        for k, bad in ((0, 9), (1, None), (4, 0), (5, 0), (6, 1025), (7, 4), (8, None), (9, None), (10, None), (11, None)):
            assert not b.hip_balance_grad_dev(*(ok[:k] + (bad,) + ok[k + 1:])), (k, bad)
        assert not b.hip_balance_grad_dev(0, p, None, None, 2, 4, 8, 0, p, p, p, p)
        assert not b.hip_moe_last_balance_dev(None, None, None, 1, p, p, p)


@pytest.mark.parametrize("n", [1023, 1024, 5000])
@pytest.mark.parametrize("mode", [0, 3])
def test_many_sequences(session, mode, n):
    """Offsets held in LDS up to 1023 sequences, read from memory beyond."""
    rng = np.random.default_rng(n + mode)
    T, E, K = 6001, 20, 2
    z, idx = routed(rng, T, E, K)
    off = np.concatenate(([3], np.sort(rng.integers(3, T - 4, n - 1)), [T - 4])).astype(np.int32)
    check(session, z, idx, None, (rng.random(T) < 0.9).astype(np.uint8), off, mode, n)


@pytest.mark.parametrize("E,off", [(130, [0, 2900, 3000]), (130, [7, 900, 2990]), (1000, [0, 1, 3000])])
def test_long_sequences_joined_by_columns(session, E, off):
    """Sequences of so many rows that the join takes 64 columns a workgroup; the
    last to arrive adds the pieces of the loss, also on a second call."""
    rng = np.random.default_rng(E + off[1])
    z, idx = routed(rng, 3000, E, 4)
    for mode in (0, 1):
        check(session, z, idx, None, None, np.asarray(off, np.int32), mode)


class LayerOf:
    """A MoE layer of `E` random experts with its router, and the routing of S rows by the host forward."""

    def __init__(self, session, mode, E, K, D, rows, seed):
        self.session, self.b, self.mode, self.E, self.K, self.D = session, session.b, mode, E, K, D
        rng = np.random.default_rng(seed)
        layer = Layer(rng, 4, D, 128, E, shared=False)
        self.x, self.W, bias = make_router_inputs(rng, rows, D, E, K, mode, bias=mode != 0)
        self.hs = layer.upload(session)
        self.m = C.c_void_p()
        (g, _a), (u, _b), (w, _c) = (tensor_array([t[k] for t in self.hs[:E]]) for k in range(3))
        cfg = ColiHipMoeConfig(D, 128, E, K, mode, 1, 0.0, 1.0, 0)
        assert self.b.hip_moe_create(C.byref(self.m), 0, C.byref(cfg), f32p(self.W), None if bias is None else f32p(bias),
                                     g, u, w, None, None, None)
        self.d = Bufs(self.b)
        self.px, self.py = self.d.up(self.x), self.d.up(np.zeros_like(self.x))
        self.pl, self.pc, self.pr = self.d.up(np.zeros(1, np.float32)), self.d.up(np.zeros(E, np.int32)), self.d.up(np.zeros(1, np.int32))

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.b.hip_moe_free(self.m)
        for t in self.hs:
            for h in t:
                self.session.free(h)
        self.d.__exit__()

    def forward(self, S, at=0):
        """S rows from row `at` on."""
        assert self.b.hip_moe_forward_dev(self.m, self.px + 4 * at * self.D, self.py, S)

    def balance(self):
        return self.b.hip_moe_last_balance_dev(self.m, None, None, 1, self.pl, self.pc, self.pr)

    def routing(self, S, at=0):
        out, idx = np.zeros((S, self.D), np.float32), np.zeros((S, self.K), np.int32)
        wt, keff = np.zeros((S, self.K), np.float32), np.zeros(S, np.int32)
        x = np.ascontiguousarray(self.x[at: at + S])
        assert self.b.hip_moe_forward(self.m, f32p(x), f32p(out), S, i32p(idx), f32p(wt), i32p(keff))
        return idx, keff

    def check(self, S, routing, at=0):
        """What the last call of balance() left is that of these S rows."""
        loss, counts, rows = self.d.down(self.pl, (1,)), self.d.down(self.pc, (1, self.E), np.int32), self.d.down(self.pr, (1,), np.int32)
        x = self.x[at: at + S].astype(np.float64)
        z = x @ self.W.astype(np.float64).T
        rl, rc, rr, _, _ = balance(z, routing[0], routing[1], None, None, self.E, self.mode)
        assert np.array_equal(rows, rr) and np.array_equal(counts, rc), (S, rows, rr)
        dz = ((np.abs(x) @ np.abs(self.W).astype(np.float64).T).max() * (2 * self.D + 16)) * 2.0 ** -24
        assert (np.abs(loss - rl) <= (p_tol(z) + (S / 16 + 96) * 2.0 ** -24 + 2 * dz) * rl).all()


# one-token forms (gate/up that selects for itself; the shared overlap is not
# taken without a shared expert), the one-launch routing, the selection by four
# waves and the separate union
@pytest.mark.parametrize("mode,E,K,D,few", [(0, 64, 8, 2048, 1), (0, 64, 8, 256, 5), (2, 96, 8, 1536, 9), (3, 40, 4, 384, 70)])
def test_last_forward_after_replays(session, mode, E, K, D, few):
    """The last forward is the last one that ran: a replayed graph's, also where
    another number of rows was queued or captured after the graph was."""
    with LayerOf(session, mode, E, K, D, 300, E + few) as o:
        ref = {S: o.routing(S) for S in (300, few)}
        o.forward(300)
        assert o.balance()                          # (workspaces)
        graphs = {}
        for S in (few, 300):
            with hiprt.Graph(o.b.hip_stream(0)) as graphs[S]:
                o.forward(S)
        with hiprt.Graph(o.b.hip_stream(0)) as alone:
            assert o.balance()
        for rep in range(2):
            for S in (few, 300):
                other = few + 300 - S
                graphs[S].launch()                  # (300 rows captured last)
                assert o.balance()
                o.check(S, ref[S])
                o.forward(other)
                graphs[S].launch()                  # (the other number queued last)
                assert o.balance()
                o.check(S, ref[S])
                o.b.hip_fill_random_u8(0, o.pc, 4 * E, rep + 1)
                alone.launch()
                o.check(S, ref[S])
                o.forward(other)
                alone.launch()
                o.check(other, ref[other])


@pytest.mark.parametrize("mode,E,K,D,S", [(0, 64, 8, 2048, 1), (2, 96, 8, 384, 9), (1, 40, 4, 256, 70)])
def test_graphs_outlive_larger_forwards(session, mode, E, K, D, S):
    """A captured forward with its balance, and a balance captured alone, after
    forwards of more rows have outgrown the layer's buffers; the union read back
    is the replayed forward's."""
    b = session.b
    with LayerOf(session, mode, E, K, D, 300, E + S) as o:
        small, large = o.routing(S), None

        def outputs():
            return [o.d.down(p, n, np.uint32) for p, n in ((o.py, (S, D)), (o.pl, (1,)), (o.pc, (E,)), (o.pr, (1,)))]

        o.forward(S)
        assert o.balance()
        eager = outputs()
        with hiprt.Graph(b.hip_stream(0)) as both:
            o.forward(S)
            assert o.balance()
        with hiprt.Graph(b.hip_stream(0)) as alone:
            assert o.balance()
        nu, uniq = C.c_int(), np.zeros(E, np.int32)
        for rep, rows in enumerate((S + 1, 130, 300)):   # (each needs larger buffers)
            large = o.routing(rows)
            alone.launch()
            o.check(rows, large)
            for p, n in ((o.py, S * D), (o.pl, 1), (o.pc, E), (o.pr, 1)):
                assert b.hip_fill_random_u8(0, p, 4 * n, rep + 1)
            both.launch()
            for u, v in zip(outputs(), eager):
                assert np.array_equal(u, v), rep
            assert b.hip_moe_last_union(o.m, C.byref(nu), i32p(uniq))
            seen = [e for t in range(S) for e in small[0][t, : small[1][t]]]
            assert list(uniq[: nu.value]) == list(dict.fromkeys(seen))
            alone.launch()
            o.check(S, small)
            o.forward(rows)
            assert o.balance()
            o.check(rows, large)


def test_outputs_over_inputs_are_refused(session):
    b = session.b
    T, E, K, n = 40, 8, 2, 2
    with Bufs(b) as d:
        z, idx, keff, mask = d.up(np.zeros((T, E), np.float32)), d.up(np.zeros((T, K), np.int32)), d.up(np.zeros(T, np.int32)), d.up(np.ones(T, np.uint8))
        off = d.up(np.array([0, 20, 40], np.int32))
        loss, counts, rows, dl = d.up(np.zeros(n, np.float32)), d.up(np.zeros((n, E), np.int32)), d.up(np.zeros(n, np.int32)), d.up(np.zeros(n, np.float32))
        dz = d.up(np.zeros((T, E), np.float32))
        ok = (0, z, idx, keff, mask, off, n, T, E, K, 0, loss, counts, rows)
        assert b.hip_balance_dev(*ok)
        for k, size in ((11, 4 * n), (12, 4 * n * E), (13, 4 * n)):
            for p, nb in ((z, 4 * T * E), (idx, 4 * T * K), (keff, 4 * T), (mask, T), (off, 4 * (n + 1))):
                for bad in (p, p + nb - 4, p - size + 4):
                    assert not b.hip_balance_dev(*(ok[:k] + (bad,) + ok[k + 1:])), (k, bad)
        for k, bad in ((11, counts + 4 * n * E - 4), (12, rows), (13, loss + 4)):
            assert not b.hip_balance_dev(*(ok[:k] + (bad,) + ok[k + 1:])), (k, bad)
        ok = (0, z, mask, off, n, T, E, 0, dl, counts, rows, dz)
        assert b.hip_balance_grad_dev(*ok)
        for p, nb in ((mask, T), (off, 4 * (n + 1)), (dl, 4 * n), (counts, 4 * n * E), (rows, 4 * n)):
            for bad in (p, p + nb - 4, p - 4 * T * E + 4):
                assert not b.hip_balance_grad_dev(*(ok[:11] + (bad,))), bad


@pytest.mark.parametrize("mode", [0, 1, 3])
def test_small_scores_beside_larger_ones(session, mode):
    """Rows whose largest logit is far below zero and whose others lie farther:
    each score keeps its own relative accuracy while it is above 2^-126."""
    rng = np.random.default_rng(60 + mode)
    T, E = 40, 24
    z, idx = routed(rng, T, E, 4)
    if mode == 3:   # rows of -50 at most (scores of 1e-11) down to -100, and of -20 down to -84
        z[:20] = -50.0 - 50.0 * rng.random((20, E))
        z[20:] = -20.0 - 64.0 * rng.random((20, E))
    else:           # from -20 down to -84: softmax's 64 under its maximum
        z[:, 0] = -20.0
        z[:, 1:] = -20.0 - 64.0 * rng.random((T, E - 1))
    z = z.astype(np.float32)
    check(session, z, idx, None, None, np.array([0, 10, 40], np.int32), mode)


@pytest.mark.parametrize("S", [5, 300])
def test_forward_captured_before_any_ran(session, S):
    """A layer whose only forward has been captured (in the mode that lets it
    allocate) and not replayed yet: no rows, then the replay's."""
    b = session.b
    with LayerOf(session, 1, 40, 4, 256, 300, 90) as warm, LayerOf(session, 1, 40, 4, 256, 300, 91) as o, \
            LayerOf(session, 1, 40, 4, 256, 300, 91) as ref:
        warm.forward(S)
        assert warm.balance() and not o.balance()
        lib, st = hiprt.lib(), b.hip_stream(0)
        graph, ex = C.c_void_p(), C.c_void_p()
        hiprt.device_sync()
        hiprt.check(lib.hipStreamBeginCapture(st, 2), "capture")
        ok = b.hip_moe_forward_dev(o.m, o.px, o.py, S)
        hiprt.check(lib.hipStreamEndCapture(st, C.byref(graph)), "capture end")
        hiprt.check(lib.hipGraphInstantiate(C.byref(ex), graph, None, None, 0), "instantiate")
        try:
            assert ok and b.hip_fill_random_u8(0, o.pc, 4 * 40, 1) and o.balance()
            assert not o.d.down(o.pc, (40,), np.int32).any() and not o.d.down(o.pr, (1,), np.int32).any()
            assert not o.d.down(o.pl, (1,)).any()
            for _ in range(2):
                hiprt.check(lib.hipGraphLaunch(ex, st), "replay")
                assert o.balance()
                o.check(S, ref.routing(S))
        finally:
            hiprt.device_sync()
            lib.hipGraphExecDestroy(ex)
            lib.hipGraphDestroy(graph)
