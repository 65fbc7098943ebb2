"""Adapters beside a resident projection (coli_hip_lora_*) against 64-bit
products with the dequantized matrix and the adapters' stored values."""
import ctypes as C

import numpy as np
import pytest

from colibri_amd import hiprt
from op_util import Bufs, bits, close, gemm_tol, matrix, sum_tol

pytestmark = pytest.mark.gpu


class Case:
    """A projection, a bank with some slots filled, and rows with slots."""

    def __init__(self, session, seed, kind, O, I, S, slots, rank, dtype, pattern="runs", ranks=None):
        b, rng = session.b, np.random.default_rng(seed)
        self.session, self.b, self.O, self.I, self.S, self.slots, self.rank = session, b, O, I, S, slots, rank
        self.h, self.w = matrix(session, rng, kind, O, I)
        self.bank = C.c_void_p()
        assert b.hip_lora_create(C.byref(self.bank), 0, I, O, slots, rank, dtype)
        self.d = Bufs(b)
        self.a, self.bm, self.sc = np.zeros((slots, rank, I)), np.zeros((slots, O, rank)), np.zeros(slots)
        # one slot stays empty where there are several; ranks from the largest down to 1
        self.ranks = ranks or [rank if s == 0 else 0 if s == 2 else max(1, rank - 3 * s) for s in range(slots)]
        for s, r in enumerate(self.ranks):
            if r:
                self.set(s, rng.standard_normal((r, I)) / np.sqrt(I), rng.standard_normal((O, r)), 0.5 + s, dtype)
        if pattern == "runs":
            self.slot = np.repeat(rng.integers(-1, slots + 1, (S + 6) // 7), 7)[:S].astype(np.int32)
        elif pattern == "mixed":
            self.slot = rng.integers(-1, slots + 1, S).astype(np.int32)
        else:
            self.slot = np.full(S, int(pattern), np.int32)
        self.x = rng.standard_normal((S, I)).astype(np.float32)
        self.dy = rng.standard_normal((S, O)).astype(np.float32)

    def set(self, s, a, bm, scale, dtype):
        ra, va = bits(dtype, a)
        rb, vb = bits(dtype, bm)
        r = a.shape[0]
        assert self.b.hip_lora_set_dev(self.bank, s, self.d.up(ra), self.d.up(rb), r, scale)
        self.a[s], self.bm[s], self.sc[s] = 0, 0, np.float32(scale)
        self.a[s, :r], self.bm[s, :, :r] = va, vb

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.b.hip_lora_free(self.bank)
        self.session.free(self.h)
        self.d.__exit__()

    def delta(self, x, a, bm, sgn=lambda v: v):
        """scale B A x of every row (sgn np.abs: the terms' magnitudes)."""
        out = np.zeros((len(x), bm.shape[1]))
        for s in range(self.slots):
            at = self.slot == s
            out[at] = self.sc[s] * (sgn(x[at].astype(np.float64)) @ sgn(a[s]).T) @ sgn(bm[s]).T
        return out

    def check_forward(self):
        S, O, I = self.S, self.O, self.I
        px, py, ps = self.d.up(self.x), self.d.up(np.full((S + 2, O), 7.0, np.float32)), self.d.up(self.slot)
        assert self.b.hip_lora_gemm_dev(self.h, self.bank, py, px, S, ps)
        got = self.d.down(py, (S + 2, O))
        assert (got[S:] == 7.0).all()
        x = self.x.astype(np.float64)
        ref = x @ self.w.T + self.delta(x, self.a, self.bm)
        mag = np.abs(x) @ np.abs(self.w).T
        close(got[:S], ref, mag * gemm_tol(I) + self.delta(x, self.a, self.bm, np.abs) * sum_tol(I + self.rank), 1.0)
        return got[:S]

    def check_grads(self, want_dx=True):
        S, O, I, n, r = self.S, self.O, self.I, self.slots, self.rank
        d = self.d
        px, pdy, ps = d.up(self.x), d.up(self.dy), d.up(self.slot)
        pdx, pda = d.up(np.full((S, I), 7.0, np.float32)), d.up(np.full((n, r, I), 7.0, np.float32))
        pdb = d.up(np.full((n, O, r), 7.0, np.float32))
        assert self.b.hip_lora_grad_dev(self.h, self.bank, px, pdy, S, ps, pdx if want_dx else None, pda, pdb)
        dx, da, db = d.down(pdx, (S, I)), d.down(pda, (n, r, I)), d.down(pdb, (n, O, r))
        x, dy = self.x.astype(np.float64), self.dy.astype(np.float64)
        if want_dx:
            bt, at = self.bm.transpose(0, 2, 1), self.a.transpose(0, 2, 1)
            ref = dy @ self.w + self.delta(dy, bt, at)
            close(dx, ref, np.abs(dy) @ np.abs(self.w) * gemm_tol(O) +
                  self.delta(dy, bt, at, np.abs) * sum_tol(O + r), 1.0, "dx")
        else:
            assert (dx == 7.0).all()
        for s in range(n):
            at = self.slot == s
            xs, ds, a, bm, k = x[at], dy[at], self.a[s], self.bm[s], self.sc[s]
            t = sum_tol(max(I, O) + S)
            close(da[s], k * (ds @ bm).T @ xs, k * (np.abs(ds) @ np.abs(bm)).T @ np.abs(xs), t, f"dA {s}")
            close(db[s], k * ds.T @ (xs @ a.T), k * np.abs(ds).T @ (np.abs(xs) @ np.abs(a).T), t, f"dB {s}")
        return dx, da, db


SHAPES = [  # kind, O, I, S, slots, rank, dtype, pattern
    ("i4h", 4, 5, 1, 1, 1, 0, "0"),
    ("i4f", 7, 6, 70, 2, 3, 1, "mixed"),
    ("i4h", 64, 96, 1, 1, 8, 1, "0"),
    ("fp4", 200, 130, 1, 3, 16, 2, "1"),
    ("i4f", 33, 65, 5, 4, 5, 0, "mixed"),
    ("row4", 300, 128, 16, 4, 17, 2, "mixed"),
    ("gen", 90, 200, 17, 2, 32, 1, "mixed"),
    ("i4h", 640, 512, 33, 3, 33, 2, "0"),          # 33 rows of one slot: tiles of 16, 16 and 1
    ("fp4", 516, 260, 64, 8, 64, 1, "runs"),
    ("i4h", 513, 259, 65, 8, 70, 0, "runs"),       # beyond the ballot: listed rows
    ("i4h", 256, 1024, 200, 5, 9, 2, "mixed"),
    ("fp4", 130, 384, 257, 1, 256, 1, "0"),
    ("i4h", 128, 128, 1000, 600, 4, 2, "mixed"),   # more slots than the sort has threads
    ("i4h", 96, 2050, 130, 4, 128, 0, "-1"),       # no row has an adapter
    ("gen", 70, 120, 90, 3, 12, 0, "mixed"),
]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s)))
def test_forward(session, shape):
    with Case(session, 100 + SHAPES.index(shape), *shape) as c:
        c.check_forward()


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s)))
def test_gradients(session, shape):
    with Case(session, 200 + SHAPES.index(shape), *shape) as c:
        c.check_grads(want_dx=SHAPES.index(shape) % 4 != 3)


@pytest.mark.parametrize("pin", ["few", "many"])
@pytest.mark.parametrize("shape", [("i4h", 200, 300, 40, 3, 16, 1, "mixed"), ("fp4", 515, 260, 150, 4, 24, 2, "runs"),
                                   ("i4f", 300, 129, 300, 2, 70, 0, "mixed"),
                                   ("i4h", 130, 140, 400, 600, 4, 2, "mixed")], ids=lambda s: "-".join(map(str, s)))
def test_gradients_with_either_product(session, monkeypatch, shape, pin):
    monkeypatch.setenv("COLI_HIP_GEMM_T", pin)
    with Case(session, 300 + shape[3], *shape) as c:
        c.check_grads()


def test_rows_without_an_adapter_keep_the_projection(session):
    """Slots outside the bank or empty: bitwise coli_cuda_pipe_gemm."""
    for S in (7, 90):
        with Case(session, 31, "i4h", 160, 256, S, 4, 8, 1, "mixed") as c:
            got = c.check_forward()
            px, py = c.d.up(c.x), c.d.up(np.zeros((S, c.O), np.float32))
            assert c.b.cuda_pipe_gemm(c.h, py, px, S)
            plain = c.d.down(py, (S, c.O))
            none = np.isin(c.slot, [s for s in range(4) if c.ranks[s]], invert=True)
            assert none.any() and np.array_equal(got[none].view(np.uint32), plain[none].view(np.uint32))


def test_forward_repeats_bitwise(session):
    with Case(session, 32, "fp4", 192, 320, 200, 3, 16, 2, "mixed") as c:
        d, S, O = c.d, c.S, c.O
        px, ps = d.up(c.x), d.up(c.slot)
        py = d.up(np.zeros((S, O), np.float32))
        assert c.b.hip_lora_gemm_dev(c.h, c.bank, py, px, S, ps)
        whole = d.down(py, (S, O))
        again = d.up(np.zeros((S, O), np.float32))
        assert c.b.hip_lora_gemm_dev(c.h, c.bank, again, px, S, ps)
        assert np.array_equal(whole.view(np.uint32), d.down(again, (S, O)).view(np.uint32))

def test_gradients_repeat_bitwise(session):
    with Case(session, 33, "i4h", 144, 272, 300, 3, 24, 1, "mixed") as c:
        one, two = c.check_grads(), c.check_grads()
        for u, v in zip(one, two):
            assert np.array_equal(u.view(np.uint32), v.view(np.uint32))


def test_replaced_and_emptied_slots(session):
    """A smaller adapter over a larger one leaves nothing of it; rank 0 empties the slot."""
    rng = np.random.default_rng(6)
    with Case(session, 34, "i4h", 80, 96, 20, 2, 40, 1, "0", ranks=[40, 7]) as c:
        c.check_forward()
        c.set(0, rng.standard_normal((3, 96)), rng.standard_normal((80, 3)), 2.0, 1)
        c.check_forward()
        c.check_grads()
        assert c.b.hip_lora_set_dev(c.bank, 0, None, None, 0, 1.0)
        c.a[0], c.bm[0], c.sc[0] = 0, 0, 0
        c.check_forward()
        c.check_grads()


def test_infinite_rows_stay_apart(session):
    """A row of infinities or NaN does not reach rows of the same tile, nor (without an adapter) any gradient."""
    with Case(session, 35, "i4h", 64, 128, 30, 2, 5, 0, "0", ranks=[5, 2]) as c:
        c.slot[3] = c.slot[9] = -1
        clean_x, clean_dy = c.x.copy(), c.dy.copy()
        c.x[3, 4], c.x[9], c.dy[3, 1], c.dy[9] = np.inf, np.nan, np.inf, np.nan
        d = c.d
        px, pdy, ps = d.up(c.x), d.up(c.dy), d.up(c.slot)
        py, pdx = d.up(np.zeros((30, 64), np.float32)), d.up(np.zeros((30, 128), np.float32))
        pda, pdb = d.up(np.zeros((2, 5, 128), np.float32)), d.up(np.zeros((2, 64, 5), np.float32))
        assert c.b.hip_lora_gemm_dev(c.h, c.bank, py, px, 30, ps)
        assert c.b.hip_lora_grad_dev(c.h, c.bank, px, pdy, 30, ps, pdx, pda, pdb)
        y, dx, da, db = d.down(py, (30, 64)), d.down(pdx, (30, 128)), d.down(pda, (2, 5, 128)), d.down(pdb, (2, 64, 5))
        keep = [r for r in range(30) if r not in (3, 9)]
        assert np.isfinite(y[keep]).all() and np.isfinite(dx[keep]).all()
        assert np.isfinite(da).all() and np.isfinite(db).all()
        c.x, c.dy = clean_x, clean_dy
        cdx, cda, cdb = c.check_grads()
        assert np.array_equal(da, cda) and np.array_equal(db, cdb) and np.array_equal(dx[keep], cdx[keep])


def test_gradients_against_differences(session):
    """The gradients are those of the forward call itself: central differences of L = <y, dy>.

    y is linear in x, in A and in B, so a difference over any step is the
    derivative but for roundings: both y's errors over the step, 2 gemm_tol
    (and the adapters' sum_tol) of the magnitudes."""
    with Case(session, 36, "i4h", 48, 64, 9, 2, 4, 0, "0", ranks=[4, 2]) as c:
        dx, da, db = (v.astype(np.float64) for v in c.check_grads())
        d = c.d
        ps = d.up(c.slot)

        def loss():
            px, py = d.up(c.x), d.up(np.zeros((9, 48), np.float32))
            assert c.b.hip_lora_gemm_dev(c.h, c.bank, py, px, 9, ps)
            return float((d.down(py, (9, 48)).astype(np.float64) * c.dy).sum())

        x = c.x.astype(np.float64)
        mag = ((np.abs(x) @ np.abs(c.w).T + c.delta(x, c.a, c.bm, np.abs)) * np.abs(c.dy)).sum()
        tol = 4 * (gemm_tol(64) + sum_tol(64 + 4)) * mag
        for s, i in ((0, 0), (4, 63), (8, 17)):
            keep = c.x[s, i]
            c.x[s, i] = keep + 1.0
            up, hi = loss(), float(c.x[s, i])
            c.x[s, i] = keep - 1.0
            dn, lo = loss(), float(c.x[s, i])
            c.x[s, i] = keep
            assert abs((up - dn) / (hi - lo) - dx[s, i]) <= tol
        a0, b0 = c.a[0].copy(), c.bm[0].copy()
        for r, i in ((0, 0), (3, 40)):
            vals = []
            for sgn in (1, -1):
                a = a0.copy()
                a[r, i] += sgn
                c.set(0, a, b0, 0.5, 0)
                vals.append((loss(), c.a[0, r, i]))
            assert abs((vals[0][0] - vals[1][0]) / (vals[0][1] - vals[1][1]) - da[0, r, i]) <= 2 * tol
        for o, r in ((0, 0), (47, 3)):
            vals = []
            for sgn in (1, -1):
                bm = b0.copy()
                bm[o, r] += sgn
                c.set(0, a0, bm, 0.5, 0)
                vals.append((loss(), c.bm[0, o, r]))
            assert abs((vals[0][0] - vals[1][0]) / (vals[0][1] - vals[1][1]) - db[0, o, r]) <= 2 * tol


def test_unaligned_rows(session):
    with Case(session, 37, "i4h", 64, 128, 20, 2, 6, 1, "mixed") as c:
        d = c.d
        pad = np.zeros(1, np.float32)
        px, py = d.up(np.concatenate((pad, c.x.ravel()))), d.up(np.zeros(20 * 64 + 1, np.float32))
        assert c.b.hip_lora_gemm_dev(c.h, c.bank, py + 4, px + 4, 20, d.up(c.slot))
        got = d.down(py, (20 * 64 + 1,))[1:].reshape(20, 64)
        x = c.x.astype(np.float64)
        close(got, x @ c.w.T + c.delta(x, c.a, c.bm), np.abs(x) @ np.abs(c.w).T * gemm_tol(128) +
              c.delta(x, c.a, c.bm, np.abs) * sum_tol(128 + 6), 1.0)


@pytest.mark.parametrize("S", [5, 150])
def test_graph_replays(session, S):
    """A captured step (set, forward, gradients) replayed with other work between, against the eager result."""
    b = session.b
    with Case(session, 38 + S, "fp4", 256, 384, S, 3, 16, 2, "mixed") as c, \
            Case(session, 39, "i4h", 320, 512, 700, 4, 32, 1, "mixed") as o:
        d = c.d
        px, pdy, ps = d.up(c.x), d.up(c.dy), d.up(c.slot)
        sizes = {"y": (S, 256), "dx": (S, 384), "da": (3, 16, 384), "db": (3, 256, 16)}
        out = {k: d.up(np.zeros(v, np.float32)) for k, v in sizes.items()}
        rng = np.random.default_rng(2)
        pa, pb = d.up(bits(2, rng.standard_normal((16, 384)))[0]), d.up(bits(2, rng.standard_normal((256, 16)))[0])

        def step():
            assert b.hip_lora_set_dev(c.bank, 1, pa, pb, 16, 0.25)
            assert b.hip_lora_gemm_dev(c.h, c.bank, out["y"], px, S, ps)
            assert b.hip_lora_grad_dev(c.h, c.bank, px, pdy, S, ps, out["dx"], out["da"], out["db"])

        step()
        eager = {k: d.down(out[k], v) for k, v in sizes.items()}
        with hiprt.Graph(b.hip_stream(0)) as g:
            step()
        for rep in range(3):
            for k, v in sizes.items():
                assert b.hip_fill_random_u8(0, out[k], int(np.prod(v)) * 4, 3 + rep)
            g.launch()
            for k, v in sizes.items():
                got = d.down(out[k], v)
                assert np.array_equal(got.view(np.uint32), eager[k].view(np.uint32)), (rep, k)
            if rep == 0:
                o.check_forward()
                o.check_grads()


def test_graph_outlives_larger_products(session):
    """A captured forward and backward after larger eager calls of the same
    storage kind, which outgrow every buffer that the captured launches hold
    (row operands, partial sums of GEMV and GEMM, counters, adapter rows)."""
    b = session.b
    with Case(session, 45, "i4h", 304, 640, 90, 3, 16, 1, "mixed") as c, \
            Case(session, 46, "i4h", 256, 8192, 6, 3, 16, 1, "mixed") as few, \
            Case(session, 47, "i4h", 2048, 2304, 1500, 5, 48, 1, "mixed") as o:
        d, outs = c.d, []
        graphs = []
        for k in (few, c):
            px, pdy, ps = k.d.up(k.x), k.d.up(k.dy), k.d.up(k.slot)
            py, pdx = k.d.up(np.zeros((k.S, k.O), np.float32)), k.d.up(np.zeros((k.S, k.I), np.float32))
            pda, pdb = k.d.up(np.zeros((3, 16, k.I), np.float32)), k.d.up(np.zeros((3, k.O, 16), np.float32))

            def step():
                assert b.hip_lora_gemm_dev(k.h, k.bank, py, px, k.S, ps)
                assert b.hip_lora_grad_dev(k.h, k.bank, px, pdy, k.S, ps, pdx, pda, pdb)

            step()
            sizes = ((py, (k.S, k.O)), (pdx, (k.S, k.I)), (pda, (3, 16, k.I)), (pdb, (3, k.O, 16)))
            eager = [d.down(p, n) for p, n in sizes]
            with hiprt.Graph(b.hip_stream(0)) as g:
                step()
            graphs.append((g, sizes, eager))
        o.check_forward()
        o.check_grads()
        outs = [o.d.up(np.zeros((1500, 2048), np.float32)) for _ in range(4)]
        for rep in range(3):
            for g, sizes, eager in graphs:
                for p, n in sizes:
                    assert b.hip_fill_random_u8(0, p, int(np.prod(n)) * 4, 7 + rep)
                g.launch()
                for (p, n), want in zip(sizes, eager):
                    assert np.array_equal(d.down(p, n).view(np.uint32), want.view(np.uint32)), (rep, n)
            px = outs[rep]
            assert b.cuda_pipe_gemm(o.h, px, o.d.up(o.x), 1500 - rep)


def test_two_projections_in_sequence(session):
    """A two-layer feed-forward with adapters on both projections, forward and backward in one queue."""
    b = session.b
    with Case(session, 41, "i4h", 256, 128, 40, 3, 8, 1, "runs") as u, \
            Case(session, 42, "fp4", 128, 256, 40, 3, 8, 1, "runs") as v, Bufs(b) as d:
        v.slot = u.slot
        S = 40
        px, ps, pdy = d.up(u.x), d.up(u.slot), d.up(v.dy)
        ph, py = d.up(np.zeros((S, 256), np.float32)), d.up(np.zeros((S, 128), np.float32))
        pdh, pdx = d.up(np.zeros((S, 256), np.float32)), d.up(np.zeros((S, 128), np.float32))
        g = [d.up(np.zeros(n, np.float32)) for n in ((3, 8, 128), (3, 256, 8), (3, 8, 256), (3, 128, 8))]
        assert b.hip_lora_gemm_dev(u.h, u.bank, ph, px, S, ps)
        assert b.hip_lora_gemm_dev(v.h, v.bank, py, ph, S, ps)
        assert b.hip_lora_grad_dev(v.h, v.bank, ph, pdy, S, ps, pdh, g[2], g[3])
        assert b.hip_lora_grad_dev(u.h, u.bank, px, pdh, S, ps, pdx, g[0], g[1])
        x, dy = u.x.astype(np.float64), v.dy.astype(np.float64)
        ax = np.abs(x)

        def eff(c, s, f):
            return f(c.w) + (c.sc[s] * f(c.bm[s]) @ f(c.a[s]) if 0 <= s < 3 else 0)

        tol = gemm_tol(128) + gemm_tol(256) + 2 * sum_tol(300)
        y, dx = d.down(py, (S, 128)), d.down(pdx, (S, 128))
        for r in range(S):
            s = int(u.slot[r])
            wu, wv, au, av = (eff(c, s, f) for f in (lambda m: m, np.abs) for c in (u, v))
            close(y[r], wv @ (wu @ x[r]), av @ (au @ ax[r]), tol, r)
            close(dx[r], (dy[r] @ wv) @ wu, (np.abs(dy[r]) @ av) @ au, tol, r)


def test_refusals(session):
    b = session.b
    bank = C.c_void_p()
    for args in ((0, 3, 8, 1, 1, 0), (0, 8, 3, 1, 1, 0), (0, (1 << 20) + 1, 8, 1, 1, 0), (0, 8, (1 << 20) + 1, 1, 1, 0), (0, 8, 8, 0, 1, 0), (0, 8, 8, 1025, 1, 0), (0, 8, 8, 1, 0, 0),
                 (0, 8, 8, 1, 257, 0), (0, 8, 8, 1, 1, 3), (0, 8, 8, 1, 1, -1), (9, 8, 8, 1, 1, 0)):
        assert not b.hip_lora_create(C.byref(bank), *args) and not bank
    with Case(session, 50, "i4h", 32, 64, 4, 2, 4, 0, "0") as c, Case(session, 51, "i4h", 64, 32, 4, 2, 4, 0, "0") as o:
        d = c.d
        px, py, ps = d.up(c.x), d.up(c.dy), d.up(c.slot)
        pa, pb, pdx = (d.up(np.zeros(n, np.float32)) for n in ((2, 4, 64), (2, 32, 4), (4, 64)))
        ok = (c.h, c.bank, py, px, 4, ps)
        assert not c.b.hip_lora_gemm_dev(c.h, c.bank, px + 4 * 63, px, 4, ps)
        for k, bad in ((0, None), (1, None), (2, None), (3, None), (4, 0), (4, 65536), (5, None), (1, o.bank)):
            assert not b.hip_lora_gemm_dev(*(ok[:k] + (bad,) + ok[k + 1:])), (k, bad)
        ok = (c.h, c.bank, px, py, 4, ps, pdx, pa, pb)
        assert c.b.hip_lora_grad_dev(*ok)
        # a gradient over its inputs or over another one
        for k, bad in ((6, px), (6, py), (7, px), (8, py), (6, pa), (8, pa + 16)):
            assert not b.hip_lora_grad_dev(*(ok[:k] + (bad,) + ok[k + 1:])), (k, bad)
        for k, bad in ((0, None), (1, None), (2, None), (3, None), (4, 0), (5, None), (7, None), (8, None), (1, o.bank)):
            assert not b.hip_lora_grad_dev(*(ok[:k] + (bad,) + ok[k + 1:])), (k, bad)
        for slot, a, bb, r in ((-1, pa, pb, 1), (2, pa, pb, 1), (0, None, pb, 1), (0, pa, None, 1), (0, pa, pb, 5),
                               (0, pa, pb, -1)):
            assert not b.hip_lora_set_dev(c.bank, slot, a, bb, r, 1.0)
        assert not b.hip_lora_set_dev(None, 0, pa, pb, 1, 1.0)
    b.hip_lora_free(None)


def test_fault_injection(session, monkeypatch):
    with Case(session, 52, "i4h", 32, 64, 4, 2, 4, 0, "0") as c:
        d = c.d
        px, py, ps = d.up(c.x), d.up(np.full((4, 32), 7.0, np.float32)), d.up(c.slot)
        monkeypatch.setenv("COLI_GPU_FAIL_AFTER", "0")
        assert not c.b.hip_lora_gemm_dev(c.h, c.bank, py, px, 4, ps)
        assert not c.b.hip_gemm_t_dev(c.h, px, py, 4)
        monkeypatch.delenv("COLI_GPU_FAIL_AFTER")
        assert (d.down(py, (4, 32)) == 7.0).all()
        c.check_forward()


HIGH_RANK = [  # bf16 factors split beside four rank tiles, eight waves a workgroup; rows of more than 2048 columns
    ("i4h", 300, 2333, 130, 4, 64, 2, "mixed"),
    ("fp4", 260, 2304, 120, 3, 70, 2, "runs"),
    ("i4h", 2051, 330, 100, 3, 64, 2, "mixed"),
    ("fp4", 4100, 260, 70, 2, 70, 1, "mixed"),
]


@pytest.mark.parametrize("shape", HIGH_RANK, ids=lambda s: "-".join(map(str, s)))
def test_high_ranks_of_many_rows(session, monkeypatch, shape):
    with Case(session, 400 + HIGH_RANK.index(shape), *shape) as c:
        c.check_forward()
        c.check_grads()
        monkeypatch.setenv("COLI_HIP_GEMM_T", "many")   # (the sort builds dy's operands)
        c.check_grads()


def test_outputs_over_the_slots_are_refused(session):
    """The rows' slots are read by the last launch too."""
    b = session.b
    with Case(session, 53, "i4h", 32, 64, 20, 2, 4, 0, "0") as c:
        d = c.d
        px, py, ps = d.up(c.x), d.up(c.dy), d.up(c.slot)
        pa, pb, pdx = (d.up(np.zeros(n, np.float32)) for n in ((2, 4, 64), (2, 32, 4), (20, 64)))
        for bad in (ps, ps + 4 * 19, ps - 4 * 20 * 32 + 4):
            assert not b.hip_lora_gemm_dev(c.h, c.bank, bad, px, 20, ps)
        ok = (c.h, c.bank, px, py, 20, ps, pdx, pa, pb)
        for k, size in ((6, 4 * 20 * 64), (7, 4 * 2 * 4 * 64), (8, 4 * 2 * 32 * 4)):
            for bad in (ps, ps + 4 * 19, ps - size + 4):
                assert not b.hip_lora_grad_dev(*(ok[:k] + (bad,) + ok[k + 1:])), (k, bad)
        assert b.hip_lora_grad_dev(*ok) and b.hip_lora_gemm_dev(c.h, c.bank, py, px, 20, ps)
