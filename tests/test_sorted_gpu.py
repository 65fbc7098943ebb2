"""Rows sorted by expert and back (coli_hip_dispatch_dev, coli_hip_combine_dev,
coli_hip_combine_grad_dev) against 64-bit references."""
import numpy as np
import pytest

from colibri_amd import hiprt
from mx_ref import combine, plan
from op_util import Bufs, bits

pytestmark = pytest.mark.gpu

EPS = {0: 2.0 ** -24, 1: 2.0 ** -11, 2: 2.0 ** -8}   # half a step, relative
TINY = {0: 2.0 ** -149, 1: 2.0 ** -24, 2: 2.0 ** -133}


def values(dtype, raw):
    if dtype == 2:
        return (raw.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return raw.astype(np.float64)


def np_type(dtype):
    return (np.float32, np.float16, np.uint16)[dtype]


def routing(rng, T, E, K, keff=True, mask=True, outside=True):
    idx = rng.integers(0, E, (T, K)).astype(np.int32)
    if outside:
        idx[rng.random((T, K)) < 0.05] = rng.choice([-1, E, 2 ** 31 - 1, -2 ** 31])
    return (idx, rng.integers(0, K + 1, T).astype(np.int32) if keff else None,
            (rng.random(T) >= 0.2).astype(np.uint8) if mask else None)


def dispatch(b, idx, keff, mask, E, x, extra=2):
    """The call over buffers with guards behind them: (offsets, src, pos, xs) as they come back."""
    T, K = idx.shape
    with Bufs(b) as d:
        off, src = d.up(np.full(E + 1 + extra, 77, np.int32)), d.up(np.full(T * K + extra, 77, np.int32))
        pos = d.up(np.full(T * K + extra, 77, np.int32))
        px = xs = None
        rb = 0
        if x is not None:
            rb = x.shape[1]
            px, xs = d.up(x), d.up(np.full((T * K + extra, rb), 0x5A, np.uint8))
        opt = [None if v is None else d.up(v) for v in (keff, mask)]
        assert b.hip_dispatch_dev(0, d.up(idx), *opt, T, E, K, px, rb, off, src, pos, xs)
        return (d.down(off, E + 1 + extra, np.int32), d.down(src, T * K + extra, np.int32),
                d.down(pos, T * K + extra, np.int32), None if x is None else d.down(xs, (T * K + extra, rb), np.uint8))


def check_dispatch(b, idx, keff, mask, E, x):
    T, K = idx.shape
    off, src, pos, xs = dispatch(b, idx, keff, mask, E, x)
    ro, rs, rp = plan(idx, keff, mask, E)
    n = len(rs)
    assert np.array_equal(off[:E + 1], ro) and (off[E + 1:] == 77).all()
    assert np.array_equal(src[:n], rs) and (src[n:] == 77).all()
    assert np.array_equal(pos[:T * K].reshape(T, K), rp) and (pos[T * K:] == 77).all()
    if x is not None:
        assert np.array_equal(xs[:n], x[rs // K]) and (xs[n:] == 0x5A).all()


# one launch up to 4096 selections, three beyond; widths below, at and around 16
# bytes and a workgroup's piece of 4096
@pytest.mark.parametrize("T,E,K,rb", [(1, 1, 1, 1), (1, 64, 8, 8192), (3, 5, 2, 15), (7, 3, 6, 16), (16, 256, 8, 17),
                                      (33, 100, 6, 1998), (256, 256, 8, 4096), (1000, 17, 2, 4097), (2048, 9, 1, 31),
                                      (2049, 9, 1, 33), (257, 1024, 8, 100), (512, 1024, 8, 33), (4096, 3, 1, 20), (4097, 3, 1, 20), (586, 64, 7, 300),
                                      (65, 64, 63, 8), (513, 1024, 8, 20), (683, 8, 3, 4111), (5000, 64, 8, 48),
                                      (64, 64, 64, 9), (20000, 1000, 6, 2), (40000, 256, 8, 4)])
def test_dispatch(session, T, E, K, rb):
    rng = np.random.default_rng(T * 3 + E * 5 + K)
    x = rng.integers(0, 256, (T, rb)).astype(np.uint8)
    check_dispatch(session.b, *routing(rng, T, E, K), E, x)


@pytest.mark.parametrize("T", [40, 3000])
@pytest.mark.parametrize("keff,mask", [(False, False), (True, False), (False, True)])
def test_dispatch_without_choice_or_mask(session, T, keff, mask):
    rng = np.random.default_rng(T + keff)
    idx, k, m = routing(rng, T, 30, 4, keff, mask, False)
    check_dispatch(session.b, idx, k, m, 30, rng.integers(0, 256, (T, 40)).astype(np.uint8))
    check_dispatch(session.b, idx, k, m, 30, None)


@pytest.mark.parametrize("T", [50, 5000])
def test_dispatch_extremes(session, T):
    """Nothing live, all to one expert, a row that selects an expert twice, choices past K and below 0."""
    rng = np.random.default_rng(T)
    x = rng.integers(0, 256, (T, 20)).astype(np.uint8)
    z = np.zeros((T, 4), np.int32)
    check_dispatch(session.b, z, None, np.zeros(T, np.uint8), 10, x)
    check_dispatch(session.b, z, np.zeros(T, np.int32), None, 10, x)
    check_dispatch(session.b, z + 9, None, None, 10, x)
    check_dispatch(session.b, z + np.array([3, 1, 3, 3], np.int32), None, None, 10, x)
    check_dispatch(session.b, z + 2, rng.choice([-5, 2, 99], T).astype(np.int32), None, 10, x)


def test_dispatch_many_workgroups(session):
    """More selections than 256 workgroups of 4096: runs get longer."""
    rng = np.random.default_rng(8)
    T, E, K = 400_000, 33, 3
    idx = rng.integers(-1, E, (T, K)).astype(np.int32)
    key = np.where(idx < 0, E, idx).ravel()
    order = np.argsort(key, kind="stable").astype(np.int32)
    n = int((key < E).sum())
    off, src, pos, _ = dispatch(session.b, idx, None, None, E, None)
    assert np.array_equal(off[:E + 1], np.searchsorted(key[order], np.arange(E + 1)).astype(np.int32))
    assert np.array_equal(src[:n], order[:n])
    want = np.full(T * K, -1, np.int32)
    want[order[:n]] = np.arange(n)
    assert np.array_equal(pos[:T * K], want)


@pytest.mark.parametrize("T,E,K", [(5000, 1, 1), (9000, 1, 2), (5000, 2, 1), (3000, 2, 3)])
def test_dispatch_to_one_or_two_experts(session, T, E, K):
    """Many selections of few experts: hundreds of threads add up one expert's counts."""
    rng = np.random.default_rng(T + E + K)
    check_dispatch(session.b, *routing(rng, T, E, K), E, rng.integers(0, 256, (T, 20)).astype(np.uint8))
    check_dispatch(session.b, *routing(rng, T, E, K, False, False, False), E, None)


# past 256 workgroups of 1024 selections, where runs get longer, and past the 2^26 that are divided by a product
@pytest.mark.parametrize("T,E,K", [(87400, 33, 3), (7_500_000, 100, 9)])
def test_dispatch_of_long_runs(session, T, E, K):
    rng = np.random.default_rng(K)
    idx = rng.integers(-1, E, (T, K), dtype=np.int32)
    mask = (rng.random(T) >= 0.1).astype(np.uint8)
    off, src, pos, _ = dispatch(session.b, idx, None, mask, E, None)
    key = np.where(mask[:, None] != 0, idx, -1).ravel()
    counts = np.bincount(key + 1, minlength=E + 1)[1:]
    n = int(counts.sum())
    assert np.array_equal(off[:E + 1], np.concatenate([[0], np.cumsum(counts)])) and (off[E + 1:] == 77).all()
    # by expert, ascending within one, each live selection once
    assert np.array_equal(key[src[:n]], np.repeat(np.arange(E, dtype=np.int32), counts)) and (src[n:] == 77).all()
    up = np.diff(src[:n]) > 0
    up[off[1:E][(off[1:E] > 0) & (off[1:E] < n)] - 1] = True
    assert up.all()
    pos = pos[:T * K]
    assert np.array_equal(pos[src[:n]], np.arange(n, dtype=np.int32)) and ((pos >= 0) == (key >= 0)).all() and pos.min() == -1


@pytest.mark.parametrize("T", [60, 1500])
def test_dispatch_at_any_address(session, T):
    """Buffers that start off 16 bytes: the rows at any byte, the rest at any four (the mask at any)."""
    rng = np.random.default_rng(T)
    b, (E, K, rb) = session.b, (20, 4, 4111)
    idx, keff, mask = routing(rng, T, E, K)
    x = rng.integers(0, 256, (T, rb)).astype(np.uint8)
    ro, rs, rp = plan(idx, keff, mask, E)
    n = len(rs)

    def at(d, a, shift):
        p = d.up(np.full(a.nbytes + 32, 0x5A, np.uint8))
        d.put(p + shift, a)
        return p + shift

    for shift in (1, 7, 15):
        with Bufs(b) as d:
            i4 = [at(d, v, 4 * (1 + (shift + k) % 3)) for k, v in enumerate((idx, keff, np.full(E + 1, 77, np.int32), np.full(T * K, 77, np.int32),
                                                                          np.full(T * K, 77, np.int32)))]
            xs = at(d, np.full((T * K, rb), 0x5A, np.uint8), 16 - shift)
            assert b.hip_dispatch_dev(0, i4[0], i4[1], at(d, mask, shift), T, E, K, at(d, x, shift), rb, *i4[2:], xs)
            assert np.array_equal(d.down(i4[2], E + 1, np.int32), ro) and np.array_equal(d.down(i4[4], (T, K), np.int32), rp)
            src, got = d.down(i4[3], T * K, np.int32), d.down(xs, (T * K, rb), np.uint8)
            assert np.array_equal(src[:n], rs) and (src[n:] == 77).all()
            assert np.array_equal(got[:n], x[rs // K]) and (got[n:] == 0x5A).all()
            assert (d.down(xs + T * K * rb, shift, np.uint8) == 0x5A).all()


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("T,E,K,D", [(33, 100, 6, 999), (16, 16, 8, 1024)])
def test_combine_at_any_address(session, dtype, T, E, K, D):
    """Buffers that start at any element: the bits of those that start at 16 bytes, and nothing beside them written."""
    rng = np.random.default_rng(D + dtype)
    b = session.b
    pos, N, ys, _, dout, _, w = sorted_case(rng, dtype, T, E, K, D)
    es = ys.itemsize
    res = []
    for el in (0, 1, 3):
        with Bufs(b) as d:
            def at(a, step):
                p = d.up(np.full(a.nbytes + 32, 7, np.uint8))
                d.put(p + el * step, a)
                return p + el * step

            py, pd, pp, pw = at(ys, es), at(dout, es), at(pos, 4), at(w, 4)
            out, dys, dw = at(np.zeros((T, D), ys.dtype), es), at(np.zeros((N, D), ys.dtype), es), at(np.zeros((T, K), np.float32), 4)
            assert b.hip_combine_dev(0, py, dtype, pp, pw, T, K, N, D, out)
            assert b.hip_combine_grad_dev(0, py, dtype, pp, pw, pd, T, K, N, D, dys, dw)
            res.append([d.down(p, n, np.uint8) for p, n in ((out, T * D * es), (dys, N * D * es), (dw, T * K * 4))])
            for p, n in ((out, T * D * es), (dys, N * D * es), (dw, T * K * 4)):
                assert (d.down(p + n, 4, np.uint8) == 7).all()
                assert el == 0 or (d.down(p - 2, 2, np.uint8) == 7).all()
    for r in res[1:]:
        for a, c in zip(res[0], r):
            assert np.array_equal(a, c)


def test_dispatch_no_rows(session):
    b = session.b
    with Bufs(b) as d:
        off = d.up(np.full(8, 5, np.int32))
        assert b.hip_dispatch_dev(0, None, None, None, 0, 6, 2, None, 0, off, None, None, None)
        assert np.array_equal(d.down(off, 8, np.int32), [0] * 7 + [5])
        assert b.hip_combine_dev(0, None, 0, None, None, 0, 2, 0, 8, None)
        assert b.hip_combine_grad_dev(0, None, 0, None, None, None, 0, 2, 0, 8, off, None)
        # rows, but none sorted: zeros
        out = d.up(np.full((3, 5), 2.0, np.float32))
        pos = d.up(np.full((3, 2), -1, np.int32))
        assert b.hip_combine_dev(0, None, 0, pos, None, 3, 2, 0, 5, out)
        assert not d.down(out, (3, 5)).any()


def sorted_case(rng, dtype, T, E, K, D):
    idx, keff, mask = routing(rng, T, E, K)
    _, src, pos = plan(idx, keff, mask, E)
    N = max(1, len(src))
    ys, yv = bits(dtype, rng.standard_normal((N, D)))
    dout, dv = bits(dtype, rng.standard_normal((T, D)))
    w = rng.standard_normal((T, K)).astype(np.float32)
    return pos, N, ys, yv, dout, dv, w


SIZES = [(1, 4, 1, 1), (1, 64, 8, 2048), (3, 5, 2, 3), (9, 9, 6, 7), (16, 16, 8, 1024), (33, 100, 6, 999), (20, 8, 3, 4100),
         (130, 300, 5, 8), (7, 70, 64, 33), (50, 20, 9, 257), (6, 9, 2, 20000)]


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("T,E,K,D", SIZES)
def test_combine(session, dtype, T, E, K, D):
    """f32 sums of K products (a rounding each), and one rounding to the type."""
    rng = np.random.default_rng(T + E + K + D + dtype)
    b = session.b
    pos, N, ys, yv, _, _, w = sorted_case(rng, dtype, T, E, K, D)
    for ww in (w, None):
        with Bufs(b) as d:
            out = d.up(np.full((T + 1, D), 7, np_type(dtype)))
            assert b.hip_combine_dev(0, d.up(ys), dtype, d.up(pos), None if ww is None else d.up(ww), T, K, N, D, out)
            got = d.down(out, (T + 1, D), np_type(dtype))
        assert (got[T] == 7).all()
        ref, mag = combine(yv, pos, ww, N)
        err = np.abs(values(dtype, got[:T]) - ref)
        assert (err <= K * 2.0 ** -24 * mag + EPS[dtype] * 1.001 * np.abs(ref) + TINY[dtype]).all()


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("T,E,K,D", SIZES)
def test_combine_grad(session, dtype, T, E, K, D):
    """dys: one product, one rounding. dw: f32 sums over D, at most D / 64 + 8 additions a lane and 6 across."""
    rng = np.random.default_rng(T + E + K + D + dtype + 1)
    b = session.b
    pos, N, ys, yv, dout, dv, w = sorted_case(rng, dtype, T, E, K, D)
    live = np.argwhere(pos >= 0)
    for ww in (w, None):
        wv = np.ones((T, K)) if ww is None else w.astype(np.float64)
        with Bufs(b) as d:
            py, pp, pd = d.up(ys), d.up(pos), d.up(dout)
            pw = None if ww is None else d.up(ww)
            dys, dw = d.up(np.full((N + 1, D), 7, np_type(dtype))), d.up(np.full((T + 1, K), 7, np.float32))
            assert b.hip_combine_grad_dev(0, py, dtype, pp, pw, pd, T, K, N, D, dys, dw)
            gy, gw = d.down(dys, (N + 1, D), np_type(dtype)), d.down(dw, (T + 1, K))
            # either alone: the same bits
            one = d.up(np.full((N + 1, D), 7, np_type(dtype)))
            assert b.hip_combine_grad_dev(0, None, dtype, pp, pw, pd, T, K, N, D, one, None)
            assert np.array_equal(d.down(one, (N + 1, D), np_type(dtype)), gy)
            alone = d.up(np.full((T + 1, K), 7, np.float32))
            assert b.hip_combine_grad_dev(0, py, dtype, pp, pw, pd, T, K, N, D, None, alone)
            assert np.array_equal(d.down(alone, (T + 1, K)), gw)
        assert (gw[T] == 7).all() and not gw[:T][pos < 0].any()
        seen = np.zeros(N + 1, bool)
        for t, k in live:
            p = pos[t, k]
            seen[p] = True
            ref = wv[t, k] * dv[t]
            assert (np.abs(values(dtype, gy[p]) - ref) <= (2.0 ** -24 + EPS[dtype]) * 1.001 * np.abs(ref) + TINY[dtype]).all()
            terms = dv[t] * yv[p]
            tol = (D / 64 + 14 + 8) * 2.0 ** -24 * np.abs(terms).sum()
            assert abs(gw[t, k] - terms.sum()) <= tol
        assert (gy[~seen] == 7).all()


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("D", [5, 64, 999])
def test_combine_grad_keeps_the_sign_of_zero(session, dtype, D):
    """w dout of zeros of either sign, in every column."""
    b, (T, K) = session.b, (3, 2)
    v = np.where(np.indices((T, D)).sum(0) % 3 > 0, -0.0, 0.0)
    dout, _ = bits(dtype, v)
    w = np.array([[1, -1], [-0.5, 0.25], [2, 3]], np.float32)
    want, _ = bits(dtype, (v[:, None] * w[:, :, None]).reshape(T * K, D))
    with Bufs(b) as d:
        dys = d.up(np.full((T * K, D), 7, want.dtype))
        assert b.hip_combine_grad_dev(0, None, dtype, d.up(np.arange(T * K, dtype=np.int32)), d.up(w), d.up(dout), T, K, T * K, D, dys, None)
        assert np.array_equal(d.down(dys, want.nbytes, np.uint8), want.view(np.uint8).ravel())


def test_gradients_are_the_derivatives(session):
    """<dout, out> is linear in ys, in w, and (through dispatch) in x: the calls' own
    differences against the gradients, f32 roundings of both sides allowed for."""
    rng = np.random.default_rng(4)
    b, (T, E, K, D) = session.b, (19, 7, 3, 45)
    idx, keff, mask = routing(rng, T, E, K)
    x, w = rng.standard_normal((T, D)).astype(np.float32), rng.standard_normal((T, K)).astype(np.float32)
    dout = rng.standard_normal((T, D)).astype(np.float32)
    _, src, pos = plan(idx, keff, mask, E)
    N = T * K

    def loss(x, w):
        with Bufs(b) as d:
            xs, out = d.up(np.zeros((N, D), np.float32)), d.up(np.zeros((T, D), np.float32))
            off, ps, pp = d.up(np.zeros(E + 1, np.int32)), d.up(np.zeros(N, np.int32)), d.up(np.zeros(N, np.int32))
            assert b.hip_dispatch_dev(0, d.up(idx), d.up(keff), d.up(mask), T, E, K, d.up(x), D * 4, off, ps, pp, xs)
            assert b.hip_combine_dev(0, xs, 0, pp, d.up(w), T, K, N, D, out)
            return float((dout.astype(np.float64) * d.down(out, (T, D))).sum())

    with Bufs(b) as d:
        xs = np.zeros((N, D), np.float32)
        xs[:len(src)] = x[src // K]
        dys, dw, dx = d.up(np.zeros((N, D), np.float32)), d.up(np.zeros((T, K), np.float32)), d.up(np.zeros((T, D), np.float32))
        pp = d.up(pos)
        assert b.hip_combine_grad_dev(0, d.up(xs), 0, pp, d.up(w), d.up(dout), T, K, N, D, dys, dw)
        assert b.hip_combine_dev(0, dys, 0, pp, None, T, K, N, D, dx)
        gw, gx = d.down(dw, (T, K)).astype(np.float64), d.down(dx, (T, D)).astype(np.float64)
    for _ in range(4):
        u, v = rng.standard_normal((T, D)).astype(np.float32), rng.standard_normal((T, K)).astype(np.float32)
        # steps of 1: each side's sum of T D K terms of order 1..10 with roundings of 2^-23 each
        room = 2.0 ** -22 * 16 * T * D * K
        assert abs((loss(x + u, w) - loss(x - u, w)) / 2 - (gx * u).sum()) <= room
        assert abs((loss(x, w + v) - loss(x, w - v)) / 2 - (gw * v).sum()) <= room


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_values_that_no_place_names(session, dtype):
    """Rows of NaN that no place names, weights of NaN on selections that are not live, places past the last row."""
    b, (T, K, N, D) = session.b, (5, 3, 6, 70)
    rng = np.random.default_rng(dtype)
    pos = np.array([[0, -1, 5], [9, 2, -7], [-1, -1, -1], [1, 6, 2 ** 31 - 1], [3, -1, -1]], np.int32)
    w = np.where((pos >= 0) & (pos < N), rng.standard_normal((T, K)), np.nan).astype(np.float32)
    v = rng.standard_normal((N, D))
    v[4] = np.nan
    ys, yv = bits(dtype, v)
    if dtype == 2:
        ys[4] = 0x7FC0
    dout, dv = bits(dtype, rng.standard_normal((T, D)))
    ref, mag = combine(np.where(np.isnan(yv), 0, yv), pos, w, N)
    with Bufs(b) as d:
        out, dys, dw = d.up(np.zeros((T, D), np_type(dtype))), d.up(np.full((N, D), 7, np_type(dtype))), d.up(np.zeros((T, K), np.float32))
        py, pp, pw = d.up(ys), d.up(pos), d.up(w)
        assert b.hip_combine_dev(0, py, dtype, pp, pw, T, K, N, D, out)
        got = values(dtype, d.down(out, (T, D), np_type(dtype)))
        assert b.hip_combine_grad_dev(0, py, dtype, pp, pw, d.up(dout), T, K, N, D, dys, dw)
        gy, gw = d.down(dys, (N, D), np_type(dtype)), d.down(dw, (T, K))
    assert (np.abs(got - ref) <= 3 * 2.0 ** -24 * mag + EPS[dtype] * 1.001 * np.abs(ref) + TINY[dtype]).all()
    assert not got[2].any() and (gy[4] == 7).all()
    live = (pos >= 0) & (pos < N)
    assert np.isfinite(gw).all() and not gw[~live].any()


def test_rounds_once_and_keeps_infinities(session):
    """fp16 sums past 65504 are infinities; f32 sums keep what two fp16 roundings would lose."""
    b = session.b
    ys = np.array([[60000, 1, np.inf, 1], [60000, 2.0 ** -11, 1, 0], [0, 2.0 ** -11, 1, 0]], np.float16)
    with Bufs(b) as d:
        out = d.up(np.zeros((1, 4), np.float16))
        assert b.hip_combine_dev(0, d.up(ys), 1, d.up(np.array([[0, 1, 2]], np.int32)), None, 1, 3, 3, 4, out)
        assert np.array_equal(d.down(out, (1, 4), np.float16), np.array([[np.inf, 1 + 2.0 ** -10, np.inf, 1]], np.float16))


def test_rows_past_the_caches(session):
    """Sorted rows of more than 128 MiB, which are stored and loaded past the caches: a sample of the
    rows against 64 bits, and every row's bytes in dispatch."""
    rng = np.random.default_rng(11)
    b, (T, E, K, D) = session.b, (2400, 40, 8, 3600)
    idx, keff, mask = routing(rng, T, E, K)
    off, src, pos = plan(idx, keff, mask, E)
    N = T * K
    x = rng.standard_normal((T, D)).astype(np.float16)
    w = rng.standard_normal((T, K)).astype(np.float32)
    with Bufs(b) as d:
        xs, out, dys = (d.up(np.full((n, D), 7, np.float16)) for n in (N, T, N))
        dw, pp, px, pw = d.up(np.full((T, K), 7, np.float32)), d.up(np.zeros(N, np.int32)), d.up(x), d.up(w)
        assert b.hip_dispatch_dev(0, d.up(idx), d.up(keff), d.up(mask), T, E, K, px, D * 2, d.up(off * 0), d.up(np.zeros(N, np.int32)), pp, xs)
        assert b.hip_combine_dev(0, xs, 1, pp, pw, T, K, N, D, out)
        assert b.hip_combine_grad_dev(0, xs, 1, pp, pw, px, T, K, N, D, dys, dw)
        got, go, gy, gw = d.down(xs, (N, D), np.float16), d.down(out, (T, D), np.float16), d.down(dys, (N, D), np.float16), d.down(dw, (T, K))
    n = len(src)
    assert np.array_equal(got[:n], x[src // K]) and (got[n:] == 7).all() and (gy[n:] == 7).all()
    xv = x.astype(np.float64)
    for t in range(0, T, 37):
        live = pos[t] >= 0
        wt = w[t].astype(np.float64)[live]
        ref, mag = wt.sum() * xv[t], np.abs(wt).sum() * np.abs(xv[t])
        assert (np.abs(go[t] - ref) <= K * 2.0 ** -24 * mag + EPS[1] * 1.001 * np.abs(ref) + TINY[1]).all()
        for k in np.flatnonzero(live):
            v = float(w[t, k]) * xv[t]
            assert (np.abs(gy[pos[t, k]] - v) <= (2.0 ** -24 + EPS[1]) * 1.001 * np.abs(v) + TINY[1]).all()
            assert abs(gw[t, k] - (xv[t] ** 2).sum()) <= (D / 64 + 22) * 2.0 ** -24 * (xv[t] ** 2).sum()
        assert not gw[t][~live].any()


def test_refusals(session):
    b = session.b
    with Bufs(b) as d:
        i32, f = d.up(np.zeros(64, np.int32)), d.up(np.zeros(256, np.float32))
        o = [d.up(np.zeros(256, np.float32)) for _ in range(4)]
        ok = (0, i32, None, None, 2, 4, 3, f, 8, o[0], o[1], o[2], o[3])

        def call(fn, args, **change):
            a = list(args)
            for k, v in change.items():
                a[int(k[1:])] = v
            return fn(*a)

        assert b.hip_dispatch_dev(*ok)
        big = 2 ** 31 - 1
        for ch in ({"_0": 1}, {"_0": -1}, {"_1": None}, {"_4": -1}, {"_4": (1 << 23) + 1}, {"_5": 0}, {"_5": 1025}, {"_6": 0}, {"_6": 65},
                   {"_7": None}, {"_12": None}, {"_8": 0}, {"_8": (64 << 20) + 1},
                   {"_9": None}, {"_10": None}, {"_11": None}, {"_9": i32}, {"_10": o[0]}, {"_11": o[1]}, {"_12": f}, {"_12": o[2]},
                   {"_2": o[0]}, {"_3": o[3]}, {"_4": big}):
            assert not call(b.hip_dispatch_dev, ok, **ch), ch
        ok = (0, f, 0, i32, o[0], 2, 3, 4, 5, o[1])
        assert b.hip_combine_dev(*ok)
        for ch in ({"_0": 3}, {"_1": None}, {"_2": 3}, {"_2": -1}, {"_3": None}, {"_5": -1}, {"_5": big}, {"_6": 0}, {"_6": 65}, {"_7": -1},
                   {"_8": 0}, {"_8": big}, {"_9": None}, {"_9": f}, {"_9": i32}, {"_9": o[0]}):
            assert not call(b.hip_combine_dev, ok, **ch), ch
        ok = (0, f, 0, i32, o[0], o[1], 2, 3, 4, 5, o[2], o[3])
        assert b.hip_combine_grad_dev(*ok)
        for ch in ({"_0": 3}, {"_1": None}, {"_2": 3}, {"_3": None}, {"_5": None}, {"_6": -1}, {"_7": 0}, {"_7": 65}, {"_8": -1}, {"_9": 0},
                   {"_10": None, "_11": None}, {"_10": f}, {"_10": o[1]}, {"_11": o[0]}, {"_11": i32}, {"_11": o[2]}):
            assert not call(b.hip_combine_grad_dev, ok, **ch), ch
        assert b.cuda_pipe_sync(0)


@pytest.mark.parametrize("T", [24, 900])
def test_graph_replays(session, T):
    """Dispatch, combine and the gradients captured, replayed over changing inputs
    with eager calls of other sizes between: the eager results each time."""
    b, (E, K, D) = session.b, (20, 4, 130)
    rng = np.random.default_rng(T)
    N = T * K
    with Bufs(b) as d:
        pi, px, pw = d.up(np.zeros((T, K), np.int32)), d.up(np.zeros((T, D), np.float32)), d.up(np.zeros((T, K), np.float32))
        outs = [[d.up(np.zeros(n, np.float32)) for n in (E + 1, N, N, N * D, T * D, N * D, N)] for _ in range(2)]

        def calls(o):
            assert b.hip_dispatch_dev(0, pi, None, None, T, E, K, px, D * 4, o[0], o[1], o[2], o[3])
            assert b.hip_combine_dev(0, o[3], 0, o[2], pw, T, K, N, D, o[4])
            assert b.hip_combine_grad_dev(0, o[3], 0, o[2], pw, px, T, K, N, D, o[5], o[6])

        calls(outs[0])
        with hiprt.Graph(b.hip_stream(0)) as g:
            calls(outs[0])
        for rep in range(3):
            for p, v in ((pi, rng.integers(-1, E, (T, K)).astype(np.int32)), (px, rng.standard_normal((T, D)).astype(np.float32)),
                         (pw, rng.standard_normal((T, K)).astype(np.float32))):
                d.put(p, v)
            for o in outs:   # what is left as it was, alike on both sides
                for p, n in zip(o, (E + 1, N, N, N * D, T * D, N * D, N)):
                    d.put(p, np.zeros(n, np.float32))
            g.launch()
            calls(outs[1])
            check_dispatch(b, *routing(rng, 2100 + rep, 12, 2 + rep), 12, None)
            for p, q, n in zip(*outs, (E + 1, N, N, N * D, T * D, N * D, N)):
                assert np.array_equal(d.down(p, n, np.uint32), d.down(q, n, np.uint32)), rep
