"""MXFP4 on the device: the quantizer and its way back, products of 4-bit rows with
one resident matrix and with the experts' over sorted rows, against 64-bit
references."""
import ctypes as C

import numpy as np
import pytest

from colibri_amd import hiprt
from colibri_amd.backend import f32p, tensor_array
from mx_ref import combine, mx_quant, pack, plan, silu
from op_util import Bufs, bits
from quant_util import deq_mxfp4, mx4_scale, rand_i4, rand_mxfp4, E2M1, nibbles

pytestmark = pytest.mark.gpu


def product_tol(I):
    """Products of codes and scales are exact; the sums are f32: ceil(I / 128) MFMAs
    that add 128 products to the running sum, and joins of at most 32 parts. Each is
    allowed two units in the last place of the terms' magnitudes (2 x 2^-23)."""
    return ((I + 127) // 128 + 32) * 2.0 ** -22


def act(rng, S, I):
    """Rows whose columns differ in size."""
    return (rng.standard_normal((S, I)) * np.exp(rng.standard_normal(I))).astype(np.float32)


def quantize(b, raw, dtype, extra=3):
    rows, cols = raw.shape
    qb, eb = rows * ((cols + 1) // 2), rows * ((cols + 31) // 32)
    with Bufs(b) as d:
        q4, e8 = d.up(np.full(qb + extra, 0xA5, np.uint8)), d.up(np.full(eb + extra, 0xA5, np.uint8))
        assert b.hip_mxfp4_quantize_dev(0, d.up(raw), dtype, rows, cols, q4, e8)
        q, e = d.down(q4, qb + extra, np.uint8), d.down(e8, eb + extra, np.uint8)
    assert (q[qb:] == 0xA5).all() and (e[eb:] == 0xA5).all()
    return q[:qb].reshape(rows, -1), e[:eb].reshape(rows, -1)


def check_quantize(b, x, dtype):
    raw, val = bits(dtype, x)
    q, e = quantize(b, raw, dtype)
    codes, byte, _ = mx_quant(val)
    assert np.array_equal(e, byte)
    bad = np.repeat(byte == 255, 32, 1)[:, :x.shape[1]]
    assert np.array_equal(q, pack(np.where(bad, 0, codes)))


# around a lane's elements (4 of f32, 8 of the others), a block (32), a lane's last ones, rows of
# one workgroup's step (1024 and 2048 columns) and beyond
@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (2, 3), (6, 4), (3, 5), (2, 7), (5, 8), (4, 9), (40, 12), (70, 31), (3, 32), (9, 33), (2, 63),
                                       (5, 100), (37, 999), (6, 1028), (300, 64), (3, 2048), (2, 2050), (2, 4111), (1, 16500), (1030, 6403)])
def test_quantize(session, dtype, rows, cols):
    rng = np.random.default_rng(rows * 7 + cols + dtype)
    check_quantize(session.b, rng.standard_normal((rows, cols)) * np.exp(2 * rng.standard_normal((rows, 1))), dtype)


def test_quantize_borders(session):
    """Every border between two codes and its neighbours, under every scale, both signs."""
    mids = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    f = np.float32
    near = np.concatenate([mids, np.nextafter(mids.astype(f), f(0)), np.nextafter(mids.astype(f), f(9)), [6.0, 0.0, -0.0]])
    row = np.concatenate([near, -near[:8]])
    assert len(row) == 32
    e = np.arange(1, 254)[:, None] - 127.0
    with np.errstate(under="ignore"):
        x = (row[None, :] * 2.0 ** e).astype(np.float32)
    check_quantize(session.b, x, 0)


def test_quantize_scale_borders(session):
    """A block's largest magnitude at 6 times a power of two and next to it, over the whole range of f32, subnormals too."""
    f = np.float32
    with np.errstate(over="ignore", under="ignore"):
        top = (1.5 * 2.0 ** np.arange(-149, 128)).astype(f)
        top = np.concatenate([top, np.nextafter(top, f(0)), np.nextafter(top, f(np.inf)), [f(2.0 ** -149), f(np.finfo(f).max), f(0)]])
    rng = np.random.default_rng(1)
    x = (rng.uniform(-1, 1, (len(top), 32)) * top[:, None].astype(np.float64)).astype(f)
    x[:, 5] = top
    check_quantize(session.b, x, 0)


def test_quantize_every_bf16_and_f16(session):
    rng = np.random.default_rng(2)
    u = rng.permutation(np.arange(65536).astype(np.uint16)).reshape(32, 2048)
    v = (u.astype(np.uint32) << 16).view(np.float32)
    q, e = quantize(session.b, u, 2)
    codes, byte, _ = mx_quant(v)
    assert np.array_equal(e, byte) and np.array_equal(q, pack(np.where(np.repeat(byte == 255, 32, 1), 0, codes)))
    # blocks of one exponent: no value is lost below its neighbours
    for dtype, raw, val in ((2, np.arange(65536).astype(np.uint16), None), (1, np.arange(65536).astype(np.uint16).view(np.float16), None)):
        raw = raw.reshape(64, 1024)
        val = (raw.astype(np.uint32) << 16).view(np.float32) if dtype == 2 else raw.astype(np.float32)
        q, e = quantize(session.b, raw, dtype)
        codes, byte, _ = mx_quant(val)
        assert np.array_equal(e, byte) and np.array_equal(q, pack(np.where(np.repeat(byte == 255, 32, 1), 0, codes)))


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (2, 6), (2, 7), (5, 8), (4, 9), (70, 31), (9, 33), (37, 999), (300, 64), (2, 2050), (1, 16500)])
def test_dequantize(session, dtype, rows, cols):
    """Codes times scales, one rounding: exact in f32 (2^-127 and up), to half a step in the others. Bytes 0 and 255 too."""
    rng = np.random.default_rng(rows + cols)
    q4, e8 = rand_mxfp4(rng, rows, cols, 100, 140)
    e8.reshape(-1)[::5] = rng.choice([0, 1, 2, 253, 254, 255], len(e8.reshape(-1)[::5]))
    with np.errstate(over="ignore", invalid="ignore"):
        sc = mx4_scale(e8)[:, np.arange(cols) // 32]
        ref = (E2M1[nibbles(q4, cols)] * sc).astype(np.float32)
        want, _ = bits(dtype, ref)
    with Bufs(session.b) as d:
        y = d.up(np.full(rows * cols + 2, 7, want.dtype))
        assert session.b.hip_mxfp4_dequantize_dev(0, d.up(q4), d.up(e8), rows, cols, y, dtype)
        got = d.down(y, rows * cols + 2, want.dtype)
    assert (got[-2:] == 7).all()
    got = got[:-2].reshape(rows, cols)
    if dtype == 2:
        got, want = ((v.astype(np.uint32) << 16).view(np.float32) for v in (got, want))
    nan = np.isnan(ref)
    assert np.array_equal(np.isnan(got), nan) and np.array_equal(got[~nan], want[~nan])


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("rows,cols", [(3, 32), (5, 257)])
def test_dequantize_keeps_the_sign_of_zero(session, dtype, rows, cols):
    """Code 8 is -0 under every scale but 255, in every column."""
    codes = (np.indices((rows, cols)).sum(0) % 3 > 0) * 8
    e8 = np.broadcast_to(np.array([0, 1, 127, 254, 90], np.uint8)[:rows, None], (rows, (cols + 31) // 32))
    want, _ = bits(dtype, np.where(codes == 8, -0.0, 0.0))
    with Bufs(session.b) as d:
        y = d.up(np.full((rows, cols), 7, want.dtype))
        assert session.b.hip_mxfp4_dequantize_dev(0, d.up(pack(codes)), d.up(e8), rows, cols, y, dtype)
        assert np.array_equal(d.down(y, want.nbytes, np.uint8), want.view(np.uint8).ravel())


@pytest.mark.parametrize("dtype", [1, 2])
def test_dequantize_past_the_caches(session, dtype):
    """More than 128 MiB of 16-bit output, stored past the caches, of an odd width."""
    rng = np.random.default_rng(dtype)
    rows, cols = 9001, 7501
    q4, e8 = rand_mxfp4(rng, rows, cols, 100, 140)
    with Bufs(session.b) as d:
        y = d.up(np.full(rows * cols + 2, 7, np.uint16))
        assert session.b.hip_mxfp4_dequantize_dev(0, d.up(q4), d.up(e8), rows, cols, y, dtype)
        got = d.down(y, rows * cols + 2, np.uint16)
    assert (got[-2:] == 7).all()
    r = np.append(np.arange(0, rows, 29), rows - 1)
    with np.errstate(over="ignore"):
        want, _ = bits(dtype, deq_mxfp4(q4[r], e8[r], cols))
    assert np.array_equal(got[:-2].reshape(rows, cols)[r], want.view(np.uint16))


def test_quantize_at_any_address(session):
    """Rows from any element on and bytes from any byte on: what aligned ones give."""
    b, (rows, cols) = session.b, (70, 999)
    rng = np.random.default_rng(15)
    for dtype in (0, 1, 2):
        raw, _ = bits(dtype, rng.standard_normal((rows, cols)))
        q, e = quantize(b, raw, dtype)
        for k in (1, 3):
            with Bufs(b) as d:
                x, q4, e8 = (d.up(np.full(n + 32, 0xA5, np.uint8)) + k * m for n, m in ((raw.nbytes, raw.itemsize), (q.nbytes, 1), (e.nbytes, 1)))
                d.put(x, raw)
                assert b.hip_mxfp4_quantize_dev(0, x, dtype, rows, cols, q4, e8)
                assert np.array_equal(d.down(q4, q.shape, np.uint8), q) and np.array_equal(d.down(e8, e.shape, np.uint8), e)
                ends = [p + n for p, n in ((q4, q.nbytes), (e8, e.nbytes))]
                y, y0 = (d.up(np.full(raw.nbytes + 32, 0xA5, np.uint8)) + n * raw.itemsize for n in (k, 0))
                assert b.hip_mxfp4_dequantize_dev(0, q4, e8, rows, cols, y, dtype)
                assert b.hip_mxfp4_dequantize_dev(0, d.up(q), d.up(e), rows, cols, y0, dtype)
                assert np.array_equal(d.down(y, raw.nbytes, np.uint8), d.down(y0, raw.nbytes, np.uint8))
                for p in (*ends, y + raw.nbytes):
                    assert (d.down(p, 4, np.uint8) == 0xA5).all()
                for p in (q4 - 1, e8 - 1, y - 1):
                    assert d.down(p, 1, np.uint8)[0] == 0xA5


def test_no_rows(session):
    assert session.b.hip_mxfp4_quantize_dev(0, None, 0, 0, 8, None, None)
    assert session.b.hip_mxfp4_dequantize_dev(0, None, None, 0, 8, None, 0)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("O,I", [(1, 1), (48, 130), (33, 999), (200, 512)])
def test_tensor_from_device_weights(session, dtype, O, I):
    """The resident tensor is the one that the quantizer's bytes upload to: bitwise the same products."""
    b = session.b
    rng = np.random.default_rng(O + I + dtype)
    raw, val = bits(dtype, rng.standard_normal((O, I)) * 0.05)
    codes, byte, w = mx_quant(val)
    h, ref = C.c_void_p(), session.upload_mxfp4(pack(codes), byte, I, O)
    try:
        with Bufs(b) as d:
            pw = d.up(raw)
            assert b.cuda_pipe_sync(0)
            assert b.hip_tensor_quantize_mxfp4(C.byref(h), pw, dtype, I, O, 0)
            assert not b.hip_tensor_quantize_mxfp4(C.byref(h), pw, dtype, I, O, 0)
        assert b.hip_tensor_kind(h) == 2 and b.cuda_tensor_bytes(h) == b.cuda_tensor_bytes(ref)
        x = rng.standard_normal((3, I)).astype(np.float32)
        assert np.array_equal(session.matmul(h, x, 7, I, O), session.matmul(ref, x, 7, I, O))
    finally:
        session.free(ref)
        session.free(h)


def matmul_a4(b, h, x, O, extra=1):
    S = len(x)
    with Bufs(b) as d:
        y = d.up(np.full((S + extra, O), 7, np.float32))
        assert b.hip_fp4_matmul_a4_dev(h, y, d.up(x), S)
        got = d.down(y, (S + extra, O))
    assert (got[S:] == 7).all()
    return got[:S]


# rows around the 16-row subtiles and the tiles, widths around the 128-column steps
# and their pairs, outputs around the 16-row weight tiles
@pytest.mark.parametrize("I,O,S", [(1, 1, 1), (3, 9, 70), (4, 9, 40), (5, 20, 40), (12, 20, 200), (7, 3, 2), (8, 16, 1), (31, 17, 5), (32, 33, 16), (100, 40, 17), (128, 64, 1), (129, 15, 33),
                                   (256, 48, 64), (257, 100, 65), (384, 16, 3), (1000, 2999, 21), (999, 130, 70), (2048, 200, 128),
                                   (1152, 96, 129), (4096, 512, 1), (4096, 300, 200), (16400, 40, 9), (640, 1040, 300), (512, 4112, 2),
                                   (3000, 24, 1000), (7000, 16, 1100), (700, 14000, 21), (500, 13200, 3),
                                   (2000, 7100, 4), (1100, 13200, 50)])
def test_matmul(session, I, O, S):
    rng = np.random.default_rng(I + O * 3 + S)
    q4, e8 = rand_mxfp4(rng, O, I)
    h, w = session.upload_mxfp4(q4, e8, I, O), deq_mxfp4(q4, e8, I)
    try:
        x = act(rng, S, I)
        got = matmul_a4(session.b, h, x, O)
        xv = mx_quant(x)[2]
        assert (np.abs(got - xv @ w.T) <= product_tol(I) * (np.abs(xv) @ np.abs(w).T) + 1e-30).all()
        y = np.full((S, O), 7, np.float32)
        assert session.b.hip_fp4_matmul_a4(h, f32p(y), f32p(np.ascontiguousarray(x)), S)
        assert np.array_equal(y, got)
    finally:
        session.free(h)


@pytest.mark.parametrize("pin", ["few", "many"])
@pytest.mark.parametrize("I,O,S", [(1, 1, 1), (31, 17, 5), (128, 64, 1), (257, 100, 65), (600, 48, 33), (700, 300, 128), (999, 600, 130),
                                   (1300, 270, 260), (4096, 300, 1), (900, 520, 97)])
def test_matmul_on_both_kernels(session, monkeypatch, pin, I, O, S):
    """The kernel of few rows and that of many, pinned, at any size."""
    monkeypatch.setenv("COLI_HIP_FP4", pin)
    test_matmul(session, I, O, S)


@pytest.mark.parametrize("pin", ["few", "many"])
@pytest.mark.parametrize("pair", [False, True])
@pytest.mark.parametrize("E,I,O,counts", [(3, 300, 40, [0, 5, 0]), (4, 257, 17, [1, 64, 0, 65]), (5, 512, 48, [16, 17, 33, 2, 130]),
                                          (3, 800, 272, [300, 0, 140])])
def test_experts_on_both_kernels(session, monkeypatch, pin, pair, E, I, O, counts):
    monkeypatch.setenv("COLI_HIP_FP4", pin)
    test_experts(session, pair, E, I, O, counts)


def test_matmul_one_hot(session):
    """Rows of one 6: every weight at its place, exactly; blocks of other scales beside it."""
    rng = np.random.default_rng(3)
    I, O = 416, 72
    q4, e8 = rand_mxfp4(rng, O, I, 90, 160)
    h, w = session.upload_mxfp4(q4, e8, I, O), deq_mxfp4(q4, e8, I)
    try:
        x = np.eye(I, dtype=np.float32) * (6 * 2.0 ** rng.integers(-20, 20, (I, 1))).astype(np.float32)
        assert np.array_equal(matmul_a4(session.b, h, x, O), (x.astype(np.float64) @ w.T).astype(np.float32))
    finally:
        session.free(h)


@pytest.mark.parametrize("pin", ["few", "many"])
def test_matmul_of_every_scale(session, monkeypatch, pin):
    """One block of weights under each scale byte from 1 to 254, rows of one power of two that brings the product
    to 2^-140 .. 2^120: exactly, below f32's normal range too."""
    monkeypatch.setenv("COLI_HIP_FP4", pin)
    rng = np.random.default_rng(17)
    O, nb = 32, 254
    I = nb * 32
    q4 = rng.integers(0, 256, (O, I // 2), dtype=np.uint8)
    h = session.upload_mxfp4(q4, np.tile(np.arange(1, 255, dtype=np.uint8), (O, 1)), I, O)
    codes = E2M1[nibbles(q4, I)][:, ::32].T
    try:
        for p in (-140, -126, -60, 0, 60, 120):
            e = p - (np.arange(1, 255) - 127.0)
            ok = (e >= -127) & (e <= 126)
            x = np.zeros((nb, I), np.float32)
            x[np.flatnonzero(ok), 32 * np.flatnonzero(ok)] = 2.0 ** e[ok]
            assert np.array_equal(matmul_a4(session.b, h, x, O), np.where(ok[:, None], codes * 2.0 ** p, 0).astype(np.float32)), p
    finally:
        session.free(h)


def test_matmul_wide_ranges(session):
    """Scales from 2^-60 to 2^60 on both sides, zero blocks, a zero row."""
    rng = np.random.default_rng(4)
    I, O, S = 640, 80, 37
    q4, e8 = rand_mxfp4(rng, O, I, 67, 187)
    e8[:, 3] = 0
    q4[:, 48:64] = 0
    h, w = session.upload_mxfp4(q4, e8, I, O), deq_mxfp4(q4, e8, I)
    try:
        x = (rng.standard_normal((S, I)) * 2.0 ** np.repeat(rng.integers(-60, 60, (S, I // 32)), 32, 1)).astype(np.float32)
        x[5], x[:, 64:96] = 0, 0
        got, xv = matmul_a4(session.b, h, x, O), mx_quant(x)[2]
        assert (np.abs(got - xv @ w.T) <= product_tol(I) * (np.abs(xv) @ np.abs(w).T)).all()
        assert not got[5].any()
    finally:
        session.free(h)


@pytest.mark.parametrize("S", [1, 4, 20, 130])
def test_matmul_rows_do_not_mix(session, S):
    """A row with a NaN or an infinity is NaN, the others keep their bits."""
    rng = np.random.default_rng(5)
    I, O = 300, 50
    q4, e8 = rand_mxfp4(rng, O, I)
    h = session.upload_mxfp4(q4, e8, I, O)
    try:
        x = act(rng, S, I)
        clean = matmul_a4(session.b, h, x, O)
        bad = sorted({0, S // 2, S - 1} - {0} if S > 1 else {0})
        for k, r in enumerate(bad):
            x[r, 299 if k else 40] = np.inf if k else np.nan
        got = matmul_a4(session.b, h, x, O)
        keep = np.ones(S, bool)
        keep[bad] = False
        assert np.isnan(got[bad]).all() and np.array_equal(got[keep], clean[keep])
    finally:
        session.free(h)


def test_matmul_output_past_the_caches(session):
    """More than 128 MiB of output, stored past the caches: a sample of the rows against 64 bits, and rows
    behind the last as they were."""
    rng = np.random.default_rng(6)
    I, O, S = 300, 15000, 2300
    q4, e8 = rand_mxfp4(rng, O, I)
    h, w = session.upload_mxfp4(q4, e8, I, O), deq_mxfp4(q4, e8, I)
    try:
        x = act(rng, S, I)
        got = matmul_a4(session.b, h, x, O)
        r = np.append(np.arange(0, S, 41), S - 1)
        xv = mx_quant(x[r])[2]
        assert (np.abs(got[r] - xv @ w.T) <= product_tol(I) * (np.abs(xv) @ np.abs(w).T) + 1e-30).all()
    finally:
        session.free(h)


class Experts:
    """E random experts (pairs with `pair`) and their set."""

    def __init__(self, session, rng, E, I, O, pair, limit=0.0):
        self.s, self.I, self.O, self.E, self.limit = session, I, O, E, limit
        self.h, self.w, self.set = [], [], C.c_void_p()
        for _ in range(2 if pair else 1):
            mats = [rand_mxfp4(rng, O, I, 117, 121) for _ in range(E)]
            self.h.append([session.upload_mxfp4(q, e, I, O) for q, e in mats])
            self.w.append([deq_mxfp4(q, e, I) for q, e in mats])
        arr = [tensor_array(h) for h in self.h]
        assert session.b.hip_experts_create(C.byref(self.set), 0, E, arr[0][0], arr[1][0] if pair else None, limit)

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.s.b.hip_experts_free(self.set)
        for hs in self.h:
            for h in hs:
                self.s.free(h)

    def ref(self, e, xv):
        """(values, allowed error) of rows xv [n, I] through expert e."""
        v = [xv @ w[e].T for w in self.w]
        t = [product_tol(self.I) * (np.abs(xv) @ np.abs(w[e]).T) for w in self.w]
        if len(v) == 1:
            return v[0], t[0] + 1e-30
        g, u = v
        if self.limit > 0:
            g, u = np.minimum(g, self.limit), np.clip(u, -self.limit, self.limit)
        # |silu'| <= 1.1; exp, the division and two products: 16 roundings
        return silu(g) * u, 1.1 * t[0] * np.abs(u) + np.abs(silu(g)) * t[1] + 1.1 * t[0] * t[1] + 2.0 ** -20 * np.abs(silu(g) * u) + 1e-30

    def run(self, x, off, N, src=None, K=1, extra=2):
        b = self.s.b
        with Bufs(b) as d:
            y = d.up(np.full((N + extra, self.O), 7, np.float32))
            assert b.hip_experts_a4_dev(self.set, y, d.up(x), len(x), None if src is None else d.up(src), K, d.up(np.asarray(off, np.int32)), N)
            return d.down(y, (N + extra, self.O))

    def check(self, got, xv, off, N, rows):
        seen = np.zeros(len(got), bool)
        for e in range(self.E):
            r = np.arange(max(0, off[e]), min(N, off[e + 1]))
            if len(r):
                seen[r] = True
                v, tol = self.ref(e, xv[rows[r]])
                assert (np.abs(got[r] - v) <= tol).all(), (e, np.abs(got[r] - v).max())
        assert (got[~seen] == 7).all()


# per expert: none, one, up to and past the tiles
@pytest.mark.parametrize("pair", [False, True])
@pytest.mark.parametrize("E,I,O,counts", [(1, 1, 1, [1]), (1, 128, 16, [70]), (3, 300, 40, [0, 5, 0]), (4, 257, 17, [1, 64, 0, 65]),
                                          (5, 512, 48, [16, 17, 33, 2, 130]), (300, 64, 16, None), (2, 1000, 33, [300, 1]),
                                          (3, 256, 272, [700, 0, 140])])
def test_experts(session, pair, E, I, O, counts):
    rng = np.random.default_rng(E + I + O)
    if counts is None:
        counts = rng.choice([0, 0, 1, 2], E)
    off = np.concatenate([[0], np.cumsum(counts)])
    N = int(off[-1])
    x = act(rng, N, I)
    with Experts(session, rng, E, I, O, pair) as ex:
        got = ex.run(x, off, N)
        ex.check(got, mx_quant(x)[2], off, N, np.arange(N))
        # rows through src: bitwise the copied rows'
        perm = rng.permutation(N).astype(np.int32)
        inv = np.argsort(perm)
        again = ex.run(np.ascontiguousarray(x[inv]), off, N, src=(perm * 3 + rng.integers(0, 3, N)).astype(np.int32), K=3)
        assert np.array_equal(again, got)


def test_experts_clamped(session):
    rng = np.random.default_rng(7)
    off = [0, 3, 90]
    x = act(rng, 90, 320) * 4
    with Experts(session, rng, 2, 320, 40, True, 1.5) as ex:
        ex.check(ex.run(x, off, 90), mx_quant(x)[2], off, 90, np.arange(90))


@pytest.mark.parametrize("pin", ["few", "many"])
def test_swiglu_extremes(session, monkeypatch, pin):
    """Gates from -infinity to infinity and NaN, with and without the clamp: gate and up are
    single products here (one column of x, one weight a row), so the formula is checked alone."""
    monkeypatch.setenv("COLI_HIP_FP4", pin)
    O = 16
    q4 = np.full((O, 16), 0x00, np.uint8)
    q4[:, 0] = 2                                   # weight 1 in column 0
    one = np.full((O, 1), 127, np.uint8)
    two = np.full((O, 1), 128, np.uint8)
    g, u = session.upload_mxfp4(q4, one, 32, O), session.upload_mxfp4(q4, two, 32, O)
    x = np.zeros((26, 32), np.float32)
    big = np.array([0, 0.5, 1, 3, 4, 6, 12, 24, 64, 96, 128, 192, 2.0 ** 60, 2.0 ** 126], np.float32)
    x[:14, 0], x[14:25, 0], x[25, 0] = big, -big[1:12], np.nan
    try:
        for limit in (0.0, 1.5):
            s = C.c_void_p()
            (ga, _a), (ua, _b) = tensor_array([g]), tensor_array([u])
            assert session.b.hip_experts_create(C.byref(s), 0, 1, ga, ua, limit)
            with Bufs(session.b) as d:
                y = d.up(np.zeros((26, O), np.float32))
                assert session.b.hip_experts_a4_dev(s, y, d.up(x), 26, None, 1, d.up(np.array([0, 26], np.int32)), 26)
                got = d.down(y, (26, O))
            session.b.hip_experts_free(s)
            a = x[:, 0].astype(np.float64)
            b = 2 * a
            if limit:
                a, b = np.minimum(a, limit), np.clip(b, -limit, limit)
            with np.errstate(over="ignore", invalid="ignore"):
                ref = (silu(a) * b).astype(np.float32)
            assert np.isnan(got[25]).all()
            for r in range(25):
                if np.isinf(ref[r]):
                    assert (got[r] == ref[r]).all(), (r, got[r, 0])
                else:   # 16 roundings, results below the normal range are zero
                    assert (np.abs(got[r] - np.float64(ref[r])) <= 2.0 ** -20 * abs(float(ref[r])) + 2.0 ** -120).all(), (r, got[r, 0], ref[r])
    finally:
        session.free(g)
        session.free(u)


@pytest.mark.parametrize("S,I,O", [(1, 700, 90), (3, 333, 33), (40, 700, 90), (300, 257, 530), (100, 7000, 300)])
def test_products_at_any_address(session, S, I, O):
    """Rows and results from any float on: the bits of those that start at 16 bytes, nothing beside them written."""
    rng = np.random.default_rng(S)
    b, x = session.b, act(rng, S, I)
    off = np.array([0, S // 3, S], np.int32)
    with Experts(session, rng, 2, I, O, True) as ex:
        h = ex.h[0][0]
        want, wanted = matmul_a4(b, h, x, O), ex.run(x, off, S)[:S]
        for k in (1, 3):
            with Bufs(b) as d:
                px, d_off = d.up(np.zeros(S * I + 8, np.float32)) + 4 * k, d.up(np.zeros(8, np.int32)) + 4 * k
                d.put(px, x)
                d.put(d_off, off)
                for one in (True, False):
                    y = d.up(np.full(S * O + 8, 7, np.float32)) + 4 * k
                    assert b.hip_fp4_matmul_a4_dev(h, y, px, S) if one else b.hip_experts_a4_dev(ex.set, y, px, S, None, 1, d_off, S)
                    got = d.down(y - 4 * k, S * O + 8)
                    assert np.array_equal(got[k:k + S * O].reshape(S, O), want if one else wanted)
                    assert (got[:k] == 7).all() and (got[k + S * O:] == 7).all()


def test_expert_pairs_past_the_caches(session):
    """Pairs with more than 128 MiB of results, stored past the caches: a sample of the rows, and those behind the last."""
    rng = np.random.default_rng(16)
    E, I, O, counts = 3, 64, 8200, [1500, 0, 2700]
    off = np.concatenate([[0], np.cumsum(counts)])
    N = int(off[-1])
    x = act(rng, N, I)
    with Experts(session, rng, E, I, O, True) as ex:
        got = ex.run(x, off, N)
        assert (got[N:] == 7).all()
        for e in (0, 2):
            r = np.append(np.arange(off[e], off[e + 1], 31), off[e + 1] - 1)
            v, tol = ex.ref(e, mx_quant(x[r])[2])
            assert (np.abs(got[r] - v) <= tol).all()


@pytest.mark.parametrize("pin", ["few", "many"])
def test_swiglu_of_low_gates(session, monkeypatch, pin):
    """Gates whose sigmoid is below f32's normal range, with ups that bring the result back into it:
    a gate is the sum of three columns, exactly, and an up has a column of its own. 16 roundings of
    2^-24 and half the smallest step. Rows beside such gates keep their bits."""
    monkeypatch.setenv("COLI_HIP_FP4", pin)
    O, I = 16, 128
    gates = [(-96, 12, -2), (-96, 12, -3), (-96, 8, 0.75), (-96, 8, 0.5), (-96, 8, 0), (-96, 8, -0.5), (-96, 8, -0.75), (-96, 8, -1),
             (-96, 4, 0), (-96, 0, 0), (-96, -6, 0.5), (-96, -8, 0), (-128, 0, 0), (-128, -24, 2), (-192, 12, 0), (-192, -3, 0),
             (-2.0 ** 80, 0, 0), (-96, 64, 0), (1, 0, 0), (96, -8, 0), (-1, 0, 0)]
    ups = [1, -2.0 ** 20, 2.0 ** 60, 1.5 * 2.0 ** 126, 2.0 ** -20]
    q = np.zeros((2, O, I // 2), np.uint8)
    q[0, :, [0, 16, 32]] = 2                       # weight 1 in columns 0, 32 and 64
    q[1, :, 48] = 2                                # and in 96
    one = np.full((O, I // 32), 127, np.uint8)
    g, u = session.upload_mxfp4(q[0], one, I, O), session.upload_mxfp4(q[1], one, I, O)
    x = np.zeros((len(gates) * len(ups), I), np.float32)
    for r, (gate, up) in enumerate((a, b) for b in ups for a in gates):
        x[r, [0, 32, 64]], x[r, 96] = gate, up
    n = len(x)
    a, b = x[:, [0, 32, 64]].astype(np.float64).sum(1), x[:, 96].astype(np.float64)
    assert np.array_equal(mx_quant(x)[2], x)       # every value has a code
    s = C.c_void_p()
    (ga, _a), (ua, _b) = tensor_array([g]), tensor_array([u])

    def run(x):
        with Bufs(session.b) as d:
            y = d.up(np.zeros((len(x), O), np.float32))
            assert session.b.hip_experts_a4_dev(s, y, d.up(x), len(x), None, 1, d.up(np.array([0, len(x)], np.int32)), len(x))
            return d.down(y, (len(x), O))

    try:
        for limit in (0.0, 2.0 ** 125):
            assert session.b.hip_experts_create(C.byref(s), 0, 1, ga, ua, limit)
            got = run(x)
            c = np.clip(b, -limit, limit) if limit else b
            ref = silu(a) * c
            over = np.abs(ref) >= 2.0 ** 128       # infinities of f32 (none of the others is near)
            assert (got[over] == np.sign(ref[over])[:, None] * np.inf).all()
            ref = np.where(over, 0, ref)
            bad = (np.abs(got - ref[:, None]) > 2.0 ** -20 * np.abs(ref[:, None]) + 2.0 ** -150) & ~over[:, None]
            assert not bad.any(), [(float(a[r]), float(c[r]), float(got[r, 0]), float(ref[r])) for r in np.flatnonzero(bad.any(1))]
            high = np.flatnonzero(a > -64)
            assert np.array_equal(run(np.ascontiguousarray(x[high])), got[high])
            session.b.hip_experts_free(s)
            s = C.c_void_p()
    finally:
        session.b.hip_experts_free(s)
        session.free(g)
        session.free(u)


@pytest.mark.parametrize("pin,O", [("few", 144000), ("many", 1160000)])
def test_experts_of_more_workgroups_than_a_launch(session, monkeypatch, pin, O):
    """1024 experts of a row each and so many outputs that their workgroups pass 2^23: rows before, at
    and behind the place where the launches part, and the row behind the last as it was."""
    monkeypatch.setenv("COLI_HIP_FP4", pin)
    rng = np.random.default_rng(13)
    E, I = 1024, 8
    mats = [rand_mxfp4(rng, O, I) for _ in range(2)]
    h = [session.upload_mxfp4(q, e, I, O) for q, e in mats]
    w = [deq_mxfp4(q, e, I) for q, e in mats]
    s = C.c_void_p()
    (ga, _a), (ua, _b) = tensor_array([h[0]] * E), tensor_array([h[1]] * E)
    b, x = session.b, act(rng, E, I)
    y = b.cuda_pipe_alloc(0, (E + 1) * O * 4)
    try:
        assert y and b.hip_experts_create(C.byref(s), 0, E, ga, ua, 0.0)
        with Bufs(b) as d:
            d.put(y + E * O * 4, np.full(O, 7, np.float32))
            assert b.hip_experts_a4_dev(s, y, d.up(x), E, None, 1, d.up(np.arange(E + 1, dtype=np.int32)), E)
            for r in (0, 1, 500, 900, *range(920, 936), 1000, 1023):
                got, xv = d.down(y + r * O * 4, O), mx_quant(x[r:r + 1])[2][0]
                g, u = (v @ xv for v in w)
                tg, tu = (product_tol(I) * (np.abs(v) @ np.abs(xv)) for v in w)
                tol = 1.1 * tg * np.abs(u) + np.abs(silu(g)) * tu + 1.1 * tg * tu + 2.0 ** -20 * np.abs(silu(g) * u) + 1e-30
                assert (np.abs(got - silu(g) * u) <= tol).all(), r
            assert (d.down(y + E * O * 4, O) == 7).all()
    finally:
        b.hip_experts_free(s)
        b.cuda_pipe_free(0, y)
        for t in h:
            session.free(t)


def test_experts_of_rows_beyond_2_gib(session, monkeypatch):
    """Operands of more than 2 GiB that src chooses from: the bits of the same rows copied out. Only
    the chosen rows of x hold anything."""
    rng = np.random.default_rng(14)
    b, (I, rows, N, K, O) = session.b, (1 << 20, 4200, 150, 2, 20)
    at = np.array([0, 1, 2047, 2048, 4095, 4096, 4198, 4199], np.int64)
    xr, pick, off = act(rng, len(at), I), rng.integers(0, len(at), N), [0, 20, 150]
    src = (at[pick] * K + rng.integers(0, K, N)).astype(np.int32)
    src[77] = rows * K
    x = b.cuda_pipe_alloc(0, rows * I * 4)
    try:
        assert x
        with Experts(session, rng, 2, I, O, False) as ex, Bufs(b) as d:
            for r, v in zip(at, xr):
                d.put(x + int(r) * I * 4, v)
            y = d.up(np.full((N + 1, O), 7, np.float32))
            assert b.hip_experts_a4_dev(ex.set, y, x, rows, d.up(src), K, d.up(np.array(off, np.int32)), N)
            got = d.down(y, (N + 1, O))
            assert (got[N] == 7).all() and not got[77].any()
            pick[77] = 0
            monkeypatch.setenv("COLI_HIP_FP4", "few")
            want = ex.run(xr, off, N, src=pick.astype(np.int32))[:N]
            want[77] = 0
            assert np.array_equal(got[:N], want) and np.abs(want).max() > 1
    finally:
        b.cuda_pipe_free(0, x)


def test_experts_offsets_and_rows_outside(session):
    """Rows before the first and behind the last offset stay as they were, offsets are taken
    within 0..N, sources outside x are rows of zeros, and descending offsets are empty."""
    rng = np.random.default_rng(8)
    x = act(rng, 20, 130)
    xv = mx_quant(x)[2]
    with Experts(session, rng, 3, 130, 20, False) as ex:
        for off in ([2, 9, 9, 15], [-5, 4, 1000, 2 ** 31 - 1], [0, 0, 0, 0], [-9, -3, -1, 0], [12, 4, 4, 2]):
            ex.check(ex.run(x, off, 20), xv, np.clip(off, 0, 20), 20, np.arange(20))
        # overlapping ranges of experts: no more tiles than there is room for, and inside y
        got = ex.run(x, [0, 20, 0, 20], 20)
        assert (got[20:] == 7).all()
        src = np.arange(20, dtype=np.int32)
        src[[0, 7, 19]] = [-1, 20, 2 ** 31 - 1]
        got = ex.run(x, [0, 5, 12, 20], 20, src=src)
        assert not got[[0, 7, 19]].any()
        keep = np.setdiff1d(np.arange(20), [0, 7, 19])
        assert np.array_equal(got[keep], ex.run(x, [0, 5, 12, 20], 20)[keep])
        assert session.b.hip_experts_a4_dev(ex.set, None, None, 0, None, 1, None, 0)


@pytest.mark.parametrize("pin", ["few", "many"])
def test_experts_more_sorted_rows_than_rows(session, monkeypatch, pin):
    """Without src the rows past x are rows of zeros, whole tiles of them too."""
    monkeypatch.setenv("COLI_HIP_FP4", pin)
    rng = np.random.default_rng(10)
    I, N, rows = 200, 700, 130
    off = [0, 100, 380, 700]
    x = act(rng, rows, I)
    xv = np.concatenate([mx_quant(x)[2], np.zeros((N - rows, I))])
    with Experts(session, rng, 3, I, 40, False) as ex:
        ex.check(ex.run(x, off, N), xv, off, N, np.arange(N))


@pytest.mark.parametrize("pin", ["few", "many"])
@pytest.mark.parametrize("S", [2, 70])
def test_weights_of_scale_255_and_0(session, monkeypatch, pin, S):
    """A scale byte of 255 makes its output NaN and no other; a byte of 0 counts as 2^-127: nothing here."""
    monkeypatch.setenv("COLI_HIP_FP4", pin)
    rng = np.random.default_rng(12)
    I, O = 300, 50
    q4, e8 = rand_mxfp4(rng, O, I)
    e8[17, 9], e8[40, 0], e8[3, 4], e8[20, :] = 255, 255, 0, 0
    h = session.upload_mxfp4(q4, e8, I, O)
    try:
        x = act(rng, S, I)
        got = matmul_a4(session.b, h, x, O)
    finally:
        session.free(h)
    bad = np.isin(np.arange(O), [17, 40])
    w = deq_mxfp4(q4, np.where(e8 == 255, 127, e8).astype(np.uint8), I)
    xv = mx_quant(x)[2]
    assert np.isnan(got[:, bad]).all()
    assert (np.abs(got - xv @ w.T) <= product_tol(I) * (np.abs(xv) @ np.abs(w).T) + 1e-30)[:, ~bad].all()


def route(rng, T, E, K):
    z = rng.standard_normal((T, E))
    idx = np.argsort(-z, 1)[:, :K].astype(np.int32)
    w = np.exp(np.take_along_axis(z, idx, 1))
    return idx, (w / w.sum(1, keepdims=True)).astype(np.float32)


@pytest.mark.parametrize("T", [1, 16, 300])
def test_layer_of_sorted_rows(session, T):
    """Dispatch, the experts' pair, their down matrices, combine: eager and as a graph replayed
    over changing rows, through src and over copied rows alike; and over rows that were sent in
    4 bits (quantized, dispatched, read back): the same values to Q, under half the scale where
    a block's largest became 3 scales."""
    rng = np.random.default_rng(T)
    b, (E, K, D, I) = session.b, (12, 4, 288, 160)
    N = T * K
    with Experts(session, rng, E, D, I, True) as up, Experts(session, rng, E, I, D, False) as down, Bufs(b) as d:
        px, pi, pw = d.up(np.zeros((T, D), np.float32)), d.up(np.zeros((T, K), np.int32)), d.up(np.zeros((T, K), np.float32))
        off, src, pos = (d.up(np.zeros(n, np.int32)) for n in (E + 1, N, N))
        xs, h, ys = (d.up(np.zeros((N, n), np.float32)) for n in (D, I, D))
        out = [d.up(np.zeros((T, D), np.float32)) for _ in range(2)]
        q4, e8 = d.up(np.zeros((T, D // 2), np.uint8)), d.up(np.zeros((T, D // 32), np.uint8))
        q4s, e8s = d.up(np.zeros((N, D // 2), np.uint8)), d.up(np.zeros((N, D // 32), np.uint8))

        def layer(o, how):
            if how == "src":
                assert b.hip_dispatch_dev(0, pi, None, None, T, E, K, None, 0, off, src, pos, None)
                assert b.hip_experts_a4_dev(up.set, h, px, T, src, K, off, N)
            else:
                if how == "rows":
                    assert b.hip_dispatch_dev(0, pi, None, None, T, E, K, px, D * 4, off, src, pos, xs)
                else:
                    assert b.hip_mxfp4_quantize_dev(0, px, 0, T, D, q4, e8)
                    assert b.hip_dispatch_dev(0, pi, None, None, T, E, K, q4, D // 2, off, src, pos, q4s)
                    assert b.hip_dispatch_dev(0, pi, None, None, T, E, K, e8, D // 32, off, src, pos, e8s)
                    assert b.hip_mxfp4_dequantize_dev(0, q4s, e8s, N, D, xs, 0)
                assert b.hip_experts_a4_dev(up.set, h, xs, N, None, 1, off, N)
            assert b.hip_experts_a4_dev(down.set, ys, h, N, None, 1, off, N)
            assert b.hip_combine_dev(0, ys, 0, pos, pw, T, K, N, D, o)

        layer(out[0], "src")
        with hiprt.Graph(b.hip_stream(0)) as g:
            layer(out[0], "src")
        for rep in range(3):
            x, (idx, w) = act(rng, T, D), route(rng, T, E, K)
            for p, v in ((px, x), (pi, idx), (pw, w)):
                d.put(p, v)
            g.launch()
            first = d.down(out[0], (T, D))
            ro, rs, rp = plan(idx, None, None, E)
            # against 64 bits from the h that the device has (its own rounding decides h's codes)
            for how in ("sent", "rows"):
                layer(out[1], how)
                hd = d.down(h, (N, I))
                up.check(np.concatenate([hd, np.full((1, I), 7, np.float32)]), mx_quant(x)[2], ro, N, rs // K)
            assert np.array_equal(d.down(out[1], (T, D)).view(np.uint32), first.view(np.uint32))
            hv, yv, tol = mx_quant(hd)[2], np.zeros((N, D)), np.zeros((N, D))
            for e in range(E):
                yv[ro[e]:ro[e + 1]], tol[ro[e]:ro[e + 1]] = down.ref(e, hv[ro[e]:ro[e + 1]])
            ref, mag = combine(yv, rp, w, N)
            room, _ = combine(tol, rp, np.abs(w), N)
            assert (np.abs(first - ref) <= room + (K + 1) * 2.0 ** -24 * mag).all()


@pytest.mark.parametrize("S,I,O", [(1, 700, 90), (3, 700, 90), (40, 700, 90), (300, 700, 90), (100, 7000, 300)])
def test_matmul_graph_replays(session, S, I, O):
    """Replays over changing rows with larger eager calls between (outgrown workspaces stay); the
    last size splits K."""
    rng = np.random.default_rng(S)
    b = session.b
    q4, e8 = rand_mxfp4(rng, O, I)
    h = session.upload_mxfp4(q4, e8, I, O)
    try:
        with Bufs(b) as d:
            px, y, y2 = d.up(np.zeros((S, I), np.float32)), d.up(np.zeros((S, O), np.float32)), d.up(np.zeros((S, O), np.float32))
            assert b.hip_fp4_matmul_a4_dev(h, y, px, S)
            with hiprt.Graph(b.hip_stream(0)) as g:
                assert b.hip_fp4_matmul_a4_dev(h, y, px, S)
            for rep in range(3):
                d.put(px, act(rng, S, I))
                g.launch()
                matmul_a4(b, h, act(rng, 700 * (rep + 1), I), O)
                assert b.hip_fp4_matmul_a4_dev(h, y2, px, S)
                assert np.array_equal(d.down(y, (S, O)).view(np.uint32), d.down(y2, (S, O)).view(np.uint32))
    finally:
        session.free(h)


def test_straight_through_gradient(session):
    """dx = dy W of coli_hip_gemm_t_dev is the product's gradient for rows that Q leaves as they
    are: the call is linear along steps that stay on such rows."""
    rng = np.random.default_rng(9)
    b, (I, O, S) = session.b, (96, 40, 6)
    q4, e8 = rand_mxfp4(rng, O, I)
    h = session.upload_mxfp4(q4, e8, I, O)
    try:
        grid = E2M1[:8]
        x = rng.choice(grid, (S, I)).astype(np.float32)
        v = rng.choice([-0.5, 0.0, 0.5], (S, I)).astype(np.float32)
        x[:, ::32], v[:, ::32] = 6, 0                                # the block's scale stays 1
        v[(x > 1) | (x < 0.5)] = 0                                   # x +- v are codes too
        dy = rng.standard_normal((S, O)).astype(np.float32)
        a, c = (matmul_a4(b, h, (x + s * v).astype(np.float32), O).astype(np.float64) for s in (1, -1))
        with Bufs(b) as d:
            px = d.up(np.zeros((S, I), np.float32))
            assert b.hip_gemm_t_dev(h, px, d.up(dy), S)
            dx = d.down(px, (S, I)).astype(np.float64)
        w = deq_mxfp4(q4, e8, I)
        mag = (np.abs(dy).astype(np.float64) * (np.abs(x) @ np.abs(w).T)).sum()
        assert abs(((a - c) / 2 * dy).sum() - (dx * v).sum()) <= 2.0 ** -18 * mag
    finally:
        session.free(h)


def test_refusals(session):
    b = session.b
    rng = np.random.default_rng(0)
    I, O = 64, 32
    q4, e8 = rand_mxfp4(rng, O, I)
    h, other = session.upload_mxfp4(q4, e8, I, O), session.upload_mxfp4(*rand_mxfp4(rng, O, 96), 96, O)
    i4, sc = rand_i4(rng, O, I, 32)
    hi = session.upload(i4, sc, 4, I, O, 32)
    big = 2 ** 31 - 1
    try:
        with Bufs(b) as d:
            x, y, q, e = (d.up(np.zeros(4096, np.float32)) for _ in range(4))

            def refused(fn, ok, changes):
                assert fn(*ok)
                for ch in changes:
                    a = list(ok)
                    for k, v in ch.items():
                        a[k] = v
                    assert not fn(*a), ch

            refused(b.hip_mxfp4_quantize_dev, (0, x, 0, 4, 70, q, e),
                    [{0: 5}, {0: -1}, {1: None}, {2: 3}, {2: -1}, {3: -1}, {3: big}, {4: 0}, {4: big}, {5: None}, {6: None}, {5: x}, {6: x}, {6: q}])
            refused(b.hip_mxfp4_dequantize_dev, (0, q, e, 4, 70, y, 0),
                    [{0: 5}, {1: None}, {2: None}, {3: -1}, {3: big}, {4: 0}, {4: big}, {5: None}, {6: 3}, {5: q}, {5: e}])
            refused(b.hip_fp4_matmul_a4_dev, (h, y, x, 3), [{0: None}, {0: hi}, {1: None}, {2: None}, {3: 0}, {3: -1}, {3: big}, {1: x}])
            t = C.c_void_p()
            for a in ((None, x, 0, I, O, 0), (C.byref(h), x, 0, I, O, 0), (C.byref(t), None, 0, I, O, 0), (C.byref(t), x, 3, I, O, 0),
                      (C.byref(t), x, 0, 0, O, 0), (C.byref(t), x, 0, I, 0, 0), (C.byref(t), x, 0, I, O, 9)):
                assert not b.hip_tensor_quantize_mxfp4(*a) and not t
            host = np.zeros((3, O), np.float32)
            assert not b.hip_fp4_matmul_a4(hi, f32p(host), f32p(np.zeros((3, I), np.float32)), 3)
            assert not b.hip_fp4_matmul_a4(h, f32p(host), f32p(np.zeros((3, I), np.float32)), 0)
            s = C.c_void_p()
            two, two4, mixed = tensor_array([h, h]), tensor_array([h, hi]), tensor_array([h, other])
            gone = (C.c_void_p * 2)(h.value, None)
            for a in ((None, 0, 2, two[0], None, 0.0), (C.byref(s), 9, 2, two[0], None, 0.0), (C.byref(s), 0, 0, two[0], None, 0.0),
                      (C.byref(s), 0, 1025, two[0], None, 0.0), (C.byref(s), 0, 2, None, None, 0.0), (C.byref(s), 0, 2, two4[0], None, 0.0),
                      (C.byref(s), 0, 2, two[0], two4[0], 0.0), (C.byref(s), 0, 2, mixed[0], None, 0.0), (C.byref(s), 0, 2, two[0], mixed[0], 0.0),
                      (C.byref(s), 0, 2, C.cast(gone, C.POINTER(C.c_void_p)), None, 0.0)):
                assert not b.hip_experts_create(*a) and not s
            assert b.hip_experts_create(C.byref(s), 0, 2, two[0], two[0], 0.0)
            src, off = d.up(np.zeros(8, np.int32)), d.up(np.array([0, 1, 4], np.int32))
            refused(b.hip_experts_a4_dev, (s, y, x, 4, src, 1, off, 4),
                    [{0: None}, {1: None}, {2: None}, {3: -1}, {3: 0}, {3: big}, {5: 0}, {6: None}, {7: -1}, {7: big}, {1: x}, {1: src}, {1: off}])
            b.hip_experts_free(s)
            b.hip_experts_free(None)
            assert b.cuda_pipe_sync(0)
    finally:
        for t in (h, other, hi):
            session.free(t)
