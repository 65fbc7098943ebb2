"""coli_hip_gemm_t_dev (dx = dy W over resident quantized weights) against a
64-bit product with the dequantized matrix."""
import ctypes as C

import numpy as np
import pytest

from colibri_amd import hiprt
from op_util import KINDS, Bufs, close, gemm_tol, matrix, sum_tol
from quant_util import deq_i4, deq_mxfp4, rand_i4, rand_mxfp4

pytestmark = pytest.mark.gpu


def run(session, h, dy, I):
    with Bufs(session.b) as d:
        py, px = d.up(dy), d.up(np.full((dy.shape[0], I), 7.0, np.float32))
        assert session.b.hip_gemm_t_dev(h, px, py, dy.shape[0])
        return d.down(px, (dy.shape[0], I))


def tol(kind, O):
    return sum_tol(2 * O) if kind == "gen" else gemm_tol(O)


# O and I around the tiles (16 rows, 128 columns) and the K steps (32 rows),
# rows around the tile heights 32 / 64 / 128 and the K splits
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("O,I,S", [(1, 1, 1), (2, 40, 70), (3, 200, 9), (5, 128, 64), (16, 128, 1), (17, 33, 2), (33, 129, 5), (100, 200, 16), (31, 64, 31),
                                   (96, 256, 32), (48, 130, 33), (640, 384, 64), (200, 515, 65), (1040, 260, 128),
                                   (64, 128, 129), (2049, 131, 20), (300, 1000, 300)])
def test_matches_dense(session, kind, O, I, S):
    rng = np.random.default_rng(O * 7 + I * 3 + S + KINDS.index(kind))
    h, w = matrix(session, rng, kind, O, I)
    try:
        dy = rng.standard_normal((S, O)).astype(np.float32)
        close(run(session, h, dy, I), dy.astype(np.float64) @ w, np.abs(dy).astype(np.float64) @ np.abs(w), tol(kind, O))
    finally:
        session.free(h)


@pytest.mark.parametrize("pin", ["few", "many"])
@pytest.mark.parametrize("kind", ["i4h", "i4f", "fp4"])
@pytest.mark.parametrize("O,I,S", [(1, 1, 1), (5, 131, 33), (200, 300, 64), (64, 512, 128), (700, 70, 129), (1030, 400, 260)])
def test_both_kernels_at_any_size(session, monkeypatch, pin, kind, O, I, S):
    """The kernel that converts its rows itself and the one that reads them built, pinned."""
    monkeypatch.setenv("COLI_HIP_GEMM_T", pin)
    test_matches_dense(session, kind, O, I, S)


@pytest.mark.parametrize("S,pin", [(700, "few"), (4096, "many")])
def test_rows_choose_the_kernel(session, S, pin):
    """By the modelled times (2000 x 2044 on 256 CUs, us: 700 rows two rounds of
    few, 8 + 2 x 8 x 2.5 = 48, five splits of the other 29 + 12 + 10 = 51; 4096
    rows eight rounds, 168, against 99 + 23 = 122): bitwise the pinned kernel."""
    rng = np.random.default_rng(29)
    O, I = 2000, 2044
    h, w = matrix(session, rng, "i4h", O, I)
    try:
        dy = rng.standard_normal((S, O)).astype(np.float32)
        got = run(session, h, dy, I)
        close(got, dy.astype(np.float64) @ w, np.abs(dy).astype(np.float64) @ np.abs(w), gemm_tol(O))
        with pytest.MonkeyPatch.context() as m:
            m.setenv("COLI_HIP_GEMM_T", pin)
            assert np.array_equal(run(session, h, dy, I).view(np.uint32), got.view(np.uint32))
    finally:
        session.free(h)


def test_one_hot_rows_read_the_matrix(session):
    """dy = e_o gives row o of W: every weight at its place, as exact as its
    fp16 hi + lo: 3 x 2^-22 of an f32 scale's weight (see gemm_tol), else exact
    down to fp16's last place under the column group's largest scale."""
    rng = np.random.default_rng(3)
    for kind in ("i4h", "i4f", "fp4"):
        h, w = matrix(session, rng, kind, 80, 272)
        try:
            got = run(session, h, np.eye(80, dtype=np.float32), 272)
            close(got, w, np.abs(w).max(0, keepdims=True) + 0 * w, 3 * 2.0 ** -22, kind)
        finally:
            session.free(h)


@pytest.mark.parametrize("fmt", [4, 7])
def test_wide_ranges(session, fmt):
    """Scales 2^-20 .. 2^12 apart from one column group to the next and from row
    to row, rows of dy 2^-60 .. 2^40, a zero row and a column group of zeros."""
    rng = np.random.default_rng(11 + fmt)
    O, I, S = 144, 320, 40
    ng = I // 32
    if fmt == 7:
        q4, e8 = rand_mxfp4(rng, O, I)
        e8 = (127 + rng.integers(-20, 13, (1, ng)) + rng.integers(-6, 1, (O, ng))).astype(np.uint8)
        e8[:, 3] = 0
        h, w = session.upload_mxfp4(q4, e8, I, O), deq_mxfp4(q4, e8, I)
    else:
        q4, sc = rand_i4(rng, O, I, 32, fp16_scales=False)
        sc = (sc * 2.0 ** rng.integers(-20, 13, (1, ng)) * 2.0 ** rng.integers(-6, 1, (O, ng))).astype(np.float32)
        sc[:, 3] = 0
        h, w = session.upload(q4, sc, 4, I, O, 32), deq_i4(q4, sc, I, 32)
    try:
        dy = (rng.standard_normal((S, O)) * 2.0 ** rng.integers(-60, 41, (S, 1))).astype(np.float32)
        dy[7] = 0
        ref = dy.astype(np.float64) @ w
        mag = np.abs(dy).astype(np.float64) @ np.abs(w)
        got = run(session, h, dy, I)
        close(got, ref, mag, gemm_tol(O))
        assert not got[7].any() and not got[:, 96:128].any()
    finally:
        session.free(h)


def test_scales_follow_an_update(session):
    """The scales laid out for the gradient are those of the tensor's present weights."""
    rng = np.random.default_rng(5)
    O, I, S = 64, 256, 3
    h, _ = matrix(session, rng, "i4h", O, I)
    try:
        dy = rng.standard_normal((S, O)).astype(np.float32)
        run(session, h, dy, I)
        q4, sc = rand_i4(rng, O, I, 32)
        sc = sc * 4
        assert session.b.cuda_tensor_update(h, q4.ctypes.data_as(__import__("ctypes").c_void_p),
                                            sc.ctypes.data_as(__import__("ctypes").POINTER(__import__("ctypes").c_float)))
        w = deq_i4(q4, sc, I, 32)
        close(run(session, h, dy, I), dy.astype(np.float64) @ w, np.abs(dy).astype(np.float64) @ np.abs(w), gemm_tol(O))
    finally:
        session.free(h)


def test_rows_do_not_mix(session):
    """A row of infinities or NaN stays in its row, and what lies behind the last row is left as it was."""
    rng = np.random.default_rng(9)
    O, I, S = 70, 150, 37
    h, w = matrix(session, rng, "i4h", O, I)
    try:
        dy = rng.standard_normal((S, O)).astype(np.float32)
        dy[5, 3], dy[36, 0] = np.inf, np.nan
        with Bufs(session.b) as d:
            py, px = d.up(dy), d.up(np.full((S + 3, I), 7.0, np.float32))
            assert session.b.hip_gemm_t_dev(h, px, py, S)
            got = d.down(px, (S + 3, I))
        assert (got[S:] == 7.0).all()
        keep = [r for r in range(S) if r not in (5, 36)]
        close(got[keep], dy[keep].astype(np.float64) @ w, np.abs(dy[keep]).astype(np.float64) @ np.abs(w), gemm_tol(O))
        assert not np.isfinite(got[5]).all() and np.isnan(got[36]).any()
    finally:
        session.free(h)


def test_unaligned_rows(session):
    """Pointers that are only 4-byte aligned."""
    rng = np.random.default_rng(13)
    O, I, S = 128, 256, 18
    h, w = matrix(session, rng, "fp4", O, I)
    try:
        dy = rng.standard_normal((S, O)).astype(np.float32)
        with Bufs(session.b) as d:
            py, px = d.up(np.concatenate((np.zeros(1, np.float32), dy.ravel()))), d.up(np.zeros(S * I + 1, np.float32))
            assert session.b.hip_gemm_t_dev(h, px + 4, py + 4, S)
            got = d.down(px, (S * I + 1,))[1:].reshape(S, I)
        close(got, dy.astype(np.float64) @ w, np.abs(dy).astype(np.float64) @ np.abs(w), gemm_tol(O))
    finally:
        session.free(h)


def test_adjoint_of_the_projection(session):
    """<y, W x> = <W^T y, x>: the gradient belongs to coli_cuda_pipe_gemm's own matrix."""
    rng = np.random.default_rng(17)
    O, I, S = 272, 384, 24
    for kind in ("i4h", "fp4", "gen"):
        h, w = matrix(session, rng, kind, O, I)
        try:
            x, dy = rng.standard_normal((S, I)).astype(np.float32), rng.standard_normal((S, O)).astype(np.float32)
            with Bufs(session.b) as d:
                px, py = d.up(x), d.up(np.zeros((S, O), np.float32))
                assert session.b.cuda_pipe_gemm(h, py, px, S)
                y = d.down(py, (S, O)).astype(np.float64)
            dx = run(session, h, dy, I).astype(np.float64)
            lhs, rhs = (y * dy).sum(1), (dx * x).sum(1)
            mag = ((np.abs(x).astype(np.float64) @ np.abs(w).T) * np.abs(dy)).sum(1)
            assert (np.abs(lhs - rhs) <= (gemm_tol(O) + gemm_tol(I) + sum_tol(2 * max(O, I))) * mag).all()
        finally:
            session.free(h)


@pytest.mark.parametrize("S", [3, 70])
def test_graph_replays(session, S):
    b = session.b
    rng = np.random.default_rng(23 + S)
    O, I = 1024, 384
    h, _ = matrix(session, rng, "i4h", O, I)
    try:
        dy, other = rng.standard_normal((S, O)).astype(np.float32), rng.standard_normal((900, O)).astype(np.float32) * 3
        with Bufs(b) as d:
            py, px, po, pq = d.up(dy), d.up(np.zeros((S, I), np.float32)), d.up(other), d.up(np.zeros((900, I), np.float32))
            assert b.hip_gemm_t_dev(h, px, py, S)
            eager = d.down(px, (S, I))
            with hiprt.Graph(b.hip_stream(0)) as g:
                assert b.hip_gemm_t_dev(h, px, py, S)
            for rep in range(3):
                assert b.hip_fill_random_u8(0, px, S * I * 4, 5 + rep)
                g.launch()
                got = d.down(px, (S, I))
                assert np.array_equal(got.view(np.uint32), eager.view(np.uint32)), rep
                # eager work between the replays, larger than the capture's workspace
                assert b.hip_gemm_t_dev(h, pq, po, 900 - rep)
    finally:
        session.free(h)


def test_refusals(session):
    b = session.b
    rng = np.random.default_rng(1)
    h, _ = matrix(session, rng, "i4h", 32, 32)
    try:
        with Bufs(b) as d:
            p = d.up(np.zeros((1, 32), np.float32))
            assert not b.hip_gemm_t_dev(None, p, p, 1)
            assert not b.hip_gemm_t_dev(h, None, p, 1)
            assert not b.hip_gemm_t_dev(h, p, None, 1)
            q = d.up(np.zeros((2, 32), np.float32))
            assert not b.hip_gemm_t_dev(h, p, q, 0)
            assert not b.hip_gemm_t_dev(h, p, q, 65536)
            for dx, dy in ((q, q), (q, q + 128), (q + 4, q)):   # dx over dy
                assert not b.hip_gemm_t_dev(h, dx, dy, 2 if dx != dy else 1)
            assert b.hip_gemm_t_dev(h, q, q + 128, 1)           # next to it
    finally:
        session.free(h)


@pytest.mark.parametrize("kind", ["i4h", "i4f", "fp4"])
@pytest.mark.parametrize("O", [2050, 4100, 9001, 16500])
def test_built_rows_of_many_columns(session, monkeypatch, kind, O):
    """Rows of dy that the build holds in two, four or eight slots a thread, and
    beyond 16384 columns reads a second time."""
    monkeypatch.setenv("COLI_HIP_GEMM_T", "many")
    test_matches_dense(session, kind, O, 70, 3)


def test_scales_are_counted(session):
    """The second copy of the scales is in the tensor's bytes and the device's statistics while it is held."""
    b = session.b
    n, byt = C.c_size_t(), C.c_size_t()

    def stats():
        b.cuda_stats(0, C.byref(n), C.byref(byt))
        return byt.value

    rng = np.random.default_rng(2)
    O, I = 200, 300
    for kind, planes in (("i4h", 1), ("i4f", 2), ("fp4", 1)):
        start = stats()
        h, _ = matrix(session, rng, kind, O, I)
        loaded, own = stats(), b.cuda_tensor_bytes(h)
        run(session, h, np.ones((2, O), np.float32), I)
        # tile quads of 128 columns, four groups each, an exponent a group; rows by 32
        extra = planes * 3 * 4 * 28 * 16 + 3 * 4 * 4
        assert stats() - loaded == extra and b.cuda_tensor_bytes(h) - own == extra
        run(session, h, np.ones((2, O), np.float32), I)
        assert stats() - loaded == extra
        session.free(h)
        assert stats() == start


def test_first_gradient_is_not_captured(session):
    """Under capture a tensor's first gradient, which lays out its scales, is
    refused; the capture goes on, and calls outside it are right."""
    b = session.b
    rng = np.random.default_rng(43)
    O, I, S = 96, 160, 5
    h, w = matrix(session, rng, "i4h", O, I)
    try:
        dy = rng.standard_normal((S, O)).astype(np.float32)
        with Bufs(b) as d:
            py, px, pz = d.up(dy), d.up(np.zeros((S, I), np.float32)), d.up(np.zeros((S, O), np.float32))
            assert b.cuda_pipe_gemm(h, pz, px, S)
            with hiprt.Graph(b.hip_stream(0)) as g:
                assert not b.hip_gemm_t_dev(h, px, py, S)
                assert b.cuda_pipe_gemm(h, pz, px, S)
            want = dy.astype(np.float64) @ w
            mag = np.abs(dy).astype(np.float64) @ np.abs(w)
            for _ in range(2):
                assert b.hip_gemm_t_dev(h, px, py, S)
                close(d.down(px, (S, I)), want, mag, gemm_tol(O))
                g.launch()
            assert np.isfinite(d.down(pz, (S, O))).all()
    finally:
        session.free(h)


def spread_tol(kind, w, smax):
    """Error of a weight beyond its 6 x 2^-22 (gemm_tol): what fp16 cannot hold
    of a scale far below its column group's largest, which lies in [2^11, 2^12)
    there (MXFP4: at 2^12). int4: a scale, the odd rows' over 16, is rounded to
    2^-25, so by 2^-21 / 2^11 of the largest, times a nibble of at most 8, and
    lo to 2^-25 once more. MXFP4: e8m0 scales are powers of two, held down to
    2^-24, so at most 2^-25 / 2^12 of the largest is lost, times 6, and the
    product is rounded to 2^-25."""
    return 6 * 2.0 ** -22 * np.abs(w) + (7 * 2.0 ** -37 if kind == "fp4" else 8 * 2.0 ** -32 + 2.0 ** -36) * smax


@pytest.mark.parametrize("pin", ["few", "many"])
@pytest.mark.parametrize("kind", ["i4h", "i4f", "fp4"])
def test_weights_of_small_scales(session, monkeypatch, kind, pin):
    """One-hot rows of dy read weights whose scales lie 2^-16, 2^-30 and 2^-45
    below the column group's largest: off by no more than the bound under it."""
    monkeypatch.setenv("COLI_HIP_GEMM_T", pin)
    rng = np.random.default_rng(41)
    O, I = 80, 200
    down = np.array([0, 16, 30, 45])[np.arange(O) // 3 % 4]
    if kind == "fp4":
        q4, e8 = rand_mxfp4(rng, O, I)
        e8 = (e8 - down[:, None]).astype(np.uint8)
        h, w, s = session.upload_mxfp4(q4, e8, I, O), deq_mxfp4(q4, e8, I), 2.0 ** (e8.astype(np.float64) - 127)
    else:
        q4, sc = rand_i4(rng, O, I, 32, fp16_scales=False)
        sc = ((0.5 + sc) * 2.0 ** -down[:, None]).astype(np.float32)
        if kind == "i4h":   # (2^-30 and 2^-45 are below fp16: zero scales)
            sc = sc.astype(np.float16).astype(np.float32)
        h, w, s = session.upload(q4, sc, 4, I, O, 32), deq_i4(q4, sc, I, 32), sc.astype(np.float64)
    try:
        assert session.b.hip_tensor_kind(h) == ("i4h", "i4f", "fp4").index(kind)
        got = run(session, h, np.eye(O, dtype=np.float32), I)
        smax = np.repeat(s.max(0), 32)[None, :I]
        err = np.abs(got.astype(np.float64) - w)
        # (a result is rounded to f32: within the 6 x 2^-22)
        assert (err <= spread_tol(kind, w, smax)).all(), float((err / spread_tol(kind, w, smax)).max())
        # nothing is lost where the scales are within the range that fp16 holds whole
        exact = down <= {"i4h": 16, "i4f": -1, "fp4": 30}[kind]
        assert not err[exact].any()
    finally:
        session.free(h)
