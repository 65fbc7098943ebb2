"""Device buffers, quantized matrices and 64-bit references of the adapter,
input-gradient and balance operators' tests."""
import ctypes as C

import numpy as np

from quant_util import deq_i4, deq_mxfp4, rand_i4, rand_mxfp4

KINDS = ("i4h", "i4f", "fp4", "row4", "gen")


class Bufs:
    """Device copies of host arrays, freed together."""

    def __init__(self, b, device=0):
        self.b, self.device, self.held = b, device, []

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        for p in self.held:
            self.b.cuda_pipe_free(self.device, p)

    def up(self, a):
        a = np.ascontiguousarray(a)
        p = self.b.cuda_pipe_alloc(self.device, max(16, a.nbytes))
        assert p
        self.held.append(p)
        assert self.b.cuda_pipe_upload(self.device, p, a.ctypes.data_as(C.c_void_p), a.nbytes)
        return p

    def put(self, p, a):
        a = np.ascontiguousarray(a)
        assert self.b.cuda_pipe_upload(self.device, p, a.ctypes.data_as(C.c_void_p), a.nbytes)

    def down(self, p, shape, dtype=np.float32):
        out = np.empty(shape, dtype)
        assert self.b.cuda_pipe_sync(self.device)
        assert self.b.cuda_pipe_download(self.device, p, out.ctypes.data_as(C.c_void_p), out.nbytes)
        return out


def matrix(session, rng, kind, O, I):
    """(handle, dense 64-bit weights [O, I]) of a random matrix of a storage kind."""
    if kind == "fp4":
        q4, e8 = rand_mxfp4(rng, O, I)
        return session.upload_mxfp4(q4, e8, I, O), deq_mxfp4(q4, e8, I)
    gs = {"row4": 0, "gen": 40}.get(kind, 32)
    q4, sc = rand_i4(rng, O, I, gs, fp16_scales=kind != "i4f")
    return session.upload(q4, sc, 2 if kind == "row4" else 4, I, O, gs), deq_i4(q4, sc, I, gs)


def bits(dtype, a):
    """The values of `a` in an adapter dtype (0 f32, 1 fp16, 2 bf16): (stored array, values in 64 bits)."""
    a = np.ascontiguousarray(a, np.float32)
    if dtype == 0:
        return a, a.astype(np.float64)
    if dtype == 1:
        h = a.astype(np.float16)
        return h, h.astype(np.float64)
    u = a.view(np.uint32).astype(np.uint64)
    u = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return u, (u.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def gemm_tol(K):
    """Error of a product of K terms on fp16 hi + lo operands, relative to the sum
    of the terms' magnitudes. dy as hi + lo is off by at most 2^-22. A weight of
    an f32 scale by 3 x 2^-22: the scale as two fp16, 2^-22, and lo, which holds
    the first product's rounding (2^-11 of the weight) and n times the scale's
    second part (2^-11 again), so up to 2^-10, rounded by 2^-11 (fp16 scales: an
    exact weight). The product of the two lo parts, left out: 2^-10 2^-11 =
    2 x 2^-22. Together 6 x 2^-22 a term.
    The f32 sums add at most 3 ceil(K / 16) + 32 times (three products a step of
    16, joins of splits), each off by at most 2^-23 of the partial sum (an MFMA
    sums its 16 products in one go, allowed one more 2^-23 here)."""
    return 6 * 2.0 ** -22 + (6 * ((K + 15) // 16) + 32) * 2.0 ** -23


def sum_tol(n):
    """Error of an f32 sum of n products, relative to the terms' magnitudes: a
    rounding a product and one an addition, 2^-24 each, and 16 for joins."""
    return (2 * n + 16) * 2.0 ** -24


def close(got, ref, mag, tol, what=""):
    """|got - ref| <= tol mag element by element (mag: sum of |terms|)."""
    err = np.abs(got.astype(np.float64) - ref)
    bad = ~(err <= tol * mag + 1e-30)
    assert not bad.any(), (what, int(bad.sum()), float((err / np.maximum(mag, 1e-30)).max()), tol,
                           [tuple(int(v) for v in i) for i in np.argwhere(bad)[:4]])
