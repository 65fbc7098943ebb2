"""Without a GPU: the sorted-rows and 4-bit entry points refuse cleanly when no
device is initialised, and the references are what they stand for."""
import ctypes as C

import numpy as np

from colibri_amd import backend
from mx_ref import mx_quant, pack, plan
from quant_util import E2M1, deq_mxfp4


def test_refused_without_a_device():
    b = backend.Backend()
    assert b.cuda_device_count() == 0
    buf = np.zeros((16, 64), np.float32)
    p, h = [r.ctypes.data for r in buf], C.c_void_p()
    f = [C.cast(v, C.POINTER(C.c_float)) for v in p]
    assert not b.hip_dispatch_dev(0, p[0], None, None, 2, 4, 3, p[1], 8, p[2], p[3], p[4], p[5])
    assert not b.hip_dispatch_dev(0, None, None, None, 0, 4, 3, None, 0, p[2], None, None, None)
    assert not b.hip_combine_dev(0, p[0], 0, p[1], p[2], 2, 3, 4, 5, p[3])
    assert not b.hip_combine_grad_dev(0, p[0], 0, p[1], p[2], p[3], 2, 3, 4, 5, p[4], p[5])
    assert not b.hip_mxfp4_quantize_dev(0, p[0], 0, 2, 8, p[1], p[2])
    assert not b.hip_mxfp4_dequantize_dev(0, p[0], p[1], 2, 8, p[2], 0)
    assert not b.hip_tensor_quantize_mxfp4(C.byref(h), p[0], 0, 8, 2, 0) and not h
    assert not b.hip_fp4_matmul_a4(None, f[0], f[1], 1)
    assert not b.hip_fp4_matmul_a4_dev(None, p[0], p[1], 1)
    assert not b.hip_experts_create(C.byref(h), 0, 1, C.cast(p[0], C.POINTER(C.c_void_p)), None, 0.0) and not h
    assert not b.hip_experts_a4_dev(None, p[0], p[1], 1, None, 1, p[2], 1)
    b.hip_experts_free(None)
    assert not buf.any()


def test_quantizer_reference():
    """Nearest code under the scale, ties even, and the scale the smallest power of two that saturates nothing."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((5, 70)) * np.exp(3 * rng.standard_normal((5, 70)))
    codes, byte, val = mx_quant(x)
    assert np.array_equal(deq_mxfp4(pack(codes), byte, 70), val)
    scale = np.repeat(2.0 ** (byte - 127.0), 32, 1)[:, :70]
    every = np.abs(x[:, :, None] - E2M1 * scale[:, :, None])
    assert (np.abs(x - val) <= every.min(2)).all() and (np.abs(x) <= 6 * scale).all()
    top = np.abs(np.pad(x, ((0, 0), (0, 26)))).reshape(5, 3, 32).max(2)
    assert (top > 3 * 2.0 ** (byte - 127.0)).all()
    ties = np.array([[6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.75, -5.0]])
    assert np.array_equal(mx_quant(ties)[2], [[6, 0, 1, 1, 2, 2, 4, 4, -1, -4]])


def test_plan_reference():
    off, src, pos = plan(np.array([[2, 0], [0, 0], [5, 1], [1, 2]]), np.array([2, 2, 2, 1]), np.array([1, 1, 1, 1]), 3)
    assert off.tolist() == [0, 3, 5, 6] and src.tolist() == [1, 2, 3, 5, 6, 0]
    assert pos.tolist() == [[5, 0], [1, 2], [-1, 3], [4, -1]]
