"""Without a GPU: the adapter, input-gradient and balance entry points refuse
cleanly when no device is initialised, and the balance reference's gradient is
the derivative of its loss."""
import ctypes as C

import numpy as np
import pytest

from balance_ref import balance
from colibri_amd import backend


def test_refused_without_a_device():
    b = backend.Backend()
    assert b.cuda_device_count() == 0
    buf = np.zeros(64, np.float32)
    p, h = buf.ctypes.data, C.c_void_p()
    assert not b.hip_lora_create(C.byref(h), 0, 8, 8, 1, 4, 0) and not h
    assert not b.hip_lora_set_dev(None, 0, p, p, 1, 1.0)
    assert not b.hip_lora_gemm_dev(None, None, p, p, 1, p)
    assert not b.hip_lora_grad_dev(None, None, p, p, 1, p, p, p, p)
    assert not b.hip_gemm_t_dev(None, p, p, 1)
    assert not b.hip_balance_dev(0, p, p, None, None, None, 1, 2, 4, 1, 0, p, p, p)
    assert not b.hip_balance_grad_dev(0, p, None, None, 1, 2, 4, 0, p, p, p, p)
    assert not b.hip_moe_last_balance_dev(None, None, None, 1, p, p, p)
    b.hip_lora_free(None)
    assert not buf.any()


@pytest.mark.parametrize("mode", [0, 1, 2, 3])
def test_balance_reference_gradient_is_the_derivative(mode):
    rng = np.random.default_rng(mode)
    T, E, K, h = 9, 6, 2, 1e-5
    z = rng.standard_normal((T, E)) * 2
    idx = np.argsort(-z, 1)[:, :K].astype(np.int32)
    off, mask = np.array([0, 4, 4, 8], np.int32), np.array([1, 1, 0, 1, 1, 1, 1, 1, 1], np.uint8)
    dl = np.array([0.7, 1.0, -2.0])
    g = balance(z, idx, None, mask, off, E, mode, dl, np.zeros((T, E)))[3]
    for t in range(T):
        for e in range(E):
            zz = [z.copy(), z.copy()]
            zz[0][t, e] += h
            zz[1][t, e] -= h
            up, dn = (float((balance(v, idx, None, mask, off, E, mode)[0] * dl).sum()) for v in zz)
            # h^2 of a third derivative of at most a few units, and 64-bit roundings over h
            assert abs((up - dn) / (2 * h) - g[t, e]) <= 1e-8
