"""Device memory that the shared workspaces hold, measured in a process of its
own (what other tests have captured or allocated does not count there)."""
import json
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = """
import ctypes as C, json, sys
import numpy as np
sys.path[:0] = [{root!r}, {root!r} + "/tests"]
from colibri_amd import hiprt
from colibri_amd.backend import Session
from quant_util import rand_mxfp4

I, O, ROWS = 16384, 64, 4000
q4, e8 = rand_mxfp4(np.random.default_rng(0), O, I)


def held(sizes, capture):
    s = Session(0)
    b = s.b
    free, total = C.c_size_t(), C.c_size_t()
    h = s.upload_mxfp4(q4, e8, I, O)
    x, y = b.cuda_pipe_alloc(0, ROWS * I * 4), b.cuda_pipe_alloc(0, ROWS * O * 4)

    def left():
        assert b.cuda_pipe_sync(0) and b.cuda_mem_info(0, C.byref(free), C.byref(total))
        return free.value

    assert b.cuda_pipe_gemm(h, y, x, 1)
    if capture:
        with hiprt.Graph(b.hip_stream(0)):
            assert b.cuda_pipe_gemm(h, y, x, 1)
    before = left()
    for S in sizes:
        assert b.cuda_pipe_gemm(h, y, x, S)
    out = before - left()
    for p in (x, y):
        b.cuda_pipe_free(0, p)
    s.free(h)
    s.close()
    return out


slowly = list(range(500, ROWS, 25)) + [ROWS]
print(json.dumps([held([ROWS], False), held(slowly, False), held(slowly, True)]))
"""


def test_growing_calls_hold_what_the_largest_needs():
    """A prefill that grows by 25 rows at a time: workspaces a quarter larger than
    the largest call's, as one call of that size takes (the outgrown ones are
    freed). Where a graph has been captured they are kept, and so doubled at each
    growth: less than four times the largest call's."""
    r = subprocess.run([sys.executable, "-c", CHILD.format(root=ROOT)], capture_output=True, text=True, timeout=110)
    assert r.returncode == 0, r.stderr[-2000:]
    once, grown, kept = json.loads(r.stdout.strip().splitlines()[-1])
    rows = 4000 * 16384 * 4     # fp16 hi + lo
    assert rows <= once <= 1.25 * rows + (96 << 20)
    assert grown <= 1.25 * rows + (96 << 20), (once, grown)
    assert kept <= 4 * once, (once, kept)


CYCLES = """
import ctypes as C, json, os, sys
import numpy as np
os.environ["COLI_HIP_MX"] = "1"
sys.path[:0] = [{root!r}, {root!r} + "/tests"]
from colibri_amd.backend import ColiHipMoeConfig, Session, f32p, tensor_array
from moe_ref import Layer, make_router_inputs

D, I, E, K, S = 2048, 128, 4, 2, 2000
rng = np.random.default_rng(0)
layer = Layer(rng, 7, D, I, E, shared=False)
x, W, _ = make_router_inputs(rng, S, D, E, K, 0, bias=False)
left = []
for _ in range(3):
    s = Session(0)
    b, m = s.b, C.c_void_p()
    hs = layer.upload(s)
    (g, _a), (u, _b), (d, _c) = (tensor_array([t[k] for t in hs[:E]]) for k in range(3))
    cfg = ColiHipMoeConfig(D, I, E, K, 0, 1, 0.0, 1.0, 0)
    assert b.hip_moe_create(C.byref(m), 0, C.byref(cfg), f32p(W), None, g, u, d, None, None, None)
    out = np.zeros((S, D), np.float32)
    assert b.hip_moe_forward(m, f32p(x), f32p(out), S, None, None, None)
    b.hip_moe_free(m)
    for t in hs:
        for h in t:
            s.free(h)
    s.close()
    s = Session(0)
    free, total = C.c_size_t(), C.c_size_t()
    assert s.b.cuda_mem_info(0, C.byref(free), C.byref(total))
    left.append(free.value)
    s.close()
print(json.dumps(left))
"""


def test_shutdown_returns_the_activation_pieces():
    """Sessions one after the other, each with a block-scaled layer of 2000 rows
    (its pieces: 4 MB an e4m3 plane), leave as much memory free."""
    r = subprocess.run([sys.executable, "-c", CYCLES.format(root=ROOT)], capture_output=True, text=True, timeout=110)
    assert r.returncode == 0, r.stderr[-2000:]
    left = json.loads(r.stdout.strip().splitlines()[-1])
    assert left[0] - left[2] < 4 << 20, left
