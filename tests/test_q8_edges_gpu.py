"""Rows and products in eight bits at the ends of what the calls allow, against the restatement of tests/q8_reference.py."""
import ctypes

import numpy as np
import pytest

import test_q8_gpu as q8
from test_q8_gpu import dev  # noqa: F401  (a fixture)
from test_recorded_launches_gpu import Driver

pytestmark = pytest.mark.gpu


# --------------------------------------------------------------------------- rows that are longer than shared memory

# rows and residual of f32, more rows than there are threads for at once: from dim 28168 on the two rows are longer than the shared memory that a ring has
@pytest.mark.parametrize("rows, dim, w_f32, outputs, place", [(297, 28160, False, "q", "residual"), (297, 28168, True, "qy", "residual"), (300, 32768, False, "q", "x"), (300, 32761, True, "qy", ""),
                                                              (301, 30001, False, "y", "nothing")])
def test_norms_of_the_longest_rows(t0, rt, dev, rows, dim, w_f32, outputs, place):  # noqa: F811
    q8.test_rmsnorm(t0, rt, dev, rows, dim, True, "f32", w_f32, outputs, place)

# --------------------------------------------------------------------------- errors

def test_an_error_is_one_calls_own(t0, rt, dev):  # noqa: F811
    # a launch that the runtime refuses (its stream is in a recording that was broken off) answers with the error; the call behind it, whose launch is fine, does not
    driver = Driver()
    x, q, s = dev.up(np.ones((4, 64), np.float32)), dev.up(np.zeros((4, 64), np.int8)), dev.up(np.zeros(4, np.float32))
    y, w = dev.up(np.zeros((4, 4), np.float32)), dev.up(np.ones((700, 64), np.int8))
    ws, big = dev.up(np.ones(700, np.float32)), dev.up(np.zeros((700, 700), np.float32))
    at = lambda b: b.gpu_addr()  # noqa: E731
    filled = rt.alloc(4096)
    size = dict(n_rows=4, dim=64)
    calls = [lambda: rt.q8_quant(rt.q8_quant_args(at(x), at(q), at(s), x_f32=True, **size)), lambda: rt.q8_dequant(rt.q8_dequant_args(at(q), at(s), at(x), out_f32=True, **size)),
             lambda: rt.q8_rmsnorm(rt.q8_rmsnorm_args(at(x), at(ws), eps=1e-5, x_f32=True, weight_f32=True, q=at(q), scales=at(s), **size)),
             lambda: rt.q8_gemm(rt.q8_gemm_args(at(q), at(s), at(w), at(ws), at(y), m=4, n=4, k=64)),
             lambda: rt.q8_gemm(rt.q8_gemm_args(at(w), at(ws), at(w), at(ws), at(big), m=700, n=700, k=64))]
    for call in calls:
        call()
        rt.synchronize()
        stream, graph = ctypes.c_void_p(rt.stream()), ctypes.c_void_p()
        driver.call("cuStreamBeginCapture_v2", stream, 1)                   # 1 = this thread's recording
        broken = driver.cu.cuStreamSynchronize(stream)                      # not allowed in a recording: breaks it off
        try:
            with pytest.raises(t0.T0Error) as e:
                call()
        finally:
            ended = driver.cu.cuStreamEndCapture(stream, ctypes.byref(graph))
        assert broken != 0 and ended != 0 and e.value.code == 2, (broken, ended, e.value.code)
        rt.fill_uniform_bf16(filled.gpu_addr(), 100, 1)
        call()
        rt.synchronize()
    with pytest.raises(t0.T0Error) as e:                                    # more memory than any GPU has
        rt.alloc(1 << 50)
    assert e.value.code == 2
    rt.fill_uniform_bf16(filled.gpu_addr(), 100, 1)
    rt.synchronize()
    filled.free()
