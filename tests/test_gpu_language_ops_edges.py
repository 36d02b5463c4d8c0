"""The operators of language models at their edges, beside test_gpu_language_ops.py: waits that run out."""
import ctypes as C

import numpy as np
import pytest

import language_ref as ref
import rusttensor_b200
from helpers import rng
from test_gpu_language_ops import i64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("steps,batch,hidden", [(700, 1, 40), (9000, 1, 320), (6007, 3, 257)])
def test_a_wait_of_the_recurrence_that_runs_out(steps, batch, hidden, backward):
    """Blocks that do not wait for what another one sends: the kernel ends, the next synchronising call says so, the calls after it are right."""
    api, r = rusttensor_b200.CApi(), rng(68)
    f, v, dh = (r.standard_normal((steps, batch, hidden)).astype(np.float32) for _ in range(3))
    zero = np.zeros((batch, hidden), np.float32)
    d = [api.to_device(a) for a in (f, v, dh)]
    h, df, dv, dh0 = (api.empty(s) for s in (f.shape, f.shape, f.shape, zero.shape))
    sizes = i64(steps), i64(batch), i64(hidden)

    def forward():
        api.call("gated_scan", d[0].ptr, d[1].ptr, i64(hidden), None, *sizes, h.ptr)

    def gradient():
        api.call("gated_scan_backward", d[0].ptr, d[1].ptr, i64(hidden), None, h.ptr, d[2].ptr, *sizes, df.ptr, dv.ptr, i64(hidden), dh0.ptr)

    forward()
    api.call("lstm_sequence_polls", i64(0))
    gradient() if backward else forward()
    code = C.c_int(0)
    with pytest.raises(Exception, match="gave up"):
        api.call("device_status", C.byref(code))
    assert code.value == 82
    api.call("device_status", C.byref(code))
    assert code.value == 0
    api.call("lstm_sequence_polls", i64(-1))
    forward()
    gradient()
    got = h.numpy()
    want, bound = ref.scan(f, v, zero)
    assert np.all(np.abs(got - want) <= bound)
    for g, (x, b) in zip((df, dv, dh0), ref.scan_backward(f, v, zero, got, dh)):
        assert np.all(np.abs(g.numpy() - x) <= b)
    api.close()
