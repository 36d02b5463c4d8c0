"""The operators of language models at their edges, beside test_gpu_language_ops.py: waits that run out, infinite values."""
import ctypes as C

import numpy as np
import pytest

import language_ref as ref
import rusttensor_b200
from helpers import rng
from test_gpu_language_ops import as_near_as_fp32, f32, i64, matrix, pointers, steps_on_gpu

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


@pytest.mark.parametrize("steps,batch,hidden", [(5, 2, 8), (40, 2, 8), (300, 3, 33), (2000, 1, 64), (9000, 1, 320), (6007, 3, 257)])
def test_gated_scan_of_infinite_values(capi, steps, batch, hidden):
    """An infinite state stays infinite while the gates are above zero, however small their product is, and so does an infinite gradient."""
    r = rng(66)
    f = r.uniform(-14, 2, (steps, batch, hidden)).astype(np.float32)
    v, dh, h0 = (r.standard_normal(s).astype(np.float32) for s in (f.shape, f.shape, (batch, hidden)))
    h0[0, 0], h0[-1, 2] = np.inf, -np.inf
    v[steps // 2, 0, 3], dh[steps // 2, -1, 4] = -np.inf, np.inf
    d = [capi.to_device(a) for a in (f, v, h0, dh)]
    h, df, dv, dh0 = (capi.empty(s) for s in (f.shape, f.shape, f.shape, h0.shape))
    sizes = i64(steps), i64(batch), i64(hidden)
    capi.call("gated_scan", d[0].ptr, d[1].ptr, i64(hidden), d[2].ptr, *sizes, h.ptr)
    got = h.numpy()
    want, bound = ref.scan(f, v, h0)  # timestep by timestep
    infinite = np.isinf(want)
    assert infinite[:, 0, 0].all() and infinite[:, -1, 2].all() and infinite[steps // 2 :, 0, 3].all()
    assert np.array_equal(got[infinite], want[infinite])
    assert np.all(np.abs(got - want)[~infinite] <= bound[~infinite])
    finite = np.where(infinite, 0, got).astype(np.float32)  # states for the gradient
    capi.call("gated_scan_backward", d[0].ptr, d[1].ptr, i64(hidden), None, capi.to_device(finite).ptr, d[3].ptr, *sizes, df.ptr, dv.ptr, i64(hidden), dh0.ptr)
    rest = 1 / (1 + np.exp(f.astype(np.float64)))
    assert np.array_equal(np.isposinf(dv.numpy()[: steps // 2 + 1, -1, 4]), (rest > 0)[: steps // 2 + 1, -1, 4])
    assert np.isposinf(dh0.numpy()[-1, 4]) and np.isfinite(dv.numpy()[steps // 2 + 1 :]).all()


def test_gated_scan_forgets_entirely(capi):
    """A gate of zero leaves nothing of the state, in the middle of a stretch of small gates either."""
    r = rng(67)
    steps, hidden = 500, 40
    f = r.uniform(-14, -7, (steps, 1, hidden)).astype(np.float32)
    v = np.zeros_like(f)
    f[250] = -np.inf
    h0, h = capi.to_device(np.full((1, hidden), 1e30)), capi.empty(f.shape)
    d = [capi.to_device(a) for a in (f, v)]
    capi.call("gated_scan", d[0].ptr, d[1].ptr, i64(hidden), h0.ptr, i64(steps), i64(1), i64(hidden), h.ptr)
    assert np.all(h.numpy()[250:] == 0)


@pytest.mark.parametrize("shapes", [[(784, 128), (128, 10)], [(2000, 70)], [(1501, 1603)], [(1290, 1803)] * 5], ids=lambda s: f"{len(s)}x{s[0][0]}x{s[0][1]}")
def test_a_wait_of_muon_that_runs_out(shapes):
    """Blocks that do not wait for one another between two products: the kernel ends, the next synchronising call says so, and the parameters are as
    they were; the calls after it are right."""
    import torch

    api, r = rusttensor_b200.CApi(), rng(69)
    host, ones = [matrix(r, s) for s in shapes], [np.ones(s, np.float32) for s in shapes]
    g, m, p = ([api.to_device(x) for x in xs] for xs in (host, [0 * x for x in ones], ones))
    args = (len(shapes), pointers(p), pointers(g), pointers(m), api.i64([s[0] for s in shapes]), api.i64([s[1] for s in shapes]))
    api.call("lstm_sequence_polls", i64(0))
    api.call("muon_step_multi", *args, f32(-1.0), f32(0.0), 0, f32(0.0), 5, f32(1.0))
    code = C.c_int(0)
    with pytest.raises(Exception, match="gave up"):
        api.call("device_status", C.byref(code))
    assert code.value == 97
    api.call("device_status", C.byref(code))
    assert code.value == 0
    assert all(np.array_equal(x.numpy(), one) for x, one in zip(p, ones))
    api.call("lstm_sequence_polls", i64(-1))
    api.call("orthogonalize_list", len(shapes), pointers(g), *args[4:], 5, pointers(p))
    for x, d in zip(host, p):
        as_near_as_fp32(d.numpy(), steps_on_gpu(x, torch.float64), steps_on_gpu(x, torch.float32))
    api.close()
