"""The operators of language models at their edges, beside test_gpu_language_ops.py: waits that run out, infinite values,
rows and columns of a matrix that are faint against the others, matrices that are small as a whole, the
largest table."""
import ctypes as C

import numpy as np
import pytest

import language_ref as ref
import rusttensor_b200
from helpers import rng
from rusttensor_b200.frontend import EngineError
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


# ---- Muon: rows by themselves ---------------------------------------------------------------------------------------------------------


def rows_as_near_as_fp32(got, want, plain, x):
    """Every row against its own size.  X = D X' with rows of X' of norm 1: G = D G' D and the polynomial likewise, so that what a step adds up
    for row i has the factor d_i, and all of as_near_as_fp32's 301 U of one step hold for row i against its own norm, r_i.  Matrices whose
    rows and columns are not below sqrt(max(k, 64)) 2^-21 are held to 2^-40 (half a step of what is below 2^-22) instead: 2^-19 of a row, 32 U.  Their G
    and polynomial, too: an element of the latter is off by 4.775 * 2^-40 + 2^-39 < 2^-37.2, and a row of it, multiplied with X of norm 1, by as much (errors
    that are as often above as below): 2^-19.2 of a row of 2^-18 or more, 28 U.  So one step is off by 361 U of the row that it begins with; that is the last step's by a norm that is at most 1 / 0.63 of the result's, since a step multiplies singular values below 1.21 by
    between 0.63 and 3.4445; steps before grow as in fp32: three times what the same steps are off there."""
    norm = np.linalg.norm
    rows = norm(x.astype(np.float64), axis=1) / (norm(x.astype(np.float64)) + 1e-7)
    off = norm(got.astype(np.float64) - want, axis=1)
    allowed = 3 * norm(plain - want, axis=1) + 361 * ref.U * np.maximum(rows, norm(want, axis=1) / 0.63)
    worst = np.argmax(off / np.maximum(allowed, 1e-300))
    assert np.all(off <= allowed), (worst, off[worst], allowed[worst], rows[worst])


def check(capi, xs, steps=5):
    """Each matrix's rows and columns; all of the list in one call."""
    import torch

    d, outs = [capi.to_device(x) for x in xs], [capi.empty(x.shape) for x in xs]
    capi.call("orthogonalize_list", len(xs), pointers(d), capi.i64([x.shape[0] for x in xs]), capi.i64([x.shape[1] for x in xs]), steps, pointers(outs))
    for x, o in zip(xs, outs):
        if x.size > 1 << 20 and steps == 5:
            want, plain = steps_on_gpu(x, torch.float64), steps_on_gpu(x, torch.float32)
        else:
            want, plain = ref.orthogonalize(x, steps), ref.orthogonalize(x, steps, np.float32)
        got = o.numpy()
        rows_as_near_as_fp32(got, want, plain, x)
        rows_as_near_as_fp32(got.T, want.T, plain.T, x.T)


FACTORS = 2.0 ** -np.array([0, 4, 8, 12, 14, 16, 18, 20, 22, 24, 28, 32, 40, 60])


def graded(r, n, most=0):
    """Factors of n rows, in blocks, down to 2^-most; most rows have none."""
    f = np.ones(n)
    steps = FACTORS[FACTORS >= 2.0**-most]
    for k, block in enumerate(np.array_split(r.permutation(n)[: max(1, n // 2)], len(steps))):
        f[block] = steps[k]
    return f


@pytest.mark.parametrize("most", [8, 16, 20, 24, 60])
@pytest.mark.parametrize("side", ["rows", "columns", "both"])
def test_faint_rows_and_columns(capi, side, most):
    r = rng(61 + most)
    xs = []
    for shape in ((784, 128), (128, 784), (300, 260), (40, 700), (65, 64)):
        x = r.standard_normal(shape)
        if side != "columns":
            x = x * graded(r, shape[0], most)[:, None]
        if side != "rows":
            x = x * graded(r, shape[1], most)
        xs.append(x.astype(np.float32))
    check(capi, xs)
    check(capi, xs, 1)


def test_faint_rows_of_large_matrices(capi):
    """Tiles of pairs of CTAs; in one list with matrices that have no faint rows."""
    r = rng(62)
    shape = (1501, 1603)
    plain = matrix(r, shape)
    check(capi, [(r.standard_normal(shape) * graded(r, shape[0], 60)[:, None]).astype(np.float32), plain])
    check(capi, [(r.standard_normal(s) * graded(r, s[1], 32)).astype(np.float32) for s in [(1290, 1803)] * 2] + [matrix(r, (1803, 1290))] * 4)


def test_faint_copies_of_rows(capi):
    """Rows that are another row over again, but for a small factor, do not grow with the small singular values."""
    r = rng(63)
    x = r.standard_normal((200, 300))
    x[100:150] = x[:50] * FACTORS[np.arange(50) % len(FACTORS), None]
    check(capi, [x.astype(np.float32), x.T.astype(np.float32)])


@pytest.mark.parametrize("value", [1e-7, 1e-12, 1e-20, 1e-30])
def test_small_matrices_are_not_lost(capi, value):
    """The norm is not much more than what is added to it, or less: the result is small, and has a value."""
    r = rng(64)
    check(capi, [(value * r.standard_normal(s) / s[0]).astype(np.float32) for s in ((40, 30), (150, 200), (700, 512))])


@pytest.mark.parametrize("value", [np.nan, np.inf])
@pytest.mark.parametrize("shape", [(1, 6), (6, 1), (65, 3), (30, 700), (1290, 1803)])
def test_matrices_with_a_special_value(capi, shape, value):
    """All of the result is NaN; that of the list's other matrix is what it is by itself."""
    r = rng(70)
    x, y = matrix(r, shape), matrix(r, (33, 130))
    x[0, -1] = value
    d, outs = [capi.to_device(a) for a in (x, y)], [capi.empty(a.shape) for a in (x, y)]
    capi.call("orthogonalize_list", 2, pointers(d), capi.i64([shape[0], 33]), capi.i64([shape[1], 130]), 5, pointers(outs))
    assert np.isnan(outs[0].numpy()).all()
    as_near_as_fp32(outs[1].numpy(), ref.orthogonalize(y), ref.orthogonalize(y, 5, np.float32))


def test_sparse_rows(capi):
    """Rows of zeros stay zeros; rows with a single element, down to small ones; all of it the same in every run."""
    r = rng(65)
    x = r.standard_normal((260, 333)).astype(np.float32)
    x[::3] = 0
    for k, i in enumerate(range(0, 240, 6)):
        x[i, (7 * i) % 333] = 2.0 ** -(k + 1)
    check(capi, [x, np.ascontiguousarray(x.T)])
    d, outs = capi.to_device(x), [capi.empty(x.shape) for _ in range(3)]
    for o in outs:
        capi.call("orthogonalize_list", 1, pointers([d]), capi.i64([260]), capi.i64([333]), 5, pointers([o]))
    got = [o.numpy() for o in outs]
    assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])
    assert np.all(got[0][3::6] == 0)


def test_a_graph_goes_by_its_inputs(capi):
    """Captured with matrices that have no faint rows, replayed with some that do and back: the bits of a call on the same inputs."""
    r = rng(72)
    shapes = [(300, 200), (1290, 1803)]
    plain = [matrix(r, s) for s in shapes]
    faint = [(x * graded(r, x.shape[0], 60)[:, None]).astype(np.float32) for x in plain]
    d, outs = [capi.to_device(x) for x in plain], [capi.empty(s) for s in shapes]
    args = (len(shapes), pointers(d), capi.i64([s[0] for s in shapes]), capi.i64([s[1] for s in shapes]), 5, pointers(outs))
    fill = lambda xs: [capi.check(capi.lib.rt_memcpy_h2d(capi.ctx, t.ptr, x.ctypes.data_as(C.c_void_p), C.c_size_t(x.nbytes))) for x, t in zip(xs, d)]  # noqa: E731
    want = []
    for xs in (plain, faint, [plain[0], faint[1]]):
        fill(xs)
        capi.call("orthogonalize_list", *args)
        want.append([o.numpy() for o in outs])
    graph = C.c_void_p()
    capi.call("graph_begin")
    capi.call("orthogonalize_list", *args)
    capi.call("graph_end", C.byref(graph))
    for xs, w in zip((plain, faint, [plain[0], faint[1]], plain), want + want[:1]):
        fill(xs)
        capi.call("graph_launch", graph)
        assert all(np.array_equal(o.numpy(), b) for o, b in zip(outs, w))
    capi.call("graph_destroy", graph)


# ---- embeddings ---------------------------------------------------------------------------------------------------------------------------


def test_the_largest_table_of_the_engine(gpu_engine):
    """2^24 rows: every number is one of its own, the next one is padding as it is rounded; a row more is refused."""
    e, rows = gpu_engine, 2**24
    table = np.arange(rows, dtype=np.float32).reshape(rows, 1)
    t = e.tensor(table, requires_grad=True)
    ids = np.array([rows - 1, rows - 2, 0, rows, rows + 1])
    out = e.ops.embedding(t, e.tensor(ids.astype(np.float32)))
    assert out.numpy().ravel().tolist() == [rows - 1, rows - 2, 0, 0, 0]
    e.ops.sum(out).backward()
    assert np.flatnonzero(t.grad.numpy()).tolist() == [0, rows - 2, rows - 1]
    with pytest.raises(EngineError) as ei:
        e.ops.embedding(e.tensor(np.zeros((rows + 1, 1), np.float32)), e.tensor(ids.astype(np.float32)))
    assert ei.value.kind == "InvalidOperation"


@pytest.mark.parametrize("n", [1, 1000, 3000001])
def test_token_ids_in_place(capi, n):
    """Numbers and what is none, in the place that they are read from: the same as elsewhere."""
    r = rng(71)
    x = r.integers(-3, 2**24, n).astype(np.float32)
    x[::7] += 0.5
    x[::11] = np.nan
    d, out = capi.to_device(x), capi.empty((n,))
    capi.call("token_ids", d.ptr, i64(n), out.ptr)
    capi.call("token_ids", d.ptr, i64(n), d.ptr)
    want = np.where((x >= 0) & (x == np.trunc(x)), np.nan_to_num(x), -1).astype(np.int64)
    assert np.array_equal(out.numpy().view(np.int32), want) and np.array_equal(d.numpy().view(np.int32), want)
