"""Token embeddings, the gated linear recurrence and Muon on the GPU, through the C ABI and the engine, against their plain forms in 64 bits
(language_ref.py, which also says how far fp32 may be off): from one token to long sequences, odd sizes, strides and unaligned addresses,
padding, infinities, and runs of them together as a model is trained."""
import ctypes as C

import numpy as np
import pytest

import language_ref as ref
import rusttensor_b200
from helpers import rng

pytestmark = pytest.mark.gpu

i64, f32 = C.c_int64, C.c_float


def pointers(arrays):
    return (C.c_void_p * len(arrays))(*[a.ptr.value for a in arrays])


def device_ids(capi, ids):
    return capi.to_device(np.asarray(ids, np.int32).view(np.float32))


def offset(d, floats):
    return C.c_void_p(d.ptr.value + 4 * floats)


def within(got, want, bound):
    return np.all(np.abs(got - want) <= bound)


# ---- embeddings -----------------------------------------------------------------------------------------------------------------------

# (rows, cols, tokens)
TABLES = [(1, 1, 1), (65, 512, 1), (65, 512, 64), (3, 7, 100), (300, 4, 33), (1000, 130, 257), (257, 1028, 31), (50, 2500, 3), (70000, 3, 5000), (2, 64, 0)]


def tokens(r, rows, n, padding=True):
    ids = np.minimum(np.exp(r.uniform(0, np.log(rows + 1), n)).astype(np.int64) - 1, rows - 1)
    if padding and n > 4:
        ids[r.integers(0, n, n // 5 + 1)] = -1
        ids[r.integers(0, n)] = rows
        ids[r.integers(0, n)] = 2**31 - 1
    return ids


@pytest.mark.parametrize("rows,cols,n", TABLES)
@pytest.mark.parametrize("shift", [0, 1])
def test_embedding(capi, rows, cols, n, shift):
    """`shift`: the table and the result one float behind a 16-byte boundary."""
    r = rng(rows + cols + n)
    table, ids = r.standard_normal((rows, cols)).astype(np.float32), tokens(r, rows, n)
    d, di, out = capi.to_device(np.concatenate([np.zeros(shift, np.float32), table.ravel()])), device_ids(capi, ids), capi.to_device(np.full(n * cols + shift + 8, 7.0))
    capi.call("embedding", offset(d, shift), i64(rows), i64(cols), di.ptr, i64(n), f32(1.7), offset(out, shift))
    got = out.numpy()
    assert np.array_equal(got[shift : shift + n * cols].reshape(n, cols), ref.embedding(table, ids, 1.7))
    assert np.all(got[:shift] == 7) and np.all(got[shift + n * cols :] == 7)


@pytest.mark.parametrize("accumulate", [0, 1])
@pytest.mark.parametrize("rows,cols,n", TABLES + [(65, 512, 8192), (900, 132, 128), (900, 132, 129), (2, 300, 127), (5, 36, 20000), (40000, 20, 70000), (300, 8, 140001), (5000, 12, 2048), (130, 33, 2049), (7, 8, 1921), (70000, 40, 1), (70000, 40, 100)])
def test_embedding_backward(capi, rows, cols, n, accumulate):
    r = rng(rows + cols + n)
    g, ids, old = r.standard_normal((n, cols)).astype(np.float32), tokens(r, rows, n), r.standard_normal((rows, cols)).astype(np.float32)
    want, bound = ref.embedding_backward(g, ids, rows, 0.3, old if accumulate else None)
    dg, di, first = capi.to_device(g), device_ids(capi, ids), None
    for _ in range(2):
        d = capi.to_device(old)
        capi.call("embedding_backward", dg.ptr, di.ptr, i64(n), i64(rows), i64(cols), f32(0.3), d.ptr, accumulate)
        got = d.numpy()
        assert within(got, want, bound)
        assert first is None or np.array_equal(first, got)  # sums in a fixed order
        first = got
    untouched = ~np.isin(np.arange(rows), ids)
    assert np.array_equal(got[untouched], old[untouched] if accumulate else np.zeros_like(old[untouched]))


@pytest.mark.parametrize("count", [1, 33, 100, 3000, 70001])
def test_embedding_backward_of_one_token_only(capi, count):
    """All tokens the same, all of them padding, and rows of infinities and NaN that are padding."""
    r = rng(8)
    n, rows, cols = int(count), 40, 68
    g = r.standard_normal((n, cols)).astype(np.float32)
    for ids in (np.full(n, 39), np.full(n, 0), np.full(n, -5), np.full(n, 40)):
        bad = g.copy()
        if not 0 <= ids[0] < rows:
            bad[::3], bad[1::3] = np.inf, np.nan
        want, bound = ref.embedding_backward(g, ids, rows, 1.0)
        d, dg, di = capi.to_device(r.standard_normal((rows, cols))), capi.to_device(bad), device_ids(capi, ids)
        capi.call("embedding_backward", dg.ptr, di.ptr, i64(n), i64(rows), i64(cols), f32(1.0), d.ptr, 0)
        assert within(d.numpy(), want, bound)


@pytest.mark.parametrize("n", [60, 4000])
def test_embedding_backward_special_values(capi, n):
    """Infinities and NaN of a position go to its token's row and nowhere else, and rows without a token are zero whatever the scale is."""
    r = rng(n)
    rows, cols = 50, 20
    g, ids = r.standard_normal((n, cols)).astype(np.float32), r.integers(0, rows - 9, n)
    g[7, 3], g[11, 4] = np.nan, np.inf
    d, dg, di = capi.to_device(np.full((rows, cols), 3.0)), capi.to_device(g), device_ids(capi, ids)
    capi.call("embedding_backward", dg.ptr, di.ptr, i64(n), i64(rows), i64(cols), f32(2.0), d.ptr, 0)
    got = d.numpy()
    bad = np.zeros((rows, cols), bool)
    bad[ids[7], 3] = bad[ids[11], 4] = True
    assert np.isnan(got[ids[7], 3]) and np.isinf(got[ids[11], 4]) and np.isfinite(got[~bad]).all()
    capi.call("embedding_backward", dg.ptr, di.ptr, i64(n), i64(rows), i64(cols), f32(np.inf), d.ptr, 0)
    assert np.all(d.numpy()[rows - 9 :] == 0)


def test_embedding_scale_and_special_values(capi):
    """Padding is zero whatever the scale is; infinities and NaN of a table go where their rows go and nowhere else."""
    table = np.arange(12, dtype=np.float32).reshape(3, 4)
    table[1] = [np.inf, -np.inf, np.nan, 1]
    ids = [0, -1, 1, 2, 3]
    d, di, out = capi.to_device(table), device_ids(capi, ids), capi.empty((5, 4))
    for scale in (0.0, np.inf, np.nan, -1.0):
        capi.call("embedding", d.ptr, i64(3), i64(4), di.ptr, i64(5), f32(scale), out.ptr)
        with np.errstate(invalid="ignore"):
            want = table * np.float32(scale)
        assert np.array_equal(out.numpy(), np.stack([want[0], np.zeros(4), want[1], want[2], np.zeros(4)]), equal_nan=True)


def test_token_ids(capi):
    x = np.array([0, 1, 2.5, -1, -0.0, np.nan, np.inf, 2**31, 2**24 + 2, 2147483520.0], np.float32)
    d, out = capi.to_device(x), capi.empty(x.shape)
    capi.call("token_ids", d.ptr, i64(x.size), out.ptr)
    assert out.numpy().view(np.int32).tolist() == [0, 1, -1, -1, 0, -1, -1, -1, 2**24 + 2, 2147483520]


# ---- gated linear recurrence ---------------------------------------------------------------------------------------------------------------

# (steps, batch, hidden)
SEQUENCES = [(1, 1, 1), (1, 64, 512), (2, 3, 5), (7, 2, 33), (31, 1, 4), (128, 3, 64), (257, 2, 130), (1000, 1, 7), (1025, 5, 36), (2049, 1, 257), (33, 1, 4100), (5000, 1, 64), (9001, 2, 3), (6007, 3, 257), (9000, 1, 320), (20000, 1, 40)]


def sequence(r, steps, batch, hidden):
    f = (2 + 2 * r.standard_normal((steps, batch, hidden))).astype(np.float32)
    f[r.uniform(size=f.shape) < 0.02] = -np.inf
    f[r.uniform(size=f.shape) < 0.02] = np.inf
    f[r.uniform(size=f.shape) < 0.01] = -95.0
    f[r.uniform(size=f.shape) < 0.01] = 60.0
    return (f, *(r.standard_normal((steps, batch, hidden)).astype(np.float32) for _ in range(2)), r.standard_normal((batch, hidden)).astype(np.float32))


# how the gates lie: column blocks of one matrix, two matrices, rows with a gap and one float behind a 16-byte boundary
@pytest.mark.parametrize("layout", ["joined", "apart", "odd"])
@pytest.mark.parametrize("steps,batch,hidden", SEQUENCES)
def test_gated_scan(capi, steps, batch, hidden, layout):
    r = rng(steps + batch + hidden)
    f, v, dh, h0 = sequence(r, steps, batch, hidden)
    rows = steps * batch
    if layout == "joined":
        ld, at = 2 * hidden, (0, hidden)
    elif layout == "apart":
        ld, at = hidden, (0, rows * hidden)
    else:
        ld, at = hidden + 3, (1, rows * (hidden + 3) + 2)
    idx = [a + np.arange(rows)[:, None] * ld + np.arange(hidden) for a in at]
    size = max(int(i.max()) for i in idx) + 9
    gates = np.full(size, 5.0, np.float32)
    gates[idx[0]], gates[idx[1]] = f.reshape(rows, hidden), v.reshape(rows, hidden)
    # what is written behind the last row, or between rows, would show
    d, d0, h, g, dd = capi.to_device(gates), capi.to_device(h0), capi.to_device(np.full(rows * hidden + 8, 7.0)), capi.to_device(dh), capi.to_device(np.full(size, 7.0))
    dh0 = capi.to_device(np.full((batch, hidden), 7.0))
    sizes = (i64(steps), i64(batch), i64(hidden))
    for given in (True, False):
        start = d0.ptr if given else None
        zero = h0 if given else np.zeros_like(h0)
        capi.call("gated_scan", offset(d, at[0]), offset(d, at[1]), i64(ld), start, *sizes, h.ptr)
        got = h.numpy()
        assert np.all(got[rows * hidden :] == 7)
        got = got[: rows * hidden].reshape(steps, batch, hidden)
        want, bound = ref.scan(f, v, zero)
        assert within(got, want, bound)
        capi.call("gated_scan_backward", offset(d, at[0]), offset(d, at[1]), i64(ld), start, h.ptr, g.ptr, *sizes, offset(dd, at[0]), offset(dd, at[1]), i64(ld),
                  dh0.ptr if given else None)
        grads = dd.numpy()
        (df, bf), (dv, bv), (e0, b0) = ref.scan_backward(f, v, zero, got, dh)
        assert within(grads[idx[0]].reshape(f.shape), df, bf)
        assert within(grads[idx[1]].reshape(f.shape), dv, bv)
        if given:
            assert within(dh0.numpy(), e0, b0)
        rest = np.ones(size, bool)
        rest[idx[0]] = rest[idx[1]] = False
        assert np.all(grads[rest] == 7)


def test_gated_scan_goes_on_where_it_stopped(capi):
    """A sequence in one call, and timestep by timestep with the state updated in place: the same to the bound."""
    r = rng(21)
    steps, batch, hidden = 40, 6, 100
    f, v, _, h0 = sequence(r, steps, batch, hidden)
    state = capi.to_device(h0)
    want, bound = ref.scan(f, v, h0)
    for t in range(steps):
        df, dv = capi.to_device(f[t]), capi.to_device(v[t])
        capi.call("gated_scan", df.ptr, dv.ptr, i64(hidden), state.ptr, i64(1), i64(batch), i64(hidden), state.ptr)
        assert within(state.numpy(), want[t], bound[t])


def test_gated_scan_nan_stays_in_its_column(capi):
    r = rng(22)
    steps, batch, hidden = 700, 2, 24
    f, v, dh, h0 = sequence(r, steps, batch, hidden)
    f[300, 1, 3] = np.nan
    v[400, 0, 7] = np.inf
    d = [capi.to_device(x) for x in (f, v, h0, dh)]
    h, df, dv, dh0 = capi.empty(f.shape), capi.empty(f.shape), capi.empty(f.shape), capi.empty(h0.shape)
    sizes = (i64(steps), i64(batch), i64(hidden))
    capi.call("gated_scan", d[0].ptr, d[1].ptr, i64(hidden), d[2].ptr, *sizes, h.ptr)
    got = h.numpy()
    bad = np.zeros((batch, hidden), bool)
    bad[1, 3] = bad[0, 7] = True
    assert np.isnan(got[300:, 1, 3]).all() and np.isfinite(got[:300, 1, 3]).all() and np.isfinite(got[:400, 0, 7]).all() and not np.isfinite(got[400:420, 0, 7]).any()
    want, bound = ref.scan(f, v, h0)
    assert within(got[:, ~bad], want[:, ~bad], bound[:, ~bad])
    capi.call("gated_scan_backward", d[0].ptr, d[1].ptr, i64(hidden), d[2].ptr, h.ptr, d[3].ptr, *sizes, df.ptr, dv.ptr, i64(hidden), dh0.ptr)
    assert np.isnan(dh0.numpy()[1, 3]) and np.isfinite(dh0.numpy()[~bad]).all() and np.isfinite(df.numpy()[:, ~bad]).all()


# ---- Muon ------------------------------------------------------------------------------------------------------------------------------

SHAPES = [(1, 1), (1, 9), (7, 1), (3, 5), (16, 16), (33, 20), (64, 257), (127, 128), (129, 65), (200, 300), (784, 128), (130, 1000), (513, 140), (577, 640), (300, 260)]


def matrix(r, shape):
    return (r.standard_normal(shape) * np.exp(r.standard_normal((shape[0], 1)))).astype(np.float32)


def as_near_as_fp32(got, want, plain):
    """Errors of early steps grow by up to 3.9 a step, in fp32 as well: three times what the same steps in fp32 are off, and what one step may
    be off.  That is, with |X| = 1 (Frobenius, as all norms here) and so |G| <= 1, |b G + c G^2| <= 4.775 + 2.032 < 6.9: X is divided by a
    norm (2 U) and held to 22 bits (2 U).  A product of operands that are held to 22 bits is off by 2 U for each, 2 U for the lowest bits' product
    that is left out, 2 U for its sums: 8 U of the product of the norms.  G is off by 8 U + 2 * 4 U = 16 U, G^2 by 8 + 32 U = 40 U, the polynomial
    by 4.775 * 16 + 2.032 * 40 + 3 * 6.9 U = 179 U, its product with X by 179 + 6.9 * (8 + 4) U = 262 U, a X by 3.4445 * 5 U = 18 U, their sum by 2 U
    of 6.9 + 3.5: 301 U in all."""
    off, allowed = np.linalg.norm(got - want), 3 * np.linalg.norm(plain - want) + 301 * ref.U
    assert off <= allowed, (off, allowed)


@pytest.mark.parametrize("steps", [0, 1, 5])
def test_orthogonalize(capi, steps):
    r = rng(31)
    xs = [matrix(r, s) for s in SHAPES]
    d, outs = [capi.to_device(x) for x in xs], [capi.to_device(np.full(x.size + 8, 7.0)) for x in xs]
    rows, cols = (capi.i64([s[k] for s in SHAPES]) for k in (0, 1))
    first = None
    for _ in range(2):
        capi.call("orthogonalize_list", len(xs), pointers(d), rows, cols, steps, pointers(outs))
        got = [o.numpy() for o in outs]
        assert first is None or all(np.array_equal(a, b) for a, b in zip(first, got))
        first = got
    for x, o in zip(xs, got):
        assert np.all(o[x.size :] == 7)
        o = o[: x.size].reshape(x.shape)
        as_near_as_fp32(o, ref.orthogonalize(x, steps), ref.orthogonalize(x, steps, np.float32))
        if steps == 5 and min(x.shape) < 100 < max(x.shape):  # far from square: no tiny singular values
            s = np.linalg.svd(o, compute_uv=False)
            assert 0.6 < s.min() and s.max() < 1.25
    # in place, each by itself (how the reductions are shared among blocks, and so the last bits, goes by the whole list)
    for x, dx in zip(xs, d):
        capi.call("orthogonalize_list", 1, pointers([dx]), capi.i64([x.shape[0]]), capi.i64([x.shape[1]]), steps, pointers([dx]))
        as_near_as_fp32(dx.numpy(), ref.orthogonalize(x, steps), ref.orthogonalize(x, steps, np.float32))


# Lists whose products go by pairs of CTAs, with tiles of 128 columns and of 256, among them shared reductions, tall matrices and small ones that
# are edges only.
LARGE = [
    [(1501, 1603)],
    [(12000, 513), (513, 12001), (513, 12000)],
    [(701, 703)] * 6 + [(703, 690)] * 4 + [(3, 5), (1, 9)],
    [(1290, 1803)] * 5 + [(1803, 1290), (7, 1), (129, 300)],
    [(700, 20000)] * 3 + [(20001, 701)],
    [(3001, 2999)],
]


def steps_on_gpu(u, dtype):
    """Five Newton-Schulz steps; in 64 bits, or in fp32 as a plain program has them."""
    import torch

    x = torch.from_numpy(u).cuda().to(torch.float64)
    x = (x / (x.square().sum().sqrt() + 1e-7)).to(dtype)
    x = x.T if u.shape[0] > u.shape[1] else x
    for _ in range(5):
        g = x @ x.T
        x = 3.4445 * x + (-4.7750 * g + 2.0315 * (g @ g)) @ x
    return (x.T if u.shape[0] > u.shape[1] else x).double().cpu().numpy()


@pytest.mark.parametrize("shapes", LARGE, ids=lambda s: f"{len(s)}x{s[0][0]}x{s[0][1]}")
def test_muon_step_of_large_matrices(capi, shapes):
    """With a step of one, nothing kept of the parameters and no momentum, so that the parameters are the orthogonalised gradients themselves."""
    import torch

    r = rng(35)
    host = [matrix(r, s) for s in shapes]
    g, zeros = [capi.to_device(x) for x in host], [np.zeros(x.size + 8, np.float32) for x in host]
    for z in zeros:
        z[-8:] = 7
    p, m = ([capi.to_device(z) for z in zeros] for _ in range(2))
    capi.call("muon_step_multi", len(shapes), pointers(p), pointers(g), pointers(m), capi.i64([s[0] for s in shapes]), capi.i64([s[1] for s in shapes]), f32(-1.0), f32(0.0),
              0, f32(0.0), 5, f32(1.0))
    for x, d, s in zip(host, p, shapes):
        got = d.numpy()
        assert np.all(got[x.size :] == 7)
        got = got[: x.size].reshape(s) / max(1.0, s[1] / s[0]) ** 0.5
        as_near_as_fp32(got, steps_on_gpu(x, torch.float64), steps_on_gpu(x, torch.float32))


@pytest.mark.parametrize("steps", [1, 5])
def test_orthogonalize_by_either_path(capi, contraction_path, steps):
    r = rng(36)
    for shape in ((1, 6), (65, 30), (140, 333), (700, 512)):
        x = matrix(r, shape)
        d, out = capi.to_device(x), capi.empty(shape)
        capi.call("orthogonalize_list", 1, pointers([d]), capi.i64([shape[0]]), capi.i64([shape[1]]), steps, pointers([out]))
        as_near_as_fp32(out.numpy(), ref.orthogonalize(x, steps), ref.orthogonalize(x, steps, np.float32))


@pytest.mark.parametrize("value", [0.0, 1e-30, 1e30, 5e37, np.nan, np.inf])
def test_orthogonalize_of_special_matrices(capi, value):
    r = rng(32)
    for shape in ((40, 30), (150, 200)):
        x = r.standard_normal(shape).astype(np.float32)
        x = (x * np.float32(value)).astype(np.float32) if np.isfinite(value) else x
        if not np.isfinite(value):
            x[3, 4] = value
        d, out = capi.to_device(x), capi.empty(shape)
        capi.call("orthogonalize_list", 1, pointers([d]), capi.i64([shape[0]]), capi.i64([shape[1]]), 5, pointers([out]))
        if value == 0:
            assert np.all(out.numpy() == 0)
        elif not np.isfinite(value):
            assert np.isnan(out.numpy()).all()
        else:
            as_near_as_fp32(out.numpy(), ref.orthogonalize(x), ref.orthogonalize(x, 5, np.float32))


def test_orthogonalize_of_low_rank(capi):
    """Rank one, rank two with a small rest: most singular values are nothing but rounding."""
    r = rng(33)
    for shape, rest in (((96, 160), 0.0), ((300, 140), 1e-3)):
        x = sum(np.outer(r.standard_normal(shape[0]), r.standard_normal(shape[1])) for _ in range(1 + (rest > 0)))
        x = (x + rest * r.standard_normal(shape)).astype(np.float32)
        d, out = capi.to_device(x), capi.empty(shape)
        capi.call("orthogonalize_list", 1, pointers([d]), capi.i64([shape[0]]), capi.i64([shape[1]]), 5, pointers([out]))
        as_near_as_fp32(out.numpy(), ref.orthogonalize(x), ref.orthogonalize(x, 5, np.float32))


@pytest.mark.parametrize("nesterov", [0, 1])
def test_muon_step(capi, nesterov):
    r = rng(34)
    shapes = SHAPES[:9] + [(0, 5), (200, 300), (640, 130)]
    lr, mu, wd, scale = 0.05, 0.9, 0.02, 0.5
    host = [[matrix(r, s) for s in shapes] for _ in range(3)]
    p, g, m = ([capi.to_device(x) for x in xs] for xs in host)
    args = capi.i64([s[0] for s in shapes]), capi.i64([s[1] for s in shapes]), f32(lr), f32(mu), nesterov, f32(wd), 5, f32(scale)
    capi.call("muon_step_multi", len(shapes), pointers(p), pointers(g), pointers(m), *args)
    for k, s in enumerate(shapes):
        if 0 in s:
            continue
        want, want_m = ref.muon(host[0][k], host[1][k], host[2][k], lr, mu, nesterov, wd, 5, scale)
        plain, _ = ref.muon(host[0][k], host[1][k], host[2][k], lr, mu, nesterov, wd, 5, scale, np.float32)
        got, got_m = p[k].numpy(), m[k].numpy()
        assert within(got_m, want_m, 2 * ref.U * (np.abs(mu * host[2][k]) + np.abs(scale * host[1][k])))
        step = lr * max(1.0, s[1] / s[0]) ** 0.5
        # the update like the steps in fp32; keeping, subtracting: rounded three times
        allowed = 3 * np.linalg.norm(plain - want) + 4 * ref.U * (np.linalg.norm(host[0][k]) + 2 * step * np.sqrt(min(s)))
        assert np.linalg.norm(got - want) <= allowed, s
    assert all(np.array_equal(a.numpy(), b) for a, b in zip(g, host[1]))


@pytest.mark.parametrize("steps", [0, 5])
def test_muon_step_by_either_path(capi, contraction_path, steps):
    r = rng(37)
    lr, mu, wd, scale = 0.05, 0.9, 0.02, 0.5
    for s in ((1, 1), (40, 90), (333, 140)):
        p0, g0, m0 = (matrix(r, s) for _ in range(3))
        p, g, m = (capi.to_device(x) for x in (p0, g0, m0))
        capi.call("muon_step_multi", 1, pointers([p]), pointers([g]), pointers([m]), capi.i64([s[0]]), capi.i64([s[1]]), f32(lr), f32(mu), 1, f32(wd), steps, f32(scale))
        want, want_m = ref.muon(p0, g0, m0, lr, mu, 1, wd, steps, scale)
        plain, _ = ref.muon(p0, g0, m0, lr, mu, 1, wd, steps, scale, np.float32)
        assert within(m.numpy(), want_m, 2 * ref.U * (np.abs(mu * m0) + np.abs(scale * g0)))
        step = lr * max(1.0, s[1] / s[0]) ** 0.5
        # the update is off by no more than one step and its growth (as_near_as_fp32); keeping, subtracting: rounded three times
        allowed = 3 * np.linalg.norm(plain - want) + step * 301 * ref.U + 4 * ref.U * (np.linalg.norm(p0) + 2 * step * np.sqrt(min(s)))
        assert np.linalg.norm(p.numpy() - want) <= allowed, s


def test_two_contexts_at_once(capi):
    """Cooperative launches, small and large, on two streams: the same bits as one after the other."""
    r = rng(38)
    lists = [[(300, 200), (90, 40)], [(1501, 1603)], [(1290, 1803)] * 6]
    other = rusttensor_b200.CApi()
    try:
        host = [[matrix(r, s) for s in shapes] for shapes in lists]
        results = []
        for apis in ((capi, capi), (capi, other)):
            work = [(api, xs, [api.to_device(x) for x in xs], [api.empty(x.shape) for x in xs]) for api in apis for xs in host]
            for api in apis:
                api.sync()
            for _ in range(3):
                for k in range(len(lists)):
                    for api, xs, d, o in (work[k], work[len(lists) - 1 - k + len(lists)]):
                        api.call("orthogonalize_list", len(xs), pointers(d), api.i64([x.shape[0] for x in xs]), api.i64([x.shape[1] for x in xs]), 5, pointers(o))
            results.append([[a.numpy() for a in o] for _, _, _, o in work])
            for api in apis:
                code = C.c_int(0)
                api.call("device_status", C.byref(code))
        for one, two in zip(*results):
            assert all(np.array_equal(a, b) for a, b in zip(one, two))
    finally:
        other.close()


def test_large_matrices_captured_and_replayed(capi):
    """Two graphs of the same call, an eager call between their launches."""
    r = rng(39)
    shapes = [(1501, 1603), (65, 700)]
    d, o = [capi.empty(s) for s in shapes], [capi.empty(s) for s in shapes]
    args = (len(shapes), pointers(d), capi.i64([s[0] for s in shapes]), capi.i64([s[1] for s in shapes]), 5, pointers(o))
    inputs = [[matrix(r, s) for s in shapes] for _ in range(2)]

    def fill(k):
        for x, dx in zip(inputs[k], d):
            capi.check(capi.lib.rt_memcpy_h2d(capi.ctx, dx.ptr, x.ctypes.data_as(C.c_void_p), C.c_size_t(x.nbytes)))

    want, graphs = [], []
    for k in range(2):
        fill(k)
        capi.call("orthogonalize_list", *args)
        want.append([x.numpy() for x in o])
    for _ in range(2):
        capi.call("graph_begin")
        capi.call("orthogonalize_list", *args)
        graphs.append(C.c_void_p())
        capi.call("graph_end", C.byref(graphs[-1]))
    for graph, k in ((0, 0), (1, 1), (0, 1), (1, 0)):
        fill(1 - k)
        capi.call("orthogonalize_list", *args)
        fill(k)
        capi.call("graph_launch", graphs[graph])
        assert all(np.array_equal(a.numpy(), b) for a, b in zip(o, want[k]))
    for g in graphs:
        capi.call("graph_destroy", g)


# ---- in graphs, through the engine, together ------------------------------------------------------------------------------------------------


def test_captured_and_replayed(capi):
    """All of them in one graph, replayed with other inputs, an eager call of the same kind and another graph in between: the workspaces of a
    graph are its own."""
    r = rng(41)
    rows, cols, steps, batch, hidden = 90, 64, 150, 4, 32
    n = steps * batch
    table, g, ids = capi.empty((rows, cols)), capi.empty((n, cols)), capi.empty((n,))
    h0, h, dh, dgates, dtable = capi.empty((batch, hidden)), capi.empty((n, hidden)), capi.empty((n, hidden)), capi.empty((n, cols)), capi.empty((rows, cols))
    mom = capi.empty((rows, cols))
    emb = capi.empty((n, cols))

    def calls():
        capi.call("embedding", table.ptr, i64(rows), i64(cols), ids.ptr, i64(n), f32(2.0), emb.ptr)
        sizes = (i64(steps), i64(batch), i64(hidden))
        capi.call("gated_scan", emb.ptr, offset(emb, hidden), i64(cols), h0.ptr, *sizes, h.ptr)
        capi.call("gated_scan_backward", emb.ptr, offset(emb, hidden), i64(cols), h0.ptr, h.ptr, dh.ptr, *sizes, dgates.ptr, offset(dgates, hidden), i64(cols), None)
        capi.call("embedding_backward", dgates.ptr, ids.ptr, i64(n), i64(rows), i64(cols), f32(2.0), dtable.ptr, 0)
        capi.call("muon_step_multi", 1, pointers([table]), pointers([dtable]), pointers([mom]), capi.i64([rows]), capi.i64([cols]), f32(0.1), f32(0.9), 1, f32(0.0),
                  5, f32(1.0))

    def inputs(seed):
        q = rng(seed)
        for d, shape in ((table, (rows, cols)), (h0, (batch, hidden)), (dh, (n, hidden)), (mom, (rows, cols))):
            a = q.standard_normal(shape).astype(np.float32)
            capi.check(capi.lib.rt_memcpy_h2d(capi.ctx, d.ptr, a.ctypes.data_as(C.c_void_p), C.c_size_t(a.nbytes)))
        a = tokens(q, rows, n).astype(np.int32)
        capi.check(capi.lib.rt_memcpy_h2d(capi.ctx, ids.ptr, a.ctypes.data_as(C.c_void_p), C.c_size_t(a.nbytes)))

    def results():
        return [d.numpy() for d in (emb, h, dgates, dtable, table, mom)]

    want = []
    for seed in (1, 2):
        inputs(seed)
        calls()
        want.append(results())
    graphs = []
    for _ in range(2):
        capi.call("graph_begin")
        calls()
        graph = C.c_void_p()
        capi.call("graph_end", C.byref(graph))
        graphs.append(graph)
    for seed, graph in ((1, graphs[0]), (2, graphs[1]), (2, graphs[0]), (1, graphs[1])):
        inputs(seed)
        calls()
        inputs(seed)
        capi.call("graph_launch", graph)
        assert all(np.array_equal(a, b) for a, b in zip(results(), want[seed - 1]))
    for graph in graphs:
        capi.call("graph_destroy", graph)


def test_a_recurrent_language_model(gpu_engine, oracle_engine):
    """Embedding, gates, recurrence, output layer and loss, trained with Muon and Adam for a few steps: the engine on the GPU and the chain of the
    reference's ops on the CPU have the same losses and gradients."""
    r = rng(51)
    vocab, width, hidden, steps, batch = 30, 24, 20, 12, 5
    shapes = [(vocab, width), (width, 2 * hidden), (2 * hidden,), (hidden, vocab)]
    init = [(0.3 * r.standard_normal(s)).astype(np.float32) for s in shapes]
    text = r.integers(0, vocab, steps * batch + 1).astype(np.float32)
    targets = np.eye(vocab, dtype=np.float32)[text[1:].astype(int)]
    seen = []
    for e in (gpu_engine, oracle_engine):
        ops = e.ops
        emb, w, b, out = (e.tensor(p, requires_grad=True) for p in init)
        h0 = e.tensor(np.zeros((batch, hidden)), requires_grad=True)
        opts = [e.Muon([w, out], 0.02, 0.9, True, 0.01), e.Adam([emb, b], 1e-2)]
        ids, y = e.tensor(text[:-1]), e.tensor(targets)
        log = []
        for _ in range(4):
            gates = ops.add(ops.matmul(ops.embedding(emb, ids, width**0.5), w), b)
            logits = ops.matmul(ops.gated_scan(gates, steps, h0), out)
            loss = ops.mul_scalar(ops.mean(ops.sum(ops.mul(ops.log_softmax(logits, 1), y), 1)), -1.0)
            loss.backward()
            log += [loss.numpy()] + [t.grad.numpy() for t in (emb, w, b, out, h0)]
            for o in opts:
                o.step()
                o.zero_grad()
            h0.zero_grad()
        seen.append(log + [t.numpy() for t in (emb, w, b, out)])
    for a, b in zip(*seen):
        # 1e-4 is what the framework holds its kernels to; values near zero to a part of their tensor's largest
        assert np.all(np.abs(a - b) <= 1e-4 * np.maximum(np.abs(a), np.abs(b)) + 1e-4 * np.abs(b).max())


def test_muon_with_a_parameter_listed_twice(gpu_engine, oracle_engine):
    """It is updated twice, in order; two backward passes before a step add up; a parameter that is another's gradient is read before it changes."""
    r = rng(53)
    init, other = (r.standard_normal((12, 20)).astype(np.float32) for _ in range(2))
    seen = []
    for e in (gpu_engine, oracle_engine):
        a, b = e.tensor(init, requires_grad=True), e.tensor(other, requires_grad=True)
        opt = e.Muon([a, b, a], 0.05, 0.9, False, 0.01)
        for _ in range(3):
            for _ in range(2):
                e.ops.sum(e.ops.mul(a, b)).backward()
            opt.step()
            opt.zero_grad()
        seen.append([a.numpy(), b.numpy()])
    for x, y in zip(*seen):
        assert np.all(np.abs(x - y) <= 1e-4 * np.maximum(np.abs(x), np.abs(y)) + 1e-4 * np.abs(y).max())


def test_engine_gradient_after_the_result_was_written_from_outside(gpu_engine):
    """The states that a caller has an address of may be changed: the gradient is that of the states that were computed."""
    e, r = gpu_engine, rng(52)
    gates = r.standard_normal((30, 16)).astype(np.float32)
    grads = []
    for write in (False, True):
        t = e.tensor(gates, requires_grad=True)
        h = e.ops.gated_scan(t, 10)
        loss = e.ops.sum(e.ops.square(h))
        if write:
            loss.numpy()
            p = C.c_void_p()
            assert rusttensor_b200.load_host_library().rth_tensor_device_ptr(i64(h.handle), C.byref(p)) == 0
            api = rusttensor_b200.CApi(ctx=rusttensor_b200.context_handle())
            api.call("gated_scan", p, p, i64(8), None, i64(1), i64(1), i64(8), p)
        g = e.op_backward(h, e.tensor(np.ones((30, 8))))[0]
        grads.append(g.numpy())
    assert np.array_equal(*grads)
