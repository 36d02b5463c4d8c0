"""Token embeddings, the gated linear recurrence and Muon on the CPU: the engine's ops as chains of the reference's ops against their plain
form in 64 bits, their gradients against differences, and what is refused, by the engine and by the C ABI, before anything is launched."""
import os
import subprocess

import numpy as np
import pytest

import language_ref as ref
from helpers import rng
from rusttensor_b200.frontend import EngineError

HERE = os.path.dirname(os.path.abspath(__file__))


def test_embedding_and_gradient(oracle_engine):
    e, r = oracle_engine, rng(1)
    table, ids = r.standard_normal((7, 5)).astype(np.float32), np.array([[3, 0, 3], [6, -1, 7]])
    g = r.standard_normal((2, 3, 5)).astype(np.float32)
    t = e.tensor(table, requires_grad=True)
    out = e.ops.embedding(t, e.tensor(ids), 2.5)
    assert out.shape == (2, 3, 5)
    assert np.array_equal(out.numpy().reshape(6, 5), ref.embedding(table, ids.ravel(), 2.5))
    e.ops.sum(e.ops.mul(out, e.tensor(g))).backward()
    want, bound = ref.embedding_backward(g.reshape(6, 5), ids.ravel(), 7, 2.5)
    assert np.all(np.abs(t.grad.numpy() - want) <= bound + 2 * ref.U * np.abs(want))


@pytest.mark.parametrize("given", [False, True])
def test_gated_scan_and_gradient(oracle_engine, given):
    e, r = oracle_engine, rng(2)
    steps, batch, hidden = 9, 3, 4
    gates = r.standard_normal((steps * batch, 2 * hidden)).astype(np.float32)
    h0 = r.standard_normal((batch, hidden)).astype(np.float32) * given
    dh = r.standard_normal((steps, batch, hidden)).astype(np.float32)
    f, v = (gates[:, k * hidden : (k + 1) * hidden].reshape(steps, batch, hidden) for k in range(2))
    tg, th = e.tensor(gates, requires_grad=True), e.tensor(h0, requires_grad=True)
    out = e.ops.gated_scan(tg, steps, th if given else None)
    want, bound = ref.scan(f, v, h0)
    got = out.numpy().reshape(want.shape)
    assert np.all(np.abs(got - want) <= bound)
    e.ops.sum(e.ops.mul(out, e.tensor(dh.reshape(-1, hidden)))).backward()
    (df, bf), (dv, bv), (d0, b0) = ref.scan_backward(f, v, h0, got, dh)
    grad = tg.grad.numpy().reshape(steps, batch, 2 * hidden)
    # op by op df is the difference of two terms: each is off by as much as it is large
    assert np.all(np.abs(grad[..., :hidden] - df) <= bf + 40 * ref.U * np.abs(dh).sum(0) * (np.abs(v) + np.abs(want).max()))
    assert np.all(np.abs(grad[..., hidden:] - dv) <= bv)
    if given:
        assert np.all(np.abs(th.grad.numpy() - d0) <= b0)


def test_the_plain_gradient_is_that_of_differences():
    r = rng(3)
    f, v = r.standard_normal((2, 6, 2, 3))
    h0, dh = r.standard_normal((2, 3)), r.standard_normal((6, 2, 3))
    h, _ = ref.scan(f, v, h0)
    loss = lambda f, v, h0: float((ref.scan(f, v, h0)[0] * dh).sum())  # noqa: E731
    args = [f, v, h0]
    for k, (d, _) in enumerate(ref.scan_backward(f, v, h0, h, dh)):
        for at in np.ndindex(d.shape):
            lo, hi = [a.copy() for a in args], [a.copy() for a in args]
            lo[k][at] -= 1e-5
            hi[k][at] += 1e-5
            assert abs((loss(*hi) - loss(*lo)) / 2e-5 - d[at]) <= 1e-8  # third derivatives below 10 times 1e-10, roundings 1e-16 / 1e-5


@pytest.mark.parametrize("shape", [(5, 9), (9, 5), (4, 4), (1, 6)])
@pytest.mark.parametrize("nesterov", [False, True])
def test_muon(oracle_engine, shape, nesterov):
    e, r = oracle_engine, rng(4)
    p, g, m = (r.standard_normal(shape).astype(np.float32) for _ in range(3))
    tp = e.tensor(p, requires_grad=True)
    opt = e.Muon([tp], 0.1, 0.9, nesterov, 0.01)
    m = np.zeros(shape)
    for _ in range(3):
        tp.set_grad(e.tensor(g))
        opt.step()
        p, m = ref.muon(p, g, m, 0.1, 0.9, nesterov, 0.01)
    # five steps with slopes up to 3.9: 311 times what a step is off, some 16 roundings of sums of up to nine terms
    assert np.abs(tp.numpy() - p).max() <= 3 * 0.1 * max(1, shape[1] / shape[0]) ** 0.5 * 311 * 16 * 9 * ref.U
    assert np.abs(opt.state(0, 0).numpy() - m).max() <= 12 * ref.U * np.abs(m).max()
    opt.zero_grad()
    assert tp.grad is None


def test_refusals_of_the_engine(oracle_engine):
    e = oracle_engine
    zeros = lambda *s: e.tensor(np.zeros(s))  # noqa: E731
    for call, kind in [
        (lambda: e.ops.embedding(zeros(3), zeros(2)), "InvalidOperation"),
        (lambda: e.ops.embedding(zeros(2, 3, 4), zeros(2)), "InvalidOperation"),
        (lambda: e.ops.gated_scan(zeros(6, 8), 4), "InvalidOperation"),       # 6 rows are not 4 timesteps
        (lambda: e.ops.gated_scan(zeros(6, 8), 0), "InvalidOperation"),
        (lambda: e.ops.gated_scan(zeros(6, 8), -1), "InvalidOperation"),
        (lambda: e.ops.gated_scan(zeros(6, 7), 2), "InvalidOperation"),       # not two columns a unit
        (lambda: e.ops.gated_scan(zeros(48), 2), "InvalidOperation"),
        (lambda: e.ops.gated_scan(zeros(6, 8), 2, zeros(2, 4)), "IncompatibleShapes"),
        (lambda: e.Muon([zeros(3)]), "InvalidOperation"),
        (lambda: e.Muon([zeros(3, 4)], ns_steps=-1), "InvalidOperation"),
        (lambda: e.Muon([zeros(3, 4)], ns_steps=65), "InvalidOperation"),
    ]:
        with pytest.raises(EngineError) as ei:
            call()
        assert ei.value.kind == kind


def test_refusals_of_the_c_abi(tmp_path):
    """A context that no device stands behind: every refused call answers before it would touch one."""
    exe, lib = str(tmp_path / "language_checks"), os.path.join(os.path.dirname(HERE), "rusttensor_b200")
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-O1", "-I/usr/local/cuda/include", "-o", exe,
                    os.path.join(HERE, "host", "language_checks.cpp"), "-L" + lib, "-lrt_b200", "-Wl,-rpath," + lib], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
