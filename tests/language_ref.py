"""Plain forms in 64 bits of the operators of language models (token embeddings, gated linear recurrence, Muon), with bounds on what fp32 may
be off.  `U` is half a step of fp32 relative to the value, the rounding of one operation."""
import numpy as np

U = 2.0**-24


def embedding(table, ids, scale):
    """In fp32: one product an element, rounded once."""
    there = (ids >= 0) & (ids < len(table))
    return np.where(there[:, None], table[np.where(there, ids, 0)] * np.float32(scale), np.float32(0))


def embedding_backward(g, ids, rows, scale, old=None):
    """The sums and the bound: a sum of k terms in any order is off by (k - 1) U of the sum of magnitudes, scaling and adding to what was
    there by one rounding each."""
    g, scale = g.astype(np.float64), float(np.float32(scale))
    total, size, count = np.zeros((rows, g.shape[1])), np.zeros((rows, g.shape[1])), np.zeros((rows, 1))
    keep = (ids >= 0) & (ids < rows)
    np.add.at(total, ids[keep], scale * g[keep])
    np.add.at(size, ids[keep], np.abs(scale * g[keep]))
    np.add.at(count, ids[keep], 1)
    bound = (count + 1) * U * size
    if old is not None:
        total = total + old
        bound = bound + U * np.abs(total) * (count > 0)
    return total, 1.001 * bound


def sigmoid(f):
    e = np.exp(-np.abs(f))
    return np.where(f >= 0, 1, e) / (1 + e), np.where(f >= 0, e, 1) / (1 + e)


# A gate: expf within 2 U of itself, of which 1 + e keeps at most half (1 U) and adds 1, an approximate reciprocal 2 (one unit of the last place);
# the smaller one once more e (2) and a product (1): 7 U.  A timestep multiplies with it and adds: 9 U for each timestep that a term has
# passed, however the timesteps are grouped.
GATE, STEP = 7, 9


def scan(f, v, h0):
    """States [steps, batch, hidden] and the bound."""
    f, v, h = f.astype(np.float64), v.astype(np.float64), h0.astype(np.float64)
    a, rest = sigmoid(f)
    size, age = np.abs(h), np.zeros_like(h)  # sum of the terms' magnitudes; of those times how many timesteps ago they came in
    hs, bounds = [], []
    for t in range(len(f)):
        h = a[t] * h + rest[t] * v[t]
        age = a[t] * (age + size)
        size = a[t] * size + rest[t] * np.abs(v[t])
        hs.append(h)
        bounds.append(U * (STEP * age + (STEP + GATE + 2) * size))
    return np.array(hs), 1.01 * np.array(bounds)


def scan_backward(f, v, h0, h, dh):
    """[(df, its bound), (dv, ...), (dh0, ...)] from the states h that the forward pass has left."""
    f, v, h0, h, dh = (x.astype(np.float64) for x in (f, v, h0, h, dh))
    a, rest = sigmoid(f)
    before = np.concatenate([h0[None], h[:-1]])
    d, size, age = (np.zeros_like(h0) for _ in range(3))
    df, dv = [np.zeros_like(f), np.zeros_like(f)], [np.zeros_like(f), np.zeros_like(f)]
    for t in reversed(range(len(f))):
        d, age, size = d + dh[t], age, size + np.abs(dh[t])
        off = U * (STEP * age + 2 * size)
        slope = (before[t] - v[t]) * a[t] * rest[t]
        df[0][t], df[1][t] = d * slope, (off + (2 * GATE + 5) * U * size) * np.abs(slope)
        dv[0][t], dv[1][t] = d * rest[t], (off + (GATE + 2) * U * size) * rest[t]
        d, age, size = a[t] * d, a[t] * (age + size), a[t] * size
    # below 2^-126 fp32 has steps of 2^-149; factors here stay below 32
    return [(x, 1.01 * b + 32 * 2.0**-149) for x, b in (df, dv, (d, U * (STEP * age + (STEP + 2) * size)))]


def orthogonalize(u, steps=5, dtype=np.float64):
    """Newton-Schulz steps by the shorter side's Gram matrix; in fp32 with dtype."""
    norm = np.sqrt((u.astype(np.float64) ** 2).sum()) + 1e-7
    x = (u.astype(np.float64) / norm).astype(dtype)
    x = x.T if u.shape[0] > u.shape[1] else x
    a, b, c = (dtype(k) for k in (3.4445, -4.7750, 2.0315))
    for _ in range(steps):
        g = x @ x.T
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.T if u.shape[0] > u.shape[1] else x


def muon(p, g, m, lr, momentum, nesterov, weight_decay, steps=5, scale=1.0, dtype=np.float64):
    p, g, m = (x.astype(np.float64) for x in (p, g, m))
    lr, momentum, weight_decay, scale = (float(np.float32(x)) for x in (lr, momentum, weight_decay, scale))
    m = momentum * m + scale * g
    u = scale * g + momentum * m if nesterov else m
    o = orthogonalize(u, steps, dtype)
    return p * (1 - lr * weight_decay) - lr * max(1.0, p.shape[1] / p.shape[0]) ** 0.5 * o, m
