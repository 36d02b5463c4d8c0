"""The operators that a language model is trained with, as timed cases: the lookup of token embeddings and its gradient, the gated linear
recurrence over a sequence and its gradient, and the optimizer step whose update is an orthogonalised momentum (Muon).

``listed()`` gives the cases, ``draw(rng)`` one more of the same ranges; ``prepare`` / ``run`` / ``work`` / ``exact`` take a case.  ``run``
computes the plain form with elementary torch operations, or, with ``own`` set, makes the C ABI's calls on the same device buffers.  All
data is fp32, the only type that the framework computes in; token numbers are int32 as for its row gather.
"""
import ctypes as C
import math

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)  # of the quintic x -> a x + b x^3 + c x^5 on the singular values
EPSILON = 1e-7                            # added to the norm that a matrix is divided by


def listed():
    return [
        # One character for each sequence of the character model's batch, as when it generates text: latency.
        dict(name="embed_step", op="embedding", rows=65, cols=512, tokens=64, padding=0.0),
        # A training batch of a word model: a large table, rows read as often as words occur.
        dict(name="embed_words", op="embedding", rows=50000, cols=1024, tokens=32768, padding=0.0),
        # The character model's gradient of its table: 128 timesteps of 64 sequences, every row over a hundred times.
        dict(name="embed_grad_chars", op="embedding_backward", rows=65, cols=512, tokens=8192, padding=0.0, accumulate=False),
        # The word model's: most rows without a token, a few with thousands.
        dict(name="embed_grad_words", op="embedding_backward", rows=50000, cols=1024, tokens=32768, padding=0.0, accumulate=False),
        # A table that is an output layer too: odd sizes, a padded batch, added to the gradient that is there.
        dict(name="embed_grad_tied", op="embedding_backward", rows=20011, cols=333, tokens=5000, padding=0.2, accumulate=True),
        # One timestep, as when text is generated: latency.
        dict(name="scan_step", op="gated_scan", steps=1, batch=64, hidden=512, joined=True),
        # The character model's sequences, both halves of a product's result.
        dict(name="scan_chars", op="gated_scan", steps=128, batch=64, hidden=512, joined=True),
        # One long document.
        dict(name="scan_long", op="gated_scan", steps=65536, batch=1, hidden=512, joined=True),
        # A few long sequences of an odd width, backward, gates in matrices of their own.
        dict(name="scan_grad_long", op="gated_scan_backward", steps=30011, batch=3, hidden=257, joined=False),
        # The optimizer step of a small classifier: latency of dependent products.
        dict(name="muon_mlp", op="muon", shapes="784x128,128x10", momentum=0.95, nesterov=True, weight_decay=0.0),
        # The matrices of recurrent models of several sizes in one step, odd ones, tall and wide.
        dict(name="muon_layers", op="muon", shapes="577x2048,512x65,1024x1024,1000x777,2048x512", momentum=0.9, nesterov=False, weight_decay=0.01),
        # One large layer: dense products.
        dict(name="orthogonalize_large", op="orthogonalize", shapes="4096x4096"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _even_or_odd(rng, n):
    """Every other size a multiple of four, as most models have them."""
    return max(4, n // 4 * 4) if rng.random() < 0.5 else n


def draw(rng):
    op = rng.choice(["embedding", "embedding_backward", "gated_scan", "gated_scan_backward", "muon", "orthogonalize"])
    if op.startswith("embedding"):
        c = dict(op=op, rows=_log(rng, 30, 50000), cols=_even_or_odd(rng, _log(rng, 16, 1024)), tokens=_log(rng, 1, 32768),
                 padding=rng.choice([0.0, 0.3]))
        return dict(c, accumulate=rng.random() < 0.5) if op == "embedding_backward" else c
    if op.startswith("gated_scan"):
        batch, hidden = _log(rng, 1, 64), _even_or_odd(rng, _log(rng, 16, 1024))
        return dict(op=op, steps=_log(rng, 1, max(1, min(65536, 16000000 // (batch * hidden)))), batch=batch, hidden=hidden, joined=rng.random() < 0.5)
    if op == "muon":
        shapes = ["%dx%d" % tuple(_even_or_odd(rng, _log(rng, 8, 1500)) for _ in range(2)) for _ in range(rng.randint(1, 6))]
        return dict(op=op, shapes=",".join(shapes), momentum=round(rng.uniform(0.8, 0.98), 3), nesterov=rng.random() < 0.5,
                    weight_decay=rng.choice([0.0, 0.05]))
    return dict(op=op, shapes="%dx%d" % tuple(_even_or_odd(rng, _log(rng, 100, 2600)) for _ in range(2)))


def _shapes(c):
    return [tuple(int(n) for n in s.split("x")) for s in c["shapes"].split(",")]


# ---- inputs ---------------------------------------------------------------------------------------------------------------------


def _tokens(c, g):
    """Token numbers that occur about as often as one over their number; with padding, -1 for that share of the places."""
    u = torch.rand(c["tokens"], generator=g, device="cuda", dtype=torch.float64)
    ids = ((u * math.log(c["rows"] + 1)).exp() - 1).clamp_(0, c["rows"] - 1).to(torch.int32)
    if c["padding"]:
        ids[torch.rand(c["tokens"], generator=g, device="cuda") < c["padding"]] = -1
    return ids


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    empty = lambda *s: torch.empty(s, device="cuda")  # noqa: E731
    s = {"case": dict(c)}
    if c["op"] == "embedding":
        s["scale"] = math.sqrt(c["cols"])
        s.update(table=0.02 * normal(c["rows"], c["cols"]), ids=_tokens(c, g), out=empty(c["tokens"], c["cols"]))
    elif c["op"] == "embedding_backward":
        s["scale"] = math.sqrt(c["cols"])
        s.update(g=normal(c["tokens"], c["cols"]) / c["tokens"], ids=_tokens(c, g), dtable=1e-4 * normal(c["rows"], c["cols"]))
    elif c["op"].startswith("gated_scan"):
        rows, hidden = c["steps"] * c["batch"], c["hidden"]
        if c["joined"]:
            gates = normal(rows, 2 * hidden)
            f, v = gates[:, :hidden], gates[:, hidden:]
        else:
            f, v = normal(rows, hidden), normal(rows, hidden)
        f.mul_(2).add_(2)  # states that are kept for some tens of timesteps
        s.update(f=f, v=v, h0=normal(c["batch"], hidden))
        if c["op"] == "gated_scan":
            s["h"] = empty(rows, hidden)
        else:
            s.update(h=_scan_plain(c, f, v, s["h0"]), dh=normal(rows, hidden))
            if c["joined"]:
                d = empty(rows, 2 * hidden)
                s.update(df=d[:, :hidden], dv=d[:, hidden:])
            else:
                s.update(df=empty(rows, hidden), dv=empty(rows, hidden))
            s["dh0"] = empty(c["batch"], hidden)
    else:
        shapes = _shapes(c)
        # gradients whose rows differ in size, as the inputs of a layer do
        grad = lambda m, n: 1e-2 * normal(m, n) * normal(m, 1).exp()  # noqa: E731
        if c["op"] == "orthogonalize":
            s.update(xs=[grad(m, n) for m, n in shapes], outs=[empty(m, n) for m, n in shapes])
        else:
            s.update(p=[normal(m, n) / math.sqrt(m) for m, n in shapes], g=[grad(m, n) for m, n in shapes], m=[grad(m, n) for m, n in shapes])
    s["call"] = _call(s)
    return s


def _call(s):
    """The entry point's name and its arguments behind the context."""
    c, p = s["case"], lambda t: C.c_void_p(t.data_ptr())
    i64, f32 = C.c_int64, C.c_float
    if c["op"] == "embedding":
        return ("embedding", p(s["table"]), i64(c["rows"]), i64(c["cols"]), p(s["ids"]), i64(c["tokens"]), f32(s["scale"]), p(s["out"]))
    if c["op"] == "embedding_backward":
        return ("embedding_backward", p(s["g"]), p(s["ids"]), i64(c["tokens"]), i64(c["rows"]), i64(c["cols"]), f32(s["scale"]), p(s["dtable"]),
                int(c["accumulate"]))
    if c["op"].startswith("gated_scan"):
        sizes = i64(c["steps"]), i64(c["batch"]), i64(c["hidden"])
        gates = p(s["f"]), p(s["v"]), i64(s["f"].stride(0)), p(s["h0"])
        if c["op"] == "gated_scan":
            return ("gated_scan", *gates, *sizes, p(s["h"]))
        return ("gated_scan_backward", *gates, p(s["h"]), p(s["dh"]), *sizes, p(s["df"]), p(s["dv"]), i64(s["df"].stride(0)), p(s["dh0"]))
    shapes = _shapes(c)
    n = len(shapes)
    ptrs = lambda ts: (C.c_void_p * n)(*[t.data_ptr() for t in ts])  # noqa: E731
    dims = [(i64 * n)(*[s[k] for s in shapes]) for k in (0, 1)]
    if c["op"] == "orthogonalize":
        return ("orthogonalize_list", n, ptrs(s["xs"]), *dims, 5, ptrs(s["outs"]))
    return ("muon_step_multi", n, ptrs(s["p"]), ptrs(s["g"]), ptrs(s["m"]), *dims, f32(0.02), f32(c["momentum"]), int(c["nesterov"]),
            f32(c["weight_decay"]), 5, f32(1.0))


# ---- the operators in elementary operations ----------------------------------------------------------------------------------------


def _embedding_plain(s):
    c, ids = s["case"], s["ids"].long()
    there = (ids >= 0) & (ids < c["rows"])
    s["out"].copy_(torch.where(there[:, None], s["table"][ids.clamp(0, c["rows"] - 1)] * s["scale"], 0.0))
    return s["out"]


def _embedding_backward_plain(s):
    c, ids = s["case"], s["ids"].long()
    there = (ids >= 0) & (ids < c["rows"])
    term = torch.where(there[:, None], s["g"], 0.0)
    total = torch.zeros(c["rows"], c["cols"], device="cuda").index_add_(0, ids.clamp(0, c["rows"] - 1), term).mul_(s["scale"])
    if c["accumulate"]:
        s["dtable"].add_(total)
    else:
        s["dtable"].copy_(total)
    return s["dtable"]


def _recurrence(a, b):
    """h_t = a_t h_{t-1} + b_t along the first axis, from zero: the pairs (a, b) composed over distances of 1, 2, 4, ..."""
    k = 1
    while k < a.shape[0]:
        b = torch.cat([b[:k], b[k:] + a[k:] * b[:-k]])
        a = torch.cat([a[:k], a[k:] * a[:-k]])
        k *= 2
    return b


def _scan_plain(c, f, v, h0):
    f, v = (t.reshape(c["steps"], c["batch"], c["hidden"]) for t in (f, v))
    a, b = torch.sigmoid(f), torch.sigmoid(-f) * v
    b[0] += a[0] * h0
    return _recurrence(a, b).reshape(-1, c["hidden"])


def _scan_backward_plain(s):
    c = s["case"]
    f, v, h, dh = (s[k].reshape(c["steps"], c["batch"], c["hidden"]) for k in ("f", "v", "h", "dh"))
    a, rest = torch.sigmoid(f), torch.sigmoid(-f)
    following = torch.cat([a[1:], torch.zeros_like(a[:1])])
    d = _recurrence(following.flip(0), dh.flip(0)).flip(0)
    before = torch.cat([s["h0"][None], h[:-1]])
    s["df"].copy_((d * (before - v) * a * rest).reshape(-1, c["hidden"]))
    s["dv"].copy_((d * rest).reshape(-1, c["hidden"]))
    s["dh0"].copy_(a[0] * d[0])
    return [s["df"], s["dv"], s["dh0"]]


def _orthogonalized(x):
    a, b, c = COEFFICIENTS
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    x = x / (x.double().square().sum().sqrt() + EPSILON).float()
    for _ in range(5):
        gram = x @ x.t()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.t() if tall else x


def _muon_plain(s):
    c = s["case"]
    for p, g, m in zip(s["p"], s["g"], s["m"]):
        m.mul_(c["momentum"]).add_(g)
        u = g + c["momentum"] * m if c["nesterov"] else m
        step = 0.02 * math.sqrt(max(1.0, p.shape[1] / p.shape[0]))
        p.mul_(1 - 0.02 * c["weight_decay"]).sub_(step * _orthogonalized(u))
    return s["p"] + s["m"]


def _orthogonalize_plain(s):
    for x, out in zip(s["xs"], s["outs"]):
        out.copy_(_orthogonalized(x))
    return s["outs"]


def _outputs(s):
    op = s["case"]["op"]
    if op == "gated_scan_backward":
        return [s["df"], s["dv"], s["dh0"]]
    if op == "muon":
        return s["p"] + s["m"]
    return s[{"embedding": "out", "embedding_backward": "dtable", "gated_scan": "h", "orthogonalize": "outs"}[op]]


_contexts = []


def _api():
    """The C ABI on the engine's context."""
    if not _contexts:
        import rusttensor_b200

        _contexts.append(rusttensor_b200.CApi(ctx=rusttensor_b200.context_handle()))
    return _contexts[0]


def run(state):
    if own:
        _api().call(*state["call"])
        return _outputs(state)
    op = state["case"]["op"]
    if op == "embedding":
        return _embedding_plain(state)
    if op == "embedding_backward":
        return _embedding_backward_plain(state)
    if op == "gated_scan":
        state["h"].copy_(_scan_plain(state["case"], state["f"], state["v"], state["h0"]))
        return state["h"]
    if op == "gated_scan_backward":
        return _scan_backward_plain(state)
    return _muon_plain(state) if op == "muon" else _orthogonalize_plain(state)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------------------


def _orthogonalize_flops(m, n):
    """Five times: the lower half of X X^T and of its square (both symmetric), and a product with X."""
    m, n = min(m, n), max(m, n)
    return 5 * (m * (m + 1) * n + m * (m + 1) * m + 2 * m * m * n)


def work(case):
    c = case
    if c["op"].startswith("embedding"):
        read = c["tokens"] * (1 - c["padding"]) * c["cols"]
        if c["op"] == "embedding":  # rows that occur more than once are read once
            return {"bytes": 4 * (min(read, c["rows"] * c["cols"]) + c["tokens"] * (c["cols"] + 1)), "flops": read}
        rows = 2 * min(c["tokens"], c["rows"]) if c["accumulate"] else c["rows"]
        return {"bytes": 4 * (read + c["tokens"] + rows * c["cols"]), "flops": 2 * read}
    if c["op"].startswith("gated_scan"):
        n, state = c["steps"] * c["batch"] * c["hidden"], c["batch"] * c["hidden"]
        return {"bytes": 4 * (3 * n + state), "flops": 10 * n} if c["op"] == "gated_scan" else {"bytes": 4 * (6 * n + 2 * state), "flops": 16 * n}
    shapes = _shapes(c)
    return {"bytes": (8 if c["op"] == "orthogonalize" else 20) * sum(m * n for m, n in shapes), "flops": sum(_orthogonalize_flops(*s) for s in shapes)}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------------------


def _exact_newton_schulz(u):
    """Each step by the smaller Gram matrix, on whichever side it is."""
    x = u / (torch.linalg.vector_norm(u) + EPSILON)
    a, b, c = COEFFICIENTS
    for _ in range(5):
        if x.shape[0] <= x.shape[1]:
            q = x @ x.mT
            x = a * x + b * (q @ x) + c * (q @ (q @ x))
        else:
            q = x.mT @ x
            x = a * x + b * (x @ q) + c * ((x @ q) @ q)
    return x


def exact(case, seed):
    c, s = case, prepare(case, seed)
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    if c["op"] in ("embedding", "embedding_backward"):
        keep = ((s["ids"] >= 0) & (s["ids"] < c["rows"])).nonzero()[:, 0]
        ids = s["ids"][keep].long()
        if c["op"] == "embedding":
            out = torch.zeros(c["tokens"], c["cols"], dtype=torch.float64, device="cuda")
            out[keep] = float(C.c_float(s["scale"]).value) * d["table"][ids]
            return out
        total = torch.zeros(c["rows"], c["cols"], dtype=torch.float64, device="cuda")
        total.index_put_((ids,), float(C.c_float(s["scale"]).value) * d["g"][keep], accumulate=True)
        return total + d["dtable"] if c["accumulate"] else total
    if c["op"].startswith("gated_scan"):
        if c["steps"] > 200000:
            return None
        f, v = (d[k].reshape(c["steps"], c["batch"], c["hidden"]) for k in ("f", "v"))
        a = 1 / (1 + torch.exp(-f))
        if c["op"] == "gated_scan":  # timestep by timestep
            out, h = torch.empty_like(f), d["h0"]
            add = (1 - a) * v
            for t in range(c["steps"]):
                h = torch.addcmul(add[t], a[t], h, out=out[t])
            return out.reshape(-1, c["hidden"])
        h, dh = (d[k].reshape(c["steps"], c["batch"], c["hidden"]) for k in ("h", "dh"))
        up, carry = torch.empty_like(f), torch.zeros_like(d["h0"])
        for t in range(c["steps"] - 1, -1, -1):
            torch.add(dh[t], carry, out=up[t])
            carry = a[t] * up[t]
        before = torch.cat([d["h0"][None], h[:-1]])
        return [(up * (before - v) * a * (1 - a)).reshape(-1, c["hidden"]), (up * (1 - a)).reshape(-1, c["hidden"]), carry]
    if c["op"] == "orthogonalize":
        return [_exact_newton_schulz(x.double()) for x in s["xs"]]
    ps, ms = [], []
    f32 = lambda x: float(C.c_float(x).value)  # noqa: E731
    mu, lr, wd = f32(c["momentum"]), f32(0.02), f32(c["weight_decay"])
    for p, g, m in zip(s["p"], s["g"], s["m"]):
        p, g = p.double(), g.double()
        m = mu * m.double() + g
        q = _exact_newton_schulz(g + mu * m if c["nesterov"] else m)
        ps.append(p * (1 - lr * wd) - lr * max(1.0, p.shape[1] / p.shape[0]) ** 0.5 * q)
        ms.append(m)
    return ps + ms
