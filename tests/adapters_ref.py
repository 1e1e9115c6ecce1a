"""64-bit restatement of the adapter and list operators (test infrastructure), with elementwise error bounds for float32
evaluation: a sum of n products in any order and any splitting is off by at most (n + c) u sum |products|, u = 2^-24, plus
what its inputs are off by."""
import numpy as np

U = 2.0 ** -24


def act(z, kind):
    return np.maximum(z, 0) if kind == "relu" else np.tanh(z) if kind == "tanh" else z


def act_grad(dy, y, kind):
    return dy * (y > 0) if kind == "relu" else dy * (1 - y * y) if kind == "tanh" else dy


def rows_of(idx, m, e):
    idx = np.zeros(m, np.int64) if idx is None else idx
    return [np.nonzero(idx == i)[0] for i in range(e)]


def forward(x, w, bias, a, b, s, idx, kind, base=None):
    """(y, t, bound of y, bound of t).  base: what y holds when there is no projection."""
    x, a, b, s = (v.astype(np.float64) for v in (x, a, b, s))
    m, k = x.shape
    e, n, r = b.shape
    if w is not None:
        w = w.astype(np.float64)
        z, ez = x @ w.T, (k + 16) * U * (np.abs(x) @ np.abs(w).T)
        if bias is not None:
            z, ez = z + bias, ez + 2 * U * (np.abs(x) @ np.abs(w).T + np.abs(bias))
    else:
        z = base.astype(np.float64)
        ez = np.zeros_like(z)
    t, et = np.zeros((m, r)), np.zeros((m, r))
    for i, rows in enumerate(rows_of(idx, m, e)):
        if not len(rows):
            continue
        t[rows] = x[rows] @ a[i].T
        et[rows] = (k + 16) * U * (np.abs(x[rows]) @ np.abs(a[i]).T)
        up = np.abs(t[rows]) @ np.abs(b[i]).T
        z[rows] = z[rows] + s[i] * (t[rows] @ b[i].T)
        ez[rows] = ez[rows] + s[i] * (et[rows] @ np.abs(b[i]).T + (r + 16) * U * up) + 4 * U * (np.abs(z[rows]) + s[i] * up)
    return act(z, kind), t, ez + 4 * U * np.abs(act(z, kind)) + 1e-37, et + 1e-37


def backward(x, w, a, b, s, idx, kind, y, dy, t, base=None):
    """dict name -> (value, bound) for dx, da, db, dw, dbias."""
    x, a, b, s, y, dy, t = (v.astype(np.float64) for v in (x, a, b, s, y, dy, t))
    m, k = x.shape
    e, n, r = b.shape
    g = act_grad(dy, y, kind)
    eg = (4 * U * np.abs(dy) * (1 + y * y)) if kind == "tanh" else np.zeros_like(g)
    ag, ax, at = np.abs(g), np.abs(x), np.abs(t)
    if w is not None:
        w = w.astype(np.float64)
        dx, ex = g @ w, (n + 16) * U * (ag @ np.abs(w)) + eg @ np.abs(w)
    else:
        dx = base.astype(np.float64)
        ex = np.zeros_like(dx)
    da, db, ea, eb = np.zeros_like(a), np.zeros_like(b), np.zeros_like(a), np.zeros_like(b)
    for i, rows in enumerate(rows_of(idx, m, e)):
        if not len(rows):
            continue
        dt = s[i] * (g[rows] @ b[i])
        edt = s[i] * ((n + 16) * U * (ag[rows] @ np.abs(b[i])) + eg[rows] @ np.abs(b[i])) + U * np.abs(dt)
        low = np.abs(dt) @ np.abs(a[i])
        dx[rows] = dx[rows] + dt @ a[i]
        ex[rows] = ex[rows] + edt @ np.abs(a[i]) + (r + 16) * U * low + 4 * U * (np.abs(dx[rows]) + low)
        c = len(rows)
        da[i] = dt.T @ x[rows]
        ea[i] = edt.T @ ax[rows] + (c + 16) * U * (np.abs(dt).T @ ax[rows])
        db[i] = s[i] * (g[rows].T @ t[rows])
        eb[i] = s[i] * ((c + 16) * U * (ag[rows].T @ at[rows]) + eg[rows].T @ at[rows])
    out = {"dx": (dx, ex + 1e-37), "da": (da, ea + 1e-37), "db": (db, eb + 1e-37)}
    out["dw"] = (g.T @ x, (m + 16) * U * (ag.T @ ax) + eg.T @ ax + 1e-37)
    out["dbias"] = (g.sum(0), (m + 16) * U * ag.sum(0) + eg.sum(0) + 1e-37)
    return out


def inputs(seed, m, n, k, r, e, mix):
    rng = np.random.default_rng(seed)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)   # noqa: E731
    d = dict(x=f(m, k), w=f(n, k) * np.float32(k ** -0.5), bias=f(n), a=f(e, r, k) * np.float32(k ** -0.5),
             b=f(e, n, r) * np.float32(r ** -0.5), s=(rng.random(e) * 1.5 + 0.5).astype(np.float32), y=f(m, n), dy=f(m, n), dx=f(m, k))
    if mix == "one":
        d["idx"] = None
    elif mix == "none":
        d["idx"] = np.full(m, -1, np.int32)
    elif mix == "last":           # all rows on the last adapter: the others are empty
        d["idx"] = np.full(m, e - 1, np.int32)
    elif mix == "sorted":
        d["idx"] = np.sort(rng.integers(-1, e, m)).astype(np.int32)
    else:
        d["idx"] = rng.integers(-1, e, m).astype(np.int32)
    return d


def clip(gs, max_norm, eps):
    """(norm, coefficient) in 64 bits."""
    norm = np.sqrt(sum(float((g.astype(np.float64) ** 2).sum()) for g in gs))
    return norm, min(1.0, max(0.0, max_norm / (norm + eps)))


def adam(p, g, m, v, t, coef, b1=0.9, b2=0.999, lr=1e-3, eps=1e-8, cwd=0.0, dfac=1.0):
    p, g, m, v = (q.astype(np.float64) for q in (p, g, m, v))
    g = coef * g + cwd * p
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    return p * dfac - lr * (m / (1 - b1 ** t)) / (np.sqrt(v / (1 - b2 ** t)) + eps), m, v
