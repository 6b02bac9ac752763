"""The layer operators from their definitions, in float64 on the host, with
bounds on the rounding of a computation in a type of unit roundoff u.

Each bound follows the formulas term by term: one rounding of a value x is at
most u |x|; the sigmoid's two parts, the exponential among them, are taken as
good to 8 roundings of their own size, an activation and its slope to 16.
"""

from __future__ import annotations

import math

import numpy as np

U = {np.dtype(np.float32): 2.0 ** -24, np.dtype(np.float64): 2.0 ** -53}
SIGMOID, ACT = 8, 16


def sigmoid(z):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-z)), 1.0 / (1.0 + np.exp(z))


def recurrence(a, b, state, gate, u):
    """(h, bound) along axis 1 of (outer, length, inner): with an error E of
    h_{t-1}, h_t is off by at most |alpha| E and the roundings of its terms."""
    a, b = a.astype(np.float64), b.astype(np.float64)
    if gate == "sigmoid":
        a, rest = sigmoid(a)
        b = rest * b
        k = 2 * SIGMOID + 4
    else:
        k = 4
    h, bound = np.empty_like(a), np.empty_like(a)
    x = np.zeros(a[:, 0].shape) if state is None else state.astype(np.float64)
    e = np.zeros_like(x)
    for t in range(a.shape[1]):
        kept = a[:, t] * x
        x = kept + b[:, t]
        e = np.abs(a[:, t]) * e + k * u * (np.abs(kept) + np.abs(b[:, t]) + np.abs(x))
        h[:, t], bound[:, t] = x, e
    return h, bound


def recurrence_backward(a, b, h, dh, state, dfinal, gate, u):
    """((da, db, dstate), their bounds), with h as given."""
    a, h, dh = (v.astype(np.float64) for v in (a, h, dh))
    start = np.zeros(a[:, 0].shape) if state is None else state.astype(np.float64)
    back = np.zeros_like(start) if dfinal is None else dfinal.astype(np.float64)
    k = 4 if gate == "linear" else 2 * SIGMOID + 4
    alpha, rest = sigmoid(a) if gate == "sigmoid" else (a, None)
    da, db, eda, edb = (np.empty_like(a) for _ in range(4))
    e = np.zeros_like(start)
    for t in reversed(range(a.shape[1])):
        g = dh[:, t] + back
        e = e + k * u * (np.abs(dh[:, t]) + np.abs(back) + np.abs(g))
        before = h[:, t - 1] if t else start
        if gate == "linear":
            fa, fb = before, np.ones_like(before)
        else:
            fa = (before - b[:, t].astype(np.float64)) * alpha[:, t] * rest[:, t]
            fb = rest[:, t]
        da[:, t], db[:, t] = g * fa, g * fb
        eda[:, t] = np.abs(fa) * (e + 2 * k * u * np.abs(g))
        edb[:, t] = np.abs(fb) * (e + 2 * k * u * np.abs(g))
        back = alpha[:, t] * g
        e = np.abs(alpha[:, t]) * e + k * u * np.abs(back)
    return (da, db, back), (eda, edb, e + k * u * np.abs(back))


_erfc = np.vectorize(math.erfc, otypes=[np.float64])


def activate(z, act):
    if act == "relu":
        return np.where(z < 0, 0.0, z)
    if act == "silu":
        return z * sigmoid(z)[0]
    if act == "gelu":
        return z * 0.5 * _erfc(-z / math.sqrt(2.0))
    return z


def slope(z, act):
    if act == "relu":
        return (z > 0).astype(np.float64)
    if act == "silu":
        s, rest = sigmoid(z)
        return s * (1 + z * rest)
    if act == "gelu":
        return 0.5 * _erfc(-z / math.sqrt(2.0)) + z * np.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return np.ones_like(z)


def _per_channel(v, m):
    return np.repeat(v, m, axis=1)[:, None]


def group_norm(x, groups, weight, bias, eps, act, u):
    """((y, mean, rstd), bounds) of (N, S, C).  The sums are in float64 over
    n = S m values about the group's first value k, so the mean is off by at
    most n 2^-53 mean|x - k| and the variance by 2 n 2^-53 mean (x - k)^2."""
    n, s, c = x.shape
    m = c // groups
    v = x.astype(np.float64).reshape(n, s, groups, m)
    count = s * m
    mean = v.mean((1, 3))
    d = v - mean[:, None, :, None]
    var = (d * d).mean((1, 3))
    rstd = 1.0 / np.sqrt(var + eps)
    off = v - v[:, :1, :, :1]
    d64 = (count + 8) * 2.0 ** -53
    emean = d64 * (np.abs(off).mean((1, 3)) + np.abs(v[:, 0, :, 0]))
    erstd = rstd * (4 * d64 * (off * off).mean((1, 3)) * rstd ** 2 + 2 * u)
    xhat = (d * rstd[:, None, :, None]).reshape(n, s, c)
    w = np.ones(c) if weight is None else weight.astype(np.float64)
    b = np.zeros(c) if bias is None else bias.astype(np.float64)
    z = xhat * w + b
    y = activate(z, act)
    dabs = np.abs(d).reshape(n, s, c)
    exhat = dabs * _per_channel(erstd, m) + _per_channel(emean * rstd, m) + 4 * u * np.abs(xhat)
    # An activation's slope is at most 1.13 in size.
    ey = 1.2 * (np.abs(w) * exhat + 2 * u * (np.abs(z) + np.abs(xhat * w))) + ACT * u * np.abs(y)
    return (y, mean, rstd), (ey, emean + u * np.abs(mean), erstd)


def group_norm_backward(dy, x, groups, mean, rstd, weight, bias, act, u):
    """((dx, dweight, dbias), bounds) with mean and rstd as given.  A slope
    is off by ACT u and by the error of z times its own slope (below 1.2)."""
    n, s, c = x.shape
    m = c // groups
    r = _per_channel(rstd.astype(np.float64), m)
    xhat = (x.astype(np.float64) - _per_channel(mean.astype(np.float64), m)) * r
    w = np.ones(c) if weight is None else weight.astype(np.float64)
    b = np.zeros(c) if bias is None else bias.astype(np.float64)
    z = xhat * w + b
    g = dy.astype(np.float64)
    sl = slope(z, act)
    dz = g * sl
    edz = np.abs(g) * (ACT * u + 1.2 * 4 * u * (np.abs(xhat * w) + np.abs(z))) + u * np.abs(dz)
    if act == "relu":
        # The slope jumps at 0: a z within its rounding of 0 may fall on either side.
        edz = np.where(np.abs(z) <= 4 * u * (np.abs(xhat * w) + np.abs(b)), np.abs(g), u * np.abs(dz))

    def average(v):
        return _per_channel(v.reshape(n, s, groups, m).mean((1, 3)), m)

    count, n64 = s * m, 2.0 ** -53
    m1, m2 = average(w * dz), average(w * dz * xhat)
    eprod = edz * np.abs(xhat) + 4 * u * np.abs(dz * xhat)
    em1 = average(np.abs(w) * (edz + (count + 4) * n64 * np.abs(dz))) + u * np.abs(m1)
    em2 = average(np.abs(w) * (eprod + (count + 4) * n64 * np.abs(dz * xhat))) + u * np.abs(m2)
    dx = r * (w * dz - m1 - xhat * m2)
    edx = np.abs(r) * (np.abs(w) * edz + em1 + np.abs(xhat) * em2
                       + 6 * u * (np.abs(w * dz) + np.abs(m1) + np.abs(xhat * m2)))
    rows = n * s
    dw, db = (dz * xhat).sum((0, 1)), dz.sum((0, 1))
    edw = (eprod + (rows + 4) * n64 * np.abs(dz * xhat)).sum((0, 1)) + u * np.abs(dw)
    edb = (edz + (rows + 4) * n64 * np.abs(dz)).sum((0, 1)) + u * np.abs(db)
    return (dx, dw, db), (edx, edw, edb)


def adamw(p, g, m, v, scale, lr, betas, eps, decay, step, u):
    """((p, m, v), bounds) of one step."""
    p, g, m, v = (q.astype(np.float64) for q in (p, g, m, v))
    g = g * scale
    b1, b2 = betas
    m1 = b1 * m + (1 - b1) * g
    v1 = b2 * v + (1 - b2) * g * g
    em = 5 * u * (np.abs(b1 * m) + np.abs((1 - b1) * g))
    ev = 7 * u * v1  # every term of v is positive
    root = np.sqrt(v1 / (1 - b2 ** step)) + eps
    rate = lr / (1 - b1 ** step)
    change = rate * m1 / root
    p1 = p * (1 - lr * decay) - change
    ep = 3 * u * np.abs(p) + rate * em / root + 12 * u * np.abs(change) + 2 * u * np.abs(p1)
    return (p1, m1, v1), (ep, em, ev)
