"""Gated linear recurrence and group norm with an activation, restated in float64 NumPy from their definitions, with
running bounds on what a float32 evaluation may be off by.

The bounds count roundings of half a step, ``U = 2^-24`` relative, to first order.  ``units`` is what a single factor (a gate,
an exponential, a quotient) may be off by, in such units: float32 results use functions accurate to two units in the last
place (2 ulp = 4 U each; a gate takes two of them, a sum and a product), 16-bit results the hardware's own (2 ulp and
1.2 ulp per unit of the argument, arguments below 10: 14 ulp).
"""
import numpy as np

U = 2.0 ** -24
UNITS = {4: 16.0, 2: 48.0}             # by the element size of the streams


def sigmoid(z):
    e = np.exp(-np.abs(z))
    return np.where(z >= 0, 1.0 / (1.0 + e), e / (1.0 + e))


def _coefficients(x, f, gate):
    """(a, u, w, what the gate's exponent adds to its relative error): w is 1 - a, or -da/df."""
    if gate == "sigmoid":
        a, w = sigmoid(f), sigmoid(-f)
        return a, w * x, w, np.zeros_like(f)
    with np.errstate(over="ignore", under="ignore", invalid="ignore"):
        e = np.exp(f)
        a = np.exp(-e)
        w = np.where(a == 0.0, 0.0, e * a)
        return a, x, w, np.where(a == 0.0, 0.0, e)


def gated(x, f, s, length, starts, gate, units=16.0):
    """One sequence: x, f (T, C), s (C,).  Returns (s_out, h) and the bounds of both."""
    T, C = x.shape
    a, u, w, more = _coefficients(x, f, gate)
    h, bound = s.copy(), np.zeros(C)
    s_out, s_bound = s.copy(), np.zeros(C)
    hs, bounds = np.empty((T, C)), np.empty((T, C))
    for t in range(T):
        if starts[t]:
            h, bound = np.zeros(C), np.zeros(C)
        bound = a[t] * bound + units * U * ((1.0 + more[t]) * a[t] * np.abs(h) + np.abs(u[t]))
        h = a[t] * h + u[t]
        hs[t], bounds[t] = h, bound
        if t == length - 1:
            s_out, s_bound = h, bound
    return (s_out, hs), (s_bound, bounds)


def gated_bwd(x, f, s, length, starts, gate, gs, gy, units=16.0):
    """Gradients (dx, df, ds) of one sequence and their bounds."""
    T, C = x.shape
    a, u, w, more = _coefficients(x, f, gate)
    (_, hs), (_, hb) = gated(x, f, s, length, starts, gate, units)
    dx, df, bx, bf = (np.empty((T, C)) for _ in range(4))
    c, cb = np.zeros(C), np.zeros(C)
    for t in range(T - 1, -1, -1):
        g = gy[t] + (gs if t == length - 1 else 0.0)
        dh = g + c
        db = cb + 2 * U * (np.abs(gy[t]) + (np.abs(gs) if t == length - 1 else 0.0) + np.abs(c))
        before, bb = (np.zeros(C), np.zeros(C)) if starts[t] else (hs[t - 1], hb[t - 1]) if t else (s, np.zeros(C))
        rel = units * U * (1.0 + more[t])
        if gate == "sigmoid":
            dx[t], bx[t] = w[t] * dh, w[t] * (db + rel * np.abs(dh))
            k = a[t] * w[t]
            df[t] = dh * (before - x[t]) * k
            bf[t] = k * (db * np.abs(before - x[t]) + np.abs(dh) * (bb + 2 * rel * (np.abs(before) + np.abs(x[t]))))
        else:
            dx[t], bx[t] = dh, db
            df[t] = -dh * before * w[t]
            bf[t] = w[t] * (db * np.abs(before) + np.abs(dh) * (bb + 2 * rel * np.abs(before)))
        if starts[t]:
            c, cb = np.zeros(C), np.zeros(C)
        else:
            c, cb = a[t] * dh, a[t] * (db + rel * np.abs(dh))
    if length == 0:
        c, cb = c + gs, cb + U * np.abs(gs)
    return (dx, df, c), (bx, bf, cb)


def activate(name, z):
    """act(z) and its derivative."""
    if name == "none":
        return z, np.ones_like(z)
    p, q = sigmoid(z), sigmoid(-z)
    return (p, p * q) if name == "sigmoid" else (z * p, p * (1.0 + z * q))


STEEP = {"none": (1.0, 0.0), "sigmoid": (0.25, 0.1), "silu": (1.1, 0.5)}       # most of |act'| and |act''|
SUM = 64.0                             # roundings that a sum over a group may take on one path


def group_norm(x, weight, bias, groups, gate, activation, eps, gy=None, units=16.0):
    """x (rows, C).  Returns (out,) or, with the cotangent, (out, dx, dweight, dbias, dgate or None), and the bounds."""
    rows, C = x.shape
    D = C // groups
    weight = np.ones(C) if weight is None else weight
    bias = np.zeros(C) if bias is None else bias
    fold = lambda z: z.reshape(rows, groups, D)
    flat = lambda z: np.ascontiguousarray(np.broadcast_to(z, (rows, groups, D))).reshape(rows, C)
    mean = lambda z: flat(fold(z).mean(2, keepdims=True))
    mu = mean(x)
    rstd = 1.0 / np.sqrt(mean((x - mu) ** 2) + eps)
    xh = (x - mu) * rstd
    n = xh * weight + bias
    b_xh = U * (SUM * np.abs(xh) + (SUM + 2) * (mean(np.abs(x)) + np.abs(x)) * rstd)
    b_n = np.abs(weight) * b_xh + 2 * U * (np.abs(xh * weight) + np.abs(n))
    rel = units * U
    if gate is not None:
        p, dp = activate(activation, gate)
        out, b_out = n * p, b_n * np.abs(p) + rel * np.abs(n * p)
    else:
        p, dp = activate(activation, n)
        out, b_out = p, b_n * STEEP[activation][0] + rel * np.abs(p)
    if gy is None:
        return (out,), (b_out,)
    dgate = b_gate = None
    if gate is not None:
        dn, b_dn = gy * p, np.abs(gy) * rel * np.abs(p)
        dgate = gy * n * dp
        b_gate = np.abs(gy) * (b_n * np.abs(dp) + rel * np.abs(n) * (np.abs(dp) + STEEP[activation][0]))
    else:
        dn, b_dn = gy * dp, np.abs(gy) * (STEEP[activation][1] * b_n + rel * (np.abs(dp) + STEEP[activation][0]))
    dw, db = (dn * xh).sum(0), dn.sum(0)
    b_dw = (b_dn * np.abs(xh) + np.abs(dn) * b_xh).sum(0) + rows * U * np.abs(dn * xh).sum(0)
    b_db = b_dn.sum(0) + rows * U * np.abs(dn).sum(0)
    dxh, b_dxh = dn * weight, b_dn * np.abs(weight) + U * np.abs(dn * weight)
    s1, s2 = mean(dxh), mean(dxh * xh)
    b_s1 = mean(b_dxh) + SUM * U * mean(np.abs(dxh))
    b_s2 = mean(b_dxh * np.abs(xh) + np.abs(dxh) * b_xh) + SUM * U * mean(np.abs(dxh * xh))
    dx = rstd * (dxh - s1 - xh * s2)
    b_dx = rstd * (b_dxh + b_s1 + np.abs(xh) * b_s2 + np.abs(s2) * b_xh + SUM * U * (np.abs(dxh) + np.abs(s1) + np.abs(xh * s2)))
    return (out, dx, dw, db, dgate), (b_out, b_dx, b_dw, b_db, b_gate)
