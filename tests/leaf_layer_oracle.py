"""Layers of a forest's leaves, their gradients and clipping in 64 bits, in numpy: what tests
compare with.  Each result comes with a bound of how far float32 arithmetic may be off."""
import math

import numpy as np

U = 2.0 ** -24
ACTIVATIONS = ("none", "relu", "silu", "gelu", "gelu_tanh", "sigmoid")
_erf = np.vectorize(math.erf, otypes=[np.float64])


def _sigmoid(z):
    e = np.exp(-np.abs(z))
    return np.where(z >= 0, 1, e) / (1 + e)


def activation(z, act):
    if act == "relu":
        return np.maximum(z, 0)
    if act == "silu":
        return z * _sigmoid(z)
    if act == "gelu":
        return 0.5 * z * (1 + _erf(z / math.sqrt(2)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + np.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if act == "sigmoid":
        return _sigmoid(z)
    return z


def slope(z, act):
    if act == "relu":
        return (z > 0).astype(np.float64)
    if act == "silu":
        p = _sigmoid(z)
        return p + z * p * (1 - p)
    if act == "gelu":
        return 0.5 * (1 + _erf(z / math.sqrt(2))) + z * np.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = np.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if act == "sigmoid":
        p = _sigmoid(z)
        return p * (1 - p)
    return np.ones_like(z)


# An activation's slope is 1.13 at most.  Its value in float32: the exponential's argument is
# off by 3 U |z| at most, which moves a sigmoid by 3 U |z| / 4 < U where |z| (1 - p) p is
# largest; the exponential, the reciprocal and erf are off by few ulp, erf's approximation by
# 1.5e-7 = 2.5 U, a polynomial's roundings by about as much again: 16 U |z| bounds them all
# (16 U for the sigmoid itself).
STEEPEST = 1.13


def value_error(z, act):
    if act in ("none", "relu"):
        return np.zeros_like(z)
    return 16 * U * (np.ones_like(z) if act == "sigmoid" else np.abs(z))


# A slope: p (1 - p) is off by 8 U or so and is multiplied by |z|, for gelu_tanh by |z| (1 +
# 0.134 z^2) too, as long as 1 - p is not 0 in float32 (|z| < 18, and < 6).
def slope_error(z, act):
    if act in ("none", "relu"):
        return np.zeros_like(z)
    m = np.minimum(np.abs(z), 6 if act == "gelu_tanh" else 18)
    return 16 * U * (1 + m) * (1 + 0.134 * m * m if act == "gelu_tanh" else 1)


def layer(x, w, b, leaf, leaves, act, gated, res):
    """(y, its bound, z [trees, rows, R], the size of z's terms)."""
    rows, trees = leaf.shape
    R, K = w.shape[1:]
    H = R // 2 if gated else R
    y = np.zeros((rows, H)) if res is None else res.copy()
    total, off = np.abs(y), np.zeros((rows, H))
    z, size = np.zeros((trees, rows, R)), np.zeros((trees, rows, R))
    for t in range(trees):
        for l in range(leaves):
            n, g = np.flatnonzero(leaf[:, t] == l), t * leaves + l
            if not len(n):
                continue
            v, s = x[n] @ w[g].T, np.abs(x[n]) @ np.abs(w[g]).T
            if b is not None:
                v, s = v + b[g], s + np.abs(b[g])
            z[t, n], size[t, n] = v, s
            e = 2 * (K + 3) * U * s
            f = activation(v[:, :H], act)
            ef = STEEPEST * e[:, :H] + value_error(v[:, :H], act)
            if gated:
                u, eu = v[:, H:], e[:, H:]
                f, ef = f * u, ef * np.abs(u) + np.abs(f) * eu + ef * eu + 2 * U * np.abs(f * u)
            y[n] += f
            total[n] += np.abs(f)
            off[n] += ef
    return y, off + 2 * (trees + 2) * U * total, z, size


def dz_of(dy, z, act, gated, eps, tiny):
    """dz [trees, rows, R] from the kept z, and its bound: rounded to a type of this eps and
    least normal."""
    H = dy.shape[1]
    g = z[..., :H]
    d, e = slope(g, act), slope_error(g, act)
    if gated:
        u = z[..., H:]
        f, ef = activation(g, act), value_error(g, act)
        dz = np.concatenate([dy * u * d, dy * f], -1)
        off = np.concatenate([np.abs(dy * u) * e, np.abs(dy) * ef], -1)
    else:
        dz, off = dy * d, np.abs(dy) * e
    return dz, off + 4 * U * np.abs(dz) + eps / 2 * (np.abs(dz) + off) + tiny * eps


def grads(dy, z, x, w, leaf, leaves, act, gated, eps, tiny):
    """{name: (value, bound)} of dx, dw and db."""
    rows, trees = leaf.shape
    G, R, K = w.shape
    if act == "none" and not gated:
        dz = np.broadcast_to(dy, (trees,) + dy.shape)
        off = np.zeros_like(dz)
    else:
        dz, off = dz_of(dy, z, act, gated, eps, tiny)
    dx, ex = np.zeros((rows, K)), np.zeros((rows, K))
    dw, ew = np.zeros(w.shape), np.zeros(w.shape)
    db, eb = np.zeros((G, R)), np.zeros((G, R))
    for t in range(trees):
        for l in range(leaves):
            n, g = np.flatnonzero(leaf[:, t] == l), t * leaves + l
            a, e = dz[t, n], off[t, n]
            dx[n] += a @ w[g]
            ex[n] += (e + 2 * (R * trees + 2) * U * (np.abs(a) + e)) @ np.abs(w[g])
            s = e + 2 * (rows + 2) * U * (np.abs(a) + e)
            dw[g], ew[g] = a.T @ x[n], s.T @ np.abs(x[n])
            db[g], eb[g] = a.sum(0), s.sum(0)
    return {"dx": (dx, ex), "dw": (dw, ew), "db": (db, eb)}


def clip(grads, limit):
    """(norm, the scale, the clipped gradients)"""
    norm = math.sqrt(math.fsum(float((g * g).sum()) for g in grads))
    scale = 1.0 if norm <= limit else limit / norm
    return norm, scale, [g * scale for g in grads]


# The normal distribution's tails keep their digits by erfc, where 1 + erf has none left.
_erfc = np.vectorize(math.erfc, otypes=[np.float64])


def gelu_tails(z, wide):
    """(gelu, its bound, its slope, its bound) of z as it is, relative to the values also far out.

    P = erfc(-z / sqrt 2) / 2.  float32: z / sqrt 2 is off by 2 U, which moves erfc by 2 U (z^2 + 1)
    at most; erfc by 16 ulp (what OpenCL asks of it), the products by a few U.  16 bits (`wide`
    false): the polynomial by 5e-6, its roundings by 48 U, the exponential's argument by 3 U z^2 / 2 and
    the instruction by 2 U.  The slope adds z times the density, whose argument is off as much."""
    p = 0.5 * _erfc(-z / math.sqrt(2))
    d = np.abs(z) * np.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    rel = (40 + 3 * z * z) * U if wide else 5e-6 + (56 + 3 * z * z) * U
    return z * p, rel * np.abs(z * p), p + np.copysign(d, z), rel * (p + d)


def sigmoid_slope_tails(z):
    """(the sigmoid's slope, its bound) of z as it is, relative to it also far out: with e = exp(-|z|) it is
    e / (1 + e)^2, whose exponential is off by 2 U |z| (its argument) and 6 U, the quotient by a few U."""
    e = np.exp(-np.abs(z))
    d = e / (1 + e) ** 2
    return d, (16 + 2 * np.abs(z)) * U * d
