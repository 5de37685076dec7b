"""The operators of functional/operators.py in plain float64 NumPy, written from their formulas: test oracles."""

import math

import numpy as np

ACTIVATIONS = ("silu", "gelu", "relu", "sigmoid")


def heads_inputs(rng, b, s, n, nkv, d, rot, table, dtype="float32", weights=True, positions=True):
    """Inputs by name: q, k, cos, sin, [wq, wk], [positions], gq, gk."""
    x = {"q": rng.standard_normal((b, s, n, d)) * 1.5, "k": rng.standard_normal((b, s, nkv, d)) * 1.5}
    x = {name: v.astype(dtype) for name, v in x.items()}
    angle = np.arange(table)[:, None] * 10000.0 ** (-np.arange(rot // 2) / max(rot // 2, 1))
    x["cos"], x["sin"] = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    if weights:
        x["wq"], x["wk"] = ((1 + 0.1 * rng.standard_normal(d)).astype(dtype) for _ in range(2))
    if positions:
        x["positions"] = rng.integers(0, table, (b, s)).astype(np.int32)
    x["gq"], x["gk"] = rng.standard_normal((b, s, n, d)).astype(dtype), rng.standard_normal((b, s, nkv, d)).astype(dtype)
    return x


def _matrix(cos, sin, d, interleaved):
    """The d x d matrix that turns a head by one row of the tables."""
    half = len(cos)
    r = np.eye(d)
    for i in range(half):
        p, q = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        r[p, p], r[p, q], r[q, p], r[q, q] = cos[i], -sin[i], sin[i], cos[i]
    return r


def heads(x, eps, interleaved):
    """[q, k turned, dq, dk, dwq, dwk] (the weights' gradients where there are weights) for cotangents gq and gk."""
    x = {k: np.asarray(v, np.int64 if k == "positions" else np.float64) for k, v in x.items()}
    b, s = x["q"].shape[:2]
    d = x["q"].shape[3]
    at = x.get("positions", np.broadcast_to(np.arange(s), (b, s)))
    at = np.clip(at, 0, max(len(x["cos"]) - 1, 0))
    turn = np.empty((b, s, d, d))
    for i in range(b):
        for j in range(s):
            turn[i, j] = _matrix(x["cos"][at[i, j]], x["sin"][at[i, j]], d, interleaved)
    out, dx, dw = [], [], []
    for h, w, g in (("q", "wq", "gq"), ("k", "wk", "gk")):
        weight = x.get(w, np.ones(d))
        inv = 1 / np.sqrt((x[h] ** 2).mean(-1, keepdims=True) + eps)
        xhat = x[h] * inv
        out.append(np.einsum("bsij,bsnj->bsni", turn, xhat * weight))
        dz = np.einsum("bsji,bsnj->bsni", turn, x[g])
        dxhat = dz * weight
        dx.append(inv * (dxhat - xhat * (dxhat * xhat).mean(-1, keepdims=True)))
        if w in x:
            dw.append((dz * xhat).sum((0, 1, 2)))
    return out + dx + dw


def activation(name, g):
    """act(g) and its derivative."""
    s = 1 / (1 + np.exp(-g))
    if name == "silu":
        return g * s, s + g * s * (1 - s)
    if name == "sigmoid":
        return s, s * (1 - s)
    if name == "relu":
        return np.where(g > 0, g, 0), np.where(g > 0, 1.0, 0.0)
    c, a = 0.7978845608, 0.044715
    t = np.tanh(c * (g + a * g**3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * a * g * g)


def gated(x, gate, up, dh, name):
    """[h, dx, dgate, dup] of rows ``x`` [..., K]."""
    x, gate, up, dh = (np.asarray(v, np.float64) for v in (x, gate, up, dh))
    lead = x.shape[:-1]
    rows, d = x.reshape(math.prod(lead), -1), dh.reshape(math.prod(lead), -1)
    g, u = rows @ gate.T, rows @ up.T
    a, da = activation(name, g)
    dg, du = d * u * da, d * a
    return [(a * u).reshape(*lead, -1), (dg @ gate + du @ up).reshape(x.shape), dg.T @ rows, du.T @ rows]


def differences(value, x, name, step=1e-6):
    """Central differences of ``value(x)`` by every element of ``x[name]``."""
    grad = np.zeros(x[name].shape)
    for i in np.ndindex(*x[name].shape):
        v = []
        for sign in (1, -1):
            moved = x[name].copy()
            moved[i] += sign * step
            v.append(value({**x, name: moved}))
        grad[i] = (v[0] - v[1]) / (2 * step)
    return grad
