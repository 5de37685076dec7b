"""The operators of a training step (packed attention, the linear cross entropy and AdamW) in plain float64 NumPy, written from
their formulas, with how far rounding can take a kernel from them: test oracles."""

import numpy as np

U = {"float32": 2.0**-24, "bfloat16": 2.0**-8, "float16": 2.0**-11}  # half a step of a type, relative to the value
LOW = {"float32": 0.0, "bfloat16": 0.0, "float16": 2.0**-25}  # half a step of its smallest values
F32 = 2.0**-24


def packed_inputs(rng, tokens, n, nkv, d, dv=None, std=1.0):
    dv = d if dv is None else dv
    shapes = {"q": (tokens, n, d), "k": (tokens, nkv, d), "v": (tokens, nkv, dv), "do": (tokens, n, dv)}
    return {name: rng.standard_normal(s) * std for name, s in shapes.items()}


def offsets_of(lengths, first=0):
    return np.concatenate([[first], first + np.cumsum(lengths)]) if len(lengths) else np.array([first])


def packed(x, offsets, causal, scale, dtype="float32"):
    """``([o, dq, dk, dv], their tolerances)``: a result's rounding to ``dtype``, that of every probability and of every dS to it
    (which the gradients' sums take over), of o within rowsum(dO O), and what float32 sums and exponentials add."""
    q, k, v, do = (np.asarray(x[name], np.float64) for name in ("q", "k", "v", "do"))
    t, n, d = q.shape
    group = n // k.shape[1]
    u, low = U[dtype], LOW[dtype]
    out = [np.zeros((t, n, v.shape[2])), np.zeros(q.shape), np.zeros(k.shape), np.zeros(v.shape)]
    tol = [np.zeros(y.shape) for y in out]
    for lo, hi in zip(offsets, offsets[1:]):
        if hi <= lo:
            continue
        for h in range(n):
            Q, K, V, G = q[lo:hi, h], k[lo:hi, h // group], v[lo:hi, h // group], do[lo:hi, h]
            s = Q @ K.T * scale
            size = np.abs(Q) @ np.abs(K).T * scale  # what a score's sum adds up
            seen = np.tri(hi - lo) > 0 if causal else np.ones(s.shape, bool)
            s = np.where(seen, s, -np.inf)
            p = np.exp(s - s.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            # a probability's relative error: the score's sum, its products by constants, the exponential and the row's sum
            ep = F32 * ((d + 8) * size.max() + 2 * (hi - lo) + 60)
            o = p @ V
            to = u * np.abs(o) + (u + ep) * (p @ np.abs(V)) + low * (seen @ np.abs(V))
            dp, delta = G @ V.T, (G * o).sum(1, keepdims=True)
            tdelta = (np.abs(G) * (to + F32 * (d + 8) * np.abs(o))).sum(1, keepdims=True)
            ds = p * (dp - delta) * scale
            tds = u * np.abs(ds) + low + scale * p * (ep * np.abs(dp - delta) + tdelta + F32 * (d + 16) * (np.abs(G) @ np.abs(V).T))
            tds = np.where(seen, tds, 0.0)
            tp = np.where(seen, (u + ep) * p + low, 0.0)
            more = u + F32 * (hi - lo + 8)
            out[0][lo:hi, h], tol[0][lo:hi, h] = o, to
            out[1][lo:hi, h] = ds @ K
            tol[1][lo:hi, h] = tds @ np.abs(K) + more * (np.abs(ds) @ np.abs(K))
            out[2][lo:hi, h // group] += ds.T @ Q
            tol[2][lo:hi, h // group] += tds.T @ np.abs(Q) + more * (np.abs(ds).T @ np.abs(Q))
            out[3][lo:hi, h // group] += p.T @ G
            tol[3][lo:hi, h // group] += tp.T @ np.abs(G) + more * (p.T @ np.abs(G))
    # a result below 2^-14 in float16 is a multiple of 2^-24: off by up to 2^-25, which is more than U times its value
    return out, [y + low + 1e-30 for y in tol]


def adamw(w, g, m, v, step, lr, betas, eps, decay):
    """``(w, m, v)`` after a step."""
    w, g, m, v = (np.asarray(x, np.float64) for x in (w, g, m, v))
    b1, b2 = betas
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    return w - lr * decay * w - lr * (m / (1 - b1**step)) / (np.sqrt(v / (1 - b2**step)) + eps), m, v


def adamw_tolerances(w, g, m, v, step, lr, betas, eps, decay):
    """Float32: four roundings of a moment's two terms; of the weight's product and its update a few more, the update's relative
    error doubled by that of the moments and its factors."""
    b1, b2 = betas
    w, g, m, v = (np.asarray(x, np.float64) for x in (w, g, m, v))
    tm = 6 * F32 * (b1 * np.abs(m) + (1 - b1) * np.abs(g)) + 1e-44
    tv = 6 * F32 * (b2 * np.abs(v) + (1 - b2) * g * g) + 1e-44
    _, m1, v1 = adamw(w, g, m, v, step, lr, betas, eps, decay)
    root = np.sqrt(v1 / (1 - b2**step)) + eps
    rate = lr / (1 - b1**step)
    tw = 4 * F32 * np.abs(w) + rate * tm / root + 12 * F32 * rate * np.abs(m1) / root
    tw += rate * np.abs(m1) / root**2 * np.sqrt(tv / (1 - b2**step))  # the root of a second moment near zero
    return tw + 1e-44, tm, tv


def linear_cross_entropy(h, w, target, ignore, g):
    """``(losses, dh, dw)`` for the losses' cotangents ``g``; ignored rows lose nothing."""
    h, w, g = (np.asarray(x, np.float64) for x in (h, w, g))
    logits = h @ w.T
    top = logits.max(1, keepdims=True)
    e = np.exp(logits - top)
    lse = top[:, 0] + np.log(e.sum(1))
    kept = target != ignore
    at = np.where(kept, target, 0)
    rows = np.arange(len(h))
    losses = np.where(kept, lse - logits[rows, at], 0.0)
    d = e / e.sum(1, keepdims=True)
    d[rows, at] -= 1
    d *= np.where(kept, g, 0.0)[:, None]
    return losses, d @ w, d.T @ np.where(kept[:, None], h, 0.0)


def linear_cross_entropy_tolerances(h, w, target, ignore, g, dtype):
    """Of ``(losses, dh, dw)``. A logit is a float32 sum of K products; a probability is off by that of its logit and of the lse,
    by the float32 sums and exponentials, by its 16 bits (2^-11, or 2^-40 of its block's largest) and by the rounding of the logits' gradient to ``dtype`` (float16's
    in units of at least 2^-38 of the largest cotangent); both are summed over by the products."""
    h, w, g = (np.asarray(x, np.float64) for x in (h, w, g))
    kept = target != ignore
    h = np.where(kept[:, None], h, 0.0)
    logits = h @ w.T
    size = (np.abs(h) @ np.abs(w).T).max(1) if h.shape[1] else np.zeros(len(h))
    el = F32 * (h.shape[1] + 8) * size
    top = logits.max(1, keepdims=True)
    e = np.exp(logits - top)
    p = e / e.sum(1, keepdims=True)
    lse = top[:, 0] + np.log(e.sum(1))
    spread = np.abs(logits - lse[:, None])
    tloss = np.where(kept, 2 * el + F32 * (100 + 2 * np.abs(lse) + 2 * np.abs(top[:, 0])), 1e-30)
    g = np.where(kept, g, 0.0)
    rows = np.arange(len(h))
    at = np.clip(np.where(kept, target, 0), 0, len(w) - 1)
    d = p.copy()
    d[rows, at] -= 1
    d = np.abs(d * g[:, None])
    u = U[dtype]
    low = 2.0**-38 * np.abs(g).max(initial=0) if dtype == "float16" else 0.0
    rel = 2.0**-11 + (2 * el + F32 * 100)[:, None] + 4 * F32 * spread
    td = u * d + low + np.abs(g)[:, None] * (p * rel + 2.0**-39)
    td[rows, at] += np.abs(g) * tloss
    td[~kept] = 0.0
    tdh = u * (d @ np.abs(w)) + LOW[dtype] + td @ np.abs(w) + F32 * (len(w) + 8) * (d @ np.abs(w))
    tdw = u * (d.T @ np.abs(h)) + LOW[dtype] + td.T @ np.abs(h) + F32 * (len(h) + 8) * (d.T @ np.abs(h))
    return tloss, tdh + 1e-30, tdw + 1e-30
