"""An AdamW step over many weights as one operator (``adamw``), beside ``clip_grad_norm``: the reference's optimizer
(``examples/optim.py``) is SGD, written out weight by weight."""

from __future__ import annotations

import math

from lumen_amd import dtypes as D
from lumen_amd.autograd.function import Function
from lumen_amd.functional.operators import KERNEL_DTYPES, _operator
from lumen_amd.graph import prims
from lumen_amd.graph.tracer import TracedTensor, accum_dtype, broadcast_to, lift, require_float

OPERANDS = 4  # of a weight, one after another: its values (the master's where it has one), gradient and two moments


def adamw_scalars(params):
    """The names of the scalar operands ahead of the tensors'."""
    return [n for n in ("lr", "step") if params[n] is None] + (["scale"] if params["scaled"] else [])


def adamw_body(xs, params):
    """The results of an ``adamw`` fusion's operands ``xs``: new weights, first moments, second moments, then the masters
    that there are."""
    names = adamw_scalars(params)
    given = dict(zip(names, xs))
    xs = xs[len(names):]
    lr, t = (given[n].to("float64") if n in given else prims.full((), params[n], "float64") for n in ("lr", "step"))
    b1, b2, eps, decay = (params[n] for n in ("beta1", "beta2", "eps", "weight_decay"))

    def power(b):
        return prims.pow(prims.full((), b, "float64"), t)

    keep, rate, root = 1.0 - lr * decay, lr / (1.0 - power(b1)), 1.0 / prims.sqrt(1.0 - power(b2))
    weights, first, second, masters = [], [], [], []
    for i, master in enumerate(params["masters"]):
        w, g, m, v = xs[OPERANDS * i:OPERANDS * (i + 1)]
        acc, dtype = m.dtype, g.dtype

        def factor(x):
            x = prims.full((), x, "float64") if isinstance(x, float) else x
            return broadcast_to(x.to(acc), m.shape)

        g = g.to(acc)
        if "scale" in given:
            g = (g * factor(given["scale"])).to(dtype).to(acc)
        m = m * factor(b1) + g * factor(1.0 - b1)
        v = v * factor(b2) + (g * g) * factor(1.0 - b2)
        w = w.to(acc) * factor(keep) - (m * factor(rate)) / (prims.sqrt(v) * factor(root) + factor(eps))
        weights.append(w.to(dtype))
        first.append(m)
        second.append(v)
        masters += [w] if master else []
    return weights + first + second + masters


class _AdamW(Function):
    @staticmethod
    def forward(ctx, lr, step, *tensors, **params):
        scalars = [x for x in (lr, step) if isinstance(x, TracedTensor)]
        params.update(lr=None if isinstance(lr, TracedTensor) else lr, step=None if isinstance(step, TracedTensor) else step,
                      scaled=False)
        taken = all(g.dtype in KERNEL_DTYPES for g in tensors[1::OPERANDS])
        return _operator("adamw", taken, scalars + list(tensors), lambda *xs: adamw_body(list(xs), params), **params)

    @staticmethod
    def backward(ctx, *grads):
        raise NotImplementedError("adamw: its results have no gradient")


def _number(op, name, x, ok, what):
    if isinstance(x, bool) or not isinstance(x, (int, float)) or not ok(x) or math.isinf(x):
        raise ValueError(f"{op}: {name} must be {what}, got {x!r}")
    return float(x)


def _rate(op, name, x, ok, what):
    """A rate as a float64 scalar tensor (a count also int32 or int64), or a number known when the function is compiled."""
    if not isinstance(x, TracedTensor):
        return _number(op, name, x, ok, what)
    if x.shape != () or not (D.is_float(x.dtype) or D.is_int(x.dtype)):
        raise TypeError(f"{op}: {name} must be a number or a scalar, got {x!r}")
    return x if name == "step" and x.dtype in ("int32", "int64") else x.to("float64")


def adamw(params, grads, exp_avgs, exp_avg_sqs, step, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, masters=None):
    """One AdamW step over many weights: ``(params, exp_avgs, exp_avg_sqs, masters)``, lists of their new values.

    Of each weight ``w`` with gradient ``g`` and moments ``m`` and ``v``, ``t`` being ``step``, which counts from 1::

        m = beta1 m + (1 - beta1) g        v = beta2 v + (1 - beta2) g^2
        w = w (1 - lr weight_decay) - lr / (1 - beta1^t) m / (sqrt(v) / sqrt(1 - beta2^t) + eps)

    ``params``, ``grads``, ``exp_avgs`` and ``exp_avg_sqs`` are lists of equal length of tensors of equal shapes, a gradient of
    its weight's dtype and the moments float32 (float64 of float64 weights). Everything is computed in the moments' dtype, the
    step's factors in float64. A 16-bit weight loses updates below half its last place: ``masters`` keeps its float32 value
    beside it (a tensor for each weight, or None for one without), which is stepped in its place and rounded into it.
    ``step`` and ``lr`` are numbers, or scalar tensors that a compiled function may be called with anew. The results have no
    gradient."""
    op = "adamw"
    lists = {"params": params, "grads": grads, "exp_avgs": exp_avgs, "exp_avg_sqs": exp_avg_sqs}
    if masters is not None:
        lists["masters"] = masters
    for name, xs in lists.items():
        if isinstance(xs, TracedTensor) or not isinstance(xs, (list, tuple)):
            raise TypeError(f"{op}: {name} are a list or tuple of tensors, got {xs!r}")
        if len(xs) != len(params):
            raise ValueError(f"{op}: {len(params)} params and {len(xs)} {name}")
    if not params:
        raise ValueError(f"{op}: no params")
    if not isinstance(betas, (list, tuple)) or len(betas) != 2:
        raise ValueError(f"{op}: betas are two numbers, got {betas!r}")
    b1, b2 = (_number(op, "a beta", b, lambda x: 0 <= x < 1, "at least 0 and below 1") for b in betas)
    eps = _number(op, "eps", eps, lambda x: x >= 0, "at least 0")
    weight_decay = _number(op, "weight_decay", weight_decay, lambda x: x >= 0, "at least 0")
    step = _rate(op, "step", lift(step), lambda x: x >= 1, "at least 1")
    lr = _rate(op, "lr", lift(lr), lambda x: x >= 0, "at least 0")
    masters = [None] * len(params) if masters is None else list(masters)
    operands = []
    for i, (p, g, m, v, w) in enumerate(zip(params, grads, exp_avgs, exp_avg_sqs, masters)):
        p, g, m, v, w = (lift(x) for x in (p, g, m, v, w))
        if not isinstance(p, TracedTensor):
            raise TypeError(f"{op}: params are tensors, got {p!r}")
        require_float(p, op)
        state = accum_dtype(p.dtype)
        for name, x, dtype in (("gradient", g, p.dtype), ("first moment", m, state), ("second moment", v, state),
                               ("master", p if w is None else w, p.dtype if w is None else "float32")):
            if not isinstance(x, TracedTensor) or x.dtype != dtype or x.shape != p.shape:
                raise TypeError(f"{op}: the {name} of weight {i} must be {dtype}{list(p.shape)}, got {x!r}")
        if w is not None and p.dtype not in ("bfloat16", "float16"):
            raise TypeError(f"{op}: weight {i} is {p.dtype}: masters are of 16-bit weights")
        operands += [p if w is None else w, g, m, v]
    has = tuple(w is not None for w in masters)
    out = iter(_AdamW.apply(lr, step, *operands, masters=has, beta1=b1, beta2=b2, eps=eps, weight_decay=weight_decay))
    new = [[next(out) for _ in params] for _ in range(3)]
    return (*new, [next(out) if w else None for w in has] if any(has) else None)
