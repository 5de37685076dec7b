"""Operators that run as hand-written kernels of their own: the norms and rotation of attention heads
(``qk_norm_rope``), the projections of a gated MLP (``gated_linear``) and clipping by the norm over many gradients
(``clip_grad_norm``).

Each is defined by elementary primitives. Where the hip kernels take its dtypes the trace holds one ``fusion`` of that
body, which the plan runs as a built-in step and the oracle evaluates as written; elsewhere, and with
``config.compiler.fused_operators`` off, it holds the primitives themselves. The reference has no counterpart: its
programs write these out.

A tape sees neither: both directions are a ``Function`` each, whose forward runs with the tapes paused. A gradient is
differentiated again through the primitives that define it (``_second``).
"""

from __future__ import annotations

import math

from lumen_amd import dtypes as D
from lumen_amd.autograd.function import Function
from lumen_amd.config import config
from lumen_amd.functional import functions as F
from lumen_amd.graph import prims, tracer
from lumen_amd.graph.ir import Graph
from lumen_amd.graph.tracer import TracedTensor, accum_dtype, broadcast_to, dot, lift, require_float

KERNEL_DTYPES = ("float32", "bfloat16", "float16")
MAX_HEAD = 1024  # a head's elements in the head kernels
MAX_ROW = 1 << 21  # elements of a row of the gated projections: tiles of rows within 2^31 bytes
MAX_FEATURES = 1 << 26  # of them: workgroups of 512 threads for 16 features each within 2^31 threads
ACTIVATIONS = ("silu", "gelu", "relu", "sigmoid")


def _fused(name, operands, body, **params):
    """One ``fusion`` called ``name`` of ``operands``, its body what ``body(*operands)`` traces; the body's results. Only
    within a ``Function``'s forward: an open tape would take the body's nodes, whose values are of another graph, and no
    tape takes the fusion."""
    if tracer._TAPES:
        raise RuntimeError(f"{name}: a fusion is traced with the tapes paused")
    graph = tracer.current_graph()
    inner = Graph()
    inputs = [TracedTensor(inner, inner.input(x.dtype, x.shape)) for x in operands]
    with tracer.tracing(inner):
        results = body(*inputs)
    inner.set_outputs([r.var for r in results])
    first = graph.apply("fusion", [x.var for x in operands], dict(params, name=name, body=inner))
    out = [first]
    for j, r in enumerate(results[1:], 1):
        out.append(graph.apply("fusion_output", [first], {"index": j, "ty": inner.type_of(r.var)}))
    return tuple(TracedTensor(graph, v) for v in out)


def _operator(name, taken, operands, body, **params):
    """``body(*operands)`` as one fusion where ``taken`` (the kernels take these types), else as primitives."""
    if taken and config.compiler.fused_operators:
        return _fused(name, operands, body, **params)
    return tuple(body(*operands))


def _second(grads, primals, cotangents):
    """The cotangents of ``primals`` (None where there is none) for those of ``grads(*primals)``'s results."""
    from lumen_amd.autograd.transforms import vjp

    used = [p for p in primals if p is not None]
    first = {}  # one leaf a value: of a value passed twice the first has the sum
    for p in used:
        first.setdefault(p.var, p)

    def by_leaf(*leaves):
        at = dict(zip(first, leaves))
        return grads(*(None if p is None else at[p.var] for p in primals))

    _, pullback = vjp(by_leaf, *first.values())
    back = dict(zip(first, pullback(tuple(cotangents))))
    return [None if p is None else back.pop(p.var, None) for p in primals]


# ---- norms and rotation of heads ------------------------------------------------------------------------


def _turn(x, cos, sin, interleaved):
    """``x`` ``[B, S, N, D]`` with the pairs of its first elements turned by ``cos`` and ``sin`` ``[B, S, 1, R / 2]``."""
    r, d = 2 * cos.shape[-1], x.shape[-1]
    lead = x.shape[:-1]
    if r == 0:
        return x
    part = x[..., :r] if r < d else x
    if interleaved:
        pairs = part.reshape(*lead, r // 2, 2)
        a, b = pairs[..., 0:1].reshape(*lead, r // 2), pairs[..., 1:2].reshape(*lead, r // 2)
    else:
        a, b = part[..., : r // 2], part[..., r // 2:]
    shape = a.shape
    cos, sin = broadcast_to(cos, shape), broadcast_to(sin, shape)
    p, q = a * cos - b * sin, b * cos + a * sin
    turned = F.stack([p, q], -1).reshape(*lead, r) if interleaved else F.cat([p, q], -1)
    return turned if r == d else F.cat([turned, x[..., r:]], -1)


def _rows(table, positions, b, s):
    """``table``'s row of each token ``[B, S, 1, R / 2]`` (positions clamped into it)."""
    if positions is None:
        return broadcast_to(table[:s].reshape(1, s, 1, table.shape[1]), (b, s, 1, table.shape[1]))
    return prims.gather(table, positions, 0).reshape(b, s, 1, table.shape[1])


def _normed(x, acc, eps, rules=False):
    """``x`` over its root mean square and one over that, which ``rules`` makes of primitives with gradient rules."""
    h = x.to(acc)
    square = F.mean(h * h, -1, keepdim=True) + eps
    inv = 1.0 / prims.sqrt(square) if rules else prims.rsqrt(square)
    return h * broadcast_to(inv, h.shape), inv


def _expand(w, like):
    return broadcast_to(w.to(like.dtype).reshape(1, 1, 1, w.shape[0]), like.shape)


class _QKNormRope(Function):
    """Queries and keys normed and turned in one pass each; the backward takes x alone from the forward."""

    @staticmethod
    def forward(ctx, q, k, wq, wk, cos, sin, positions, *, eps, interleaved):
        ctx.eps, ctx.interleaved = eps, interleaved
        ctx.save_for_backward(q, k, wq, wk, cos, sin, positions)
        operands, roles = _heads_operands(q, k, wq, wk, cos, sin, positions)
        b, s = q.shape[:2]

        def body(*xs):
            x = dict(zip(roles, xs))
            acc = accum_dtype(q.dtype)
            c, n = (_rows(x[t], x.get("positions"), b, s).to(acc) for t in ("cos", "sin"))
            out = []
            for h, w in (("q", "q_weight"), ("k", "k_weight")):
                z, _ = _normed(x[h], acc, eps)
                z = z * _expand(x[w], z) if w in x else z
                out.append(_turn(z, c, n, interleaved).to(q.dtype))
            return out

        return _operator("qk_norm_rope", _heads_taken(q, k), operands, body, roles=roles, eps=float(eps),
                         interleaved=bool(interleaved))

    @staticmethod
    def backward(ctx, gq, gk):
        _, _, wq, wk, *_ = ctx.saved_tensors
        out = _QKNormRopeGradients.apply(gq, gk, *ctx.saved_tensors, eps=ctx.eps, interleaved=ctx.interleaved)
        dw = iter(out[2:])
        return (out[0], out[1], next(dw) if wq is not None else None, next(dw) if wk is not None else None,
                None, None, None)


class _QKNormRopeGradients(Function):
    """The heads' gradients and, where there are weights, theirs."""

    @staticmethod
    def forward(ctx, gq, gk, q, k, wq, wk, cos, sin, positions, *, eps, interleaved):
        ctx.eps, ctx.interleaved = eps, interleaved
        ctx.save_for_backward(gq, gk, q, k, wq, wk, cos, sin, positions)
        operands, roles = _heads_operands(q, k, wq, wk, cos, sin, positions)
        operands, roles = operands + [gq, gk], roles + ("gq", "gk")
        return _operator("qk_norm_rope_backward", _heads_taken(q, k), operands,
                         lambda *xs: _heads_gradients(dict(zip(roles, xs)), eps, interleaved), roles=roles,
                         eps=float(eps), interleaved=bool(interleaved))

    @staticmethod
    def backward(ctx, *cotangents):
        gq, gk, q, k, wq, wk, cos, sin, positions = ctx.saved_tensors

        def grads(gq, gk, q, k, wq, wk):
            operands, roles = _heads_operands(q, k, wq, wk, cos, sin, positions)
            return tuple(_heads_gradients({**dict(zip(roles, operands)), "gq": gq, "gk": gk}, ctx.eps, ctx.interleaved, rules=True))

        return (*_second(grads, (gq, gk, q, k, wq, wk), cotangents), None, None, None)


def _heads_gradients(x, eps, interleaved, rules=False):
    """``[dq, dk]`` and the gradients of the weights that there are, from the operands by role."""
    q = x["q"]
    b, s = q.shape[:2]
    acc = accum_dtype(q.dtype)
    c, n = (_rows(x[t], x.get("positions"), b, s).to(acc) for t in ("cos", "sin"))
    dx, dw = [], []
    for h, w, g in (("q", "q_weight", "gq"), ("k", "k_weight", "gk")):
        xhat, inv = _normed(x[h], acc, eps, rules)
        dz = _turn(x[g].to(acc), c, -n, interleaved)
        dxhat = dz * _expand(x[w], dz) if w in x else dz
        m = broadcast_to(F.mean(dxhat * xhat, -1, keepdim=True), xhat.shape)
        dx.append((broadcast_to(inv, xhat.shape) * (dxhat - xhat * m)).to(q.dtype))
        if w in x:
            dw.append(F.sum(dz * xhat, (0, 1, 2)).to(q.dtype))
    return dx + dw


def _heads_operands(q, k, wq, wk, cos, sin, positions):
    named = [("q", q), ("k", k), ("q_weight", wq), ("k_weight", wk), ("cos", cos), ("sin", sin), ("positions", positions)]
    named = [(n, x) for n, x in named if x is not None]
    return [x for _, x in named], tuple(n for n, _ in named)


def _heads_taken(q, k):
    return q.dtype in KERNEL_DTYPES and 0 < q.shape[3] <= MAX_HEAD and q.shape[1] < 1 << 30 \
        and max(q.shape[2], k.shape[2]) < 1 << 20


def qk_norm_rope(query, key, cos, sin, query_weight=None, key_weight=None, positions=None, eps=None, interleaved=False):
    """RMS norm and rotary position of every query and key head, ahead of ``flash_attention``: ``(query, key)`` of
    the same shapes and dtype.

    ``query`` ``[B, S, N, D]`` and ``key`` ``[B, S, Nkv, D]``; each head is divided by the root of its mean square plus
    ``eps`` (the dtype's machine epsilon by default, as ``rms_norm``), times its weight ``[D]`` (None: ones), and the
    first ``R`` of its ``D`` elements are turned by position: pair ``i`` as ``(a, b) -> (a cos - b sin, b cos + a sin)``
    with ``cos`` and ``sin`` float32 tables ``[P, R / 2]``. Pairs are elements ``i`` and ``i + R / 2``, or ``2 i`` and
    ``2 i + 1`` if ``interleaved``. A token's row of the tables is its ``positions`` (int32 or int64 ``[B, S]``, clamped
    into the tables), by default its index in the sequence. Sums, norms and turns are float32 (float64 of float64
    heads), each result rounded once. Gradients reach the heads and the weights, not the tables."""
    q, k, cos, sin = lift(query), lift(key), lift(cos), lift(sin)
    wq, wk, positions = lift(query_weight), lift(key_weight), lift(positions)
    op = "qk_norm_rope"
    for role, t in (("query", q), ("key", k)):
        if not isinstance(t, TracedTensor) or t.ndim != 4:
            raise ValueError(f"{op}: the {role} is not a 4-D [batch, seq, heads, head_dim] tensor: {t!r}")
        require_float(t, op)
    if q.dtype != k.dtype:
        raise TypeError(f"{op}: query is {q.dtype} and key {k.dtype}: convert them to one with .to(dtype)")
    if q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError(f"{op}: query {list(q.shape)} and key {list(k.shape)} differ in batch, sequence or head dim")
    d = q.shape[3]
    for role, t in (("cos", cos), ("sin", sin)):
        if not isinstance(t, TracedTensor) or t.ndim != 2 or t.dtype != "float32":
            raise ValueError(f"{op}: {role} is not a float32 [positions, rotated / 2] table: {t!r}")
    if cos.shape != sin.shape or 2 * cos.shape[1] > d:
        raise ValueError(f"{op}: tables {list(cos.shape)} and {list(sin.shape)} do not turn pairs of {d} elements")
    for role, t in (("query", wq), ("key", wk)):
        if t is not None and (not isinstance(t, TracedTensor) or t.dtype != q.dtype or t.shape != (d,)):
            raise TypeError(f"{op}: the {role} weight must be {q.dtype}[{d}], got {t!r}")
    if positions is None:
        if cos.shape[0] < q.shape[1]:
            raise ValueError(f"{op}: tables of {cos.shape[0]} positions for a sequence of {q.shape[1]}")
    elif not isinstance(positions, TracedTensor) or positions.dtype not in ("int32", "int64") \
            or positions.shape != q.shape[:2]:
        raise ValueError(f"{op}: positions must be int32 or int64 {list(q.shape[:2])}, got {positions!r}")
    elif cos.shape[0] == 0 and math.prod(q.shape[:2]):
        raise ValueError(f"{op}: tables of no positions")
    if eps is None:
        eps = {"float16": 2.0**-10, "bfloat16": 2.0**-7, "float64": 2.0**-52}.get(q.dtype, 2.0**-23)
    if isinstance(eps, bool) or not isinstance(eps, (int, float)) or not eps >= 0 or math.isinf(eps):
        raise ValueError(f"{op}: eps must be a number of at least 0 known when the function is compiled, got {eps!r}")
    return _QKNormRope.apply(q, k, wq, wk, cos, sin, positions, eps=float(eps), interleaved=bool(interleaved))


# ---- gated projections ----------------------------------------------------------------------------------


def _gelu_parts(g):
    v = 0.7978845608 * (g + 0.044715 * g * g * g)
    return v, prims.logistic(v + v)  # (1 + tanh(v)) / 2


def _activated(name, g):
    if name == "silu":
        return g * prims.logistic(g)
    if name == "gelu":
        return g * _gelu_parts(g)[1]
    if name == "relu":
        return F.relu(g)
    return prims.logistic(g)


def _activated_grad(name, g):
    """``act(g)`` and its derivative."""
    if name == "silu":
        s = prims.logistic(g)
        return g * s, s * (1.0 + g * (1.0 - s))
    if name == "gelu":
        _, s = _gelu_parts(g)
        a = g * s
        t = a * (1.0 - s) * (2.0 * 0.7978845608)  # 0 for large g, and g * g may be infinite
        return a, s + t + 3.0 * 0.044715 * (t * g) * g
    if name == "relu":
        zero = prims.full(g.shape, 0.0, g.dtype)
        return F.relu(g), F.where(prims.lt(zero, g), prims.full(g.shape, 1.0, g.dtype), zero)
    s = prims.logistic(g)
    return s, s * prims.logistic(-g)  # 1 - s would cancel: at g = 10 it is off by 1e-3 of itself


def _gated_taken(x, features):
    return x.dtype in ("bfloat16", "float16") and 0 < x.shape[1] < MAX_ROW and features < MAX_FEATURES


class _GatedLinear(Function):
    """``act(x gate^T) * (x up^T)`` of rows ``x`` ``[T, K]``; the backward takes both products, float32, from the
    forward (a plan without a backward neither computes nor stores them apart)."""

    @staticmethod
    def forward(ctx, x, gate, up, *, activation):
        def body(x, gate, up):
            g, u = _gated_products(x, gate, up)
            return [(_activated(activation, g) * u).to(x.dtype), g, u]

        h, g, u = _operator("gated_linear", _gated_taken(x, gate.shape[0]), [x, gate, up], body, activation=activation)
        ctx.activation = activation
        ctx.save_for_backward(x, gate, up, g, u)
        return h

    @staticmethod
    def backward(ctx, dh):
        return _GatedGradients.apply(dh, *ctx.saved_tensors, activation=ctx.activation)


def _gated_products(x, gate, up):
    acc = accum_dtype(x.dtype)
    return tuple(dot(x, w, (((1,), (1,)), ((), ())), acc, acc) for w in (gate, up))


class _GatedGradients(Function):
    """``(dx, dgate, dup)``: ``[dg | du]`` of the elements, then the products."""

    @staticmethod
    def forward(ctx, dh, x, gate, up, g, u, *, activation):
        ctx.activation = activation
        ctx.save_for_backward(dh, x, gate, up)
        (t, k), n = x.shape, gate.shape[0]
        whole = -(-n // 8) * 8  # each half of [dg | du] in whole 16-byte chunks
        taken = _gated_taken(x, n)
        (dgu,) = _operator("gated_linear_grad", taken, [dh, g, u],
                           lambda *xs: [_gated_elements(*xs, activation, whole)], activation=activation)
        row = -(-k // 8) * 8
        taken = taken and n < 1 << 21 and whole * row < (1 << 30) - 1024
        # the weights' gradients take tokens in at most 64 parts, the rows of each within 2^31 bytes
        taken = taken and -(-t // 4096) <= ((1 << 30) - 1024) // (64 * max(2 * whole, row, 1))
        (dx,) = _operator("gated_input_grad", taken, [dgu, gate, up],
                          lambda *xs: [_gated_input_grad(*xs, whole)], features=n)
        # tokens in whole k tiles and whole rows: the plan's own dots, which take an update of the weight into their stores
        dots = t % 64 == 0 and n % 8 == 0 and k % 8 == 0
        dgate, dup = _operator("gated_weight_grad", taken and not dots, [dgu, x],
                               lambda *xs: _gated_weight_grad(*xs, n, whole), features=n)
        return dx, dgate, dup

    @staticmethod
    def backward(ctx, *cotangents):
        def grads(dh, x, gate, up):
            g, u = _gated_products(x, gate, up)
            n = gate.shape[0]
            dgu = _gated_elements(dh, g, u, ctx.activation, n)
            return (_gated_input_grad(dgu, gate, up, n), *_gated_weight_grad(dgu, x, n, n))

        return (*_second(grads, ctx.saved_tensors, cotangents), None, None)


def _gated_elements(dh, g, u, activation, whole):
    """``[dg | du]``, each half ``whole`` elements wide (zeros past its features)."""
    (t, n), dtype = dh.shape, dh.dtype
    a, da = _activated_grad(activation, g)
    d = dh.to(g.dtype)
    halves = [(d * u * da).to(dtype), (d * a).to(dtype)]
    if whole != n:
        pad = prims.full((t, whole - n), 0.0, dtype)
        halves = [halves[0], pad, halves[1], pad]
    return F.cat(halves, 1)


def _gated_input_grad(dgu, gate, up, whole):
    n, acc = gate.shape[0], accum_dtype(dgu.dtype)
    dims = (((1,), (0,)), ((), ()))
    return (prims.dot_general(dgu[:, :n], gate, dims, acc)
            + prims.dot_general(dgu[:, whole:whole + n], up, dims, acc)).to(dgu.dtype)


def _gated_weight_grad(dgu, x, n, whole):
    acc = accum_dtype(x.dtype)
    return [dot(dgu[:, lo:lo + n], x, (((0,), (0,)), ((), ())), acc, x.dtype) for lo in (0, whole)]


def gated_linear(input, gate_weight, up_weight, activation="silu"):
    """``act(input @ gate_weight^T) * (input @ up_weight^T)``, the widening half of a gated MLP: ``input`` ``[..., K]``
    and both weights ``[F, K]`` of one float dtype give ``[..., F]`` of it. ``activation`` is ``"silu"``, ``"gelu"`` (the
    tanh form), ``"relu"`` or ``"sigmoid"``. Both products and everything after them are float32 (float64 of float64
    operands), rounded once. The backward holds the two products, float32 ``[..., F]`` each, and rounds their gradients to
    the operands' dtype, as operands of the products that give the gradients of ``input`` and the weights, which are rounded
    again. bfloat16 and float16 run as kernels of their own, other dtypes as their primitives."""
    op = "gated_linear"
    x, gate, up = lift(input), lift(gate_weight), lift(up_weight)
    if activation not in ACTIVATIONS:
        raise ValueError(f"{op}: activation must be one of {', '.join(ACTIVATIONS)}, got {activation!r}")
    if not isinstance(x, TracedTensor) or x.ndim < 1:
        raise ValueError(f"{op}: the input is not a tensor of rows: {x!r}")
    require_float(x, op)
    for role, w in (("gate", gate), ("up", up)):
        if not isinstance(w, TracedTensor) or w.ndim != 2 or w.shape[1] != x.shape[-1]:
            raise ValueError(f"{op}: the {role} weight must be [features, {x.shape[-1]}], got {w!r}")
        if w.dtype != x.dtype:
            raise TypeError(f"{op}: input is {x.dtype} and the {role} weight {w.dtype}: convert them to one with .to(dtype)")
    if gate.shape != up.shape:
        raise ValueError(f"{op}: gate weight {list(gate.shape)} and up weight {list(up.shape)} differ")
    rows = x if x.ndim == 2 else x.reshape(math.prod(x.shape[:-1]), x.shape[-1])
    out = _GatedLinear.apply(rows, gate, up, activation=activation)
    return out if x.ndim == 2 else out.reshape(*x.shape[:-1], gate.shape[0])


# ---- clipping -------------------------------------------------------------------------------------------


class _ClipGradNorm(Function):
    @staticmethod
    def forward(ctx, max_norm, *grads, eps):
        limits = [] if not isinstance(max_norm, TracedTensor) else [max_norm]

        def body(*xs):
            limit, gs = (xs[0], xs[1:]) if limits else (prims.full((), float(max_norm), "float64"), xs)
            total = prims.full((), 0.0, "float64")
            for g in gs:
                v = g.to("float64")
                total = total + F.sum(v * v)
            norm = prims.sqrt(total)
            scale = F.minimum(limit / (norm + eps), prims.full((), 1.0, "float64"))
            out = [norm.to("float32"), scale.to("float32")]
            for g in gs:
                acc = accum_dtype(g.dtype)
                out.append((g.to(acc) * broadcast_to(scale.to(acc), g.shape)).to(g.dtype))
            return out

        taken = all(g.dtype in KERNEL_DTYPES for g in grads)
        return _operator("clip_grad_norm", taken, limits + list(grads), body, eps=float(eps),
                         max_norm=None if limits else float(max_norm))

    @staticmethod
    def backward(ctx, *grads):
        raise NotImplementedError("clip_grad_norm: its results have no gradient (it is applied to gradients)")


def clip_grad_norm(grads, max_norm, eps=1e-6):
    """``(clipped, norm)``: ``norm`` the float32 2-norm over every element of ``grads`` (float tensors of any shapes and
    dtypes) and ``clipped`` the list of them times ``min(1, max_norm / (norm + eps))``, each in its own dtype.

    Squares are summed in float64, in a fixed order. As with any scale, an infinite gradient makes the scale 0 (and
    itself NaN) and a NaN one makes every result NaN. ``max_norm`` is a number or a scalar tensor. The results have no
    gradient."""
    op = "clip_grad_norm"
    if isinstance(grads, TracedTensor) or not isinstance(grads, (list, tuple)):
        raise TypeError(f"{op}: gradients are a list or tuple of tensors, got {grads!r}")
    grads = [lift(g) for g in grads]
    if not grads:
        raise ValueError(f"{op}: no gradients")
    for g in grads:
        if not isinstance(g, TracedTensor):
            raise TypeError(f"{op}: gradients are tensors, got {g!r}")
        require_float(g, op)
    max_norm = lift(max_norm)
    if isinstance(max_norm, TracedTensor):
        if max_norm.shape != () or not D.is_float(max_norm.dtype):
            raise TypeError(f"{op}: max_norm must be a number or a float scalar, got {max_norm!r}")
        max_norm = max_norm.to("float64")
    elif isinstance(max_norm, bool) or not isinstance(max_norm, (int, float)) or not max_norm >= 0:
        raise ValueError(f"{op}: max_norm must be at least 0, got {max_norm!r}")
    if isinstance(eps, bool) or not isinstance(eps, (int, float)) or not eps >= 0:
        raise ValueError(f"{op}: eps must be at least 0, got {eps!r}")
    out = _ClipGradNorm.apply(max_norm, *grads, eps=float(eps))
    return list(out[2:]), out[0]
