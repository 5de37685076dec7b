"""Self attention of sequences packed one after another (``packed_attention``), beside ``flash_attention``, whose batches are
of one length: the reference has no counterpart."""

from __future__ import annotations

import ctypes as C
import math

from lumen_amd.autograd.function import Function
from lumen_amd.functional import functions as F
from lumen_amd.functional.operators import _operator, _second
from lumen_amd.graph import prims
from lumen_amd.graph.tracer import TracedTensor, accum_dtype, broadcast_to, common_dtype, dot, lift, require_float

MAX_TOKENS, MAX_SEQUENCES = 1 << 26, 1 << 20
_QK = (((2,), (2,)), ((1,), (1,)))  # [T, N, D] and [T, N, D] to [N, T, T]


def _sequences(offsets, tokens):
    """Of each token ``[T]`` how many offsets are up to it (0 before the first sequence, all of them behind the last), and
    whether it is of a sequence."""
    count = offsets.shape[0]
    token = prims.iota("int64", (count, tokens), 1)
    ahead = prims.lt(token, broadcast_to(offsets.to("int64").reshape(count, 1), (count, tokens)))
    of = F.sum(F.where(ahead, prims.full(ahead.shape, 0, "int64"), prims.full(ahead.shape, 1, "int64")), 0)
    inside = prims.lt(prims.full((tokens,), 0, "int64"), of) & prims.lt(of, prims.full((tokens,), count, "int64"))
    return of, inside


def _seen(of, inside, causal):
    """Whether token ``i`` attends to token ``j``, ``[T, T]``."""
    t = of.shape[0]
    seen = prims.eq(broadcast_to(of.reshape(t, 1), (t, t)), broadcast_to(of.reshape(1, t), (t, t)))
    seen = seen & broadcast_to(inside.reshape(t, 1), (t, t))
    if causal:
        seen = seen & ~prims.lt(prims.iota("int64", (t, t), 0), prims.iota("int64", (t, t), 1))
    return seen


def _inside(inside, *xs):
    """Each ``[T, N, D]`` with zeros for the tokens of no sequence, whatever they hold."""
    return [F.where(broadcast_to(inside.reshape(x.shape[0], 1, 1), x.shape), x, prims.full(x.shape, 0.0, x.dtype)) for x in xs]


def _heads(x, n):
    """``x`` ``[T, Nkv, D]`` with each head repeated for its ``n / Nkv`` query heads."""
    t, nkv, d = x.shape
    return x if nkv == n else x.unsqueeze(2).expand(t, nkv, n // nkv, d).reshape(t, n, d)


def _kept(x, mask, other=0.0):
    """``x`` ``[N, T, T]`` where ``mask`` ``[T, T]``."""
    return F.where(broadcast_to(mask, x.shape), x, prims.full(x.shape, other, x.dtype))


def _forward(q, k, v, offsets, scale, causal):
    """``(o, rest, lse)``: what the rounding of ``o`` left, in its dtype, and the scores' log-sum-exp ``[N, T]``, 0 of a token of no
    sequence."""
    t, n = q.shape[:2]
    acc = accum_dtype(q.dtype)
    of, inside = _sequences(offsets, t)
    seen = _seen(of, inside, causal)
    q, k, v = _inside(inside, q, k, v)
    s = _kept(prims.dot_general(q, _heads(k, n), _QK, acc) * scale, seen, -math.inf)
    top = F.amax(s, -1, keepdim=True)
    empty = prims.eq(top, prims.full(top.shape, -math.inf, acc))
    top = F.where(empty, prims.full(top.shape, 0.0, acc), top)
    e = F.exp(s - broadcast_to(top, s.shape))
    total = F.sum(e, -1, keepdim=True)
    total = F.where(empty, prims.full(top.shape, 1.0, acc), total)
    p = (e / broadcast_to(total, s.shape)).to(q.dtype)
    whole = dot(p, _heads(v, n), (((2,), (0,)), ((0,), (1,))), acc, acc).permute(1, 0, 2)
    o = whole.to(q.dtype)
    rest = (whole - o.to(acc)).to(q.dtype)
    return *_inside(inside, o, rest), (top + F.log(total)).reshape(n, t)


def _gradients(q, k, v, offsets, o, rest, lse, do, scale, causal):
    """``[dq, dk, dv]``: probabilities again from the log-sum-exp, ``dS = P (dO V^T - rowsum(dO (O + rest)))``."""
    t, n = q.shape[:2]
    nkv = k.shape[1]
    dtype, acc = q.dtype, accum_dtype(q.dtype)
    of, inside = _sequences(offsets, t)
    seen = _seen(of, inside, causal)
    q, k, v, o, rest, do = _inside(inside, q, k, v, o, rest, do)
    k_full, v_full = _heads(k, n), _heads(v, n)
    s = prims.dot_general(q, k_full, _QK, acc) * scale
    p = _kept(F.exp(_kept(s - broadcast_to(lse.reshape(n, t, 1), s.shape), seen)), seen)
    delta = F.sum(do.to(acc) * (o.to(acc) + rest.to(acc)), -1).permute(1, 0).reshape(n, t, 1)
    dp = prims.dot_general(do, v_full, _QK, acc)
    ds = _kept(p * (dp - broadcast_to(delta, dp.shape)) * scale, seen).to(dtype)
    p = p.to(dtype)
    dq = prims.dot_general(ds, k_full, (((2,), (0,)), ((0,), (1,))), acc)
    dk = prims.dot_general(ds, q, (((1,), (0,)), ((0,), (1,))), acc)
    dv = prims.dot_general(p, do, (((1,), (0,)), ((0,), (1,))), acc)
    dq, dk, dv = (x.permute(1, 0, 2) for x in (dq, dk, dv))
    if nkv != n:
        dk, dv = (F.sum(x.reshape(t, nkv, n // nkv, x.shape[2]), 2) for x in (dk, dv))
    return _inside(inside, *(x.to(dtype) for x in (dq, dk, dv)))


def _taken(q, k, v, offsets, scale):
    (t, n, d), (nkv, dv) = q.shape, v.shape[1:]
    most = max(t // 64 + min(offsets.shape[0] - 1, t) + 2, t // 8 + 1)
    # the kernels' scale is float32: one that it rounds to 0 or to infinity is the primitives'
    return q.dtype in ("bfloat16", "float16") and 0.0 < C.c_float(scale).value <= 3.4e38 \
        and all(x % 8 == 0 and 0 < x <= 128 for x in (d, dv)) and t <= MAX_TOKENS and offsets.shape[0] - 1 <= MAX_SEQUENCES \
        and most * max(n, nkv) < 1 << 24


class _PackedAttention(Function):
    @staticmethod
    def forward(ctx, q, k, v, offsets, *, scale, causal):
        o, rest, lse = _operator("packed_attention", _taken(q, k, v, offsets, scale), [q, k, v, offsets],
                                 lambda *xs: _forward(*xs, scale, causal), scale=scale, causal=causal)
        ctx.scale, ctx.causal = scale, causal
        ctx.save_for_backward(q, k, v, offsets, o, rest, lse)
        return o

    @staticmethod
    def backward(ctx, do):
        return (*_PackedGradients.apply(do, *ctx.saved_tensors, scale=ctx.scale, causal=ctx.causal), None)


class _PackedGradients(Function):
    @staticmethod
    def forward(ctx, do, q, k, v, offsets, o, rest, lse, *, scale, causal):
        ctx.scale, ctx.causal = scale, causal
        ctx.save_for_backward(do, q, k, v, offsets)
        return _operator("packed_attention_backward", _taken(q, k, v, offsets, scale), [q, k, v, offsets, o, rest, do, lse],
                         lambda q, k, v, offsets, o, rest, do, lse: _gradients(q, k, v, offsets, o, rest, lse, do, scale, causal),
                         scale=scale, causal=causal)

    @staticmethod
    def backward(ctx, *cotangents):
        do, q, k, v, offsets = ctx.saved_tensors

        def grads(do, q, k, v):
            o, rest, lse = _forward(q, k, v, offsets, ctx.scale, ctx.causal)
            return tuple(_gradients(q, k, v, offsets, o, rest, lse, do, ctx.scale, ctx.causal))

        return (*_second(grads, (do, q, k, v), cotangents), None, None, None, None)


def packed_attention(query, key, value, offsets, scale=None, is_causal=True):
    """``softmax(query @ key^T * scale) @ value`` of every head within each of the sequences that lie one after another in
    ``query`` ``[T, N, D]``, ``key`` ``[T, Nkv, D]`` and ``value`` ``[T, Nkv, Dv]``: ``[T, N, Dv]``.

    ``offsets`` (int32 or int64 ``[sequences + 1]``, not decreasing, within ``0`` to ``T``) are the sequences' first tokens and
    the last one's end: token ``t`` is of sequence ``i`` where ``offsets[i] <= t < offsets[i + 1]``, and attends to that
    sequence's tokens, up to itself if ``is_causal``. Sequences may be empty. Tokens of no sequence, before the first offset or
    from the last one on, give zeros and have zero gradients, and nothing that they hold, not even a NaN, reaches a
    sequence's results; the kernels keep one of another sequence out too. ``N`` is a multiple of ``Nkv`` (grouped heads);
    ``scale`` is ``1 / sqrt(D)`` by default. The softmax and all sums are float32 (float64 of float64 operands), the
    probabilities rounded to the operands' dtype. bfloat16 and float16 with head dims that are multiples of 8 up to 128
    (and up to 2^26 tokens and 2^20 sequences, ``N T / 8`` and ``N (T / 64 + sequences)`` below 2^24, and a scale that float32
    holds) run as kernels of their own, others as primitives, whose scores ``[N, T, T]`` exist whole. The kernels of head dims
    other than 64 and 128 need the rows of each head of an operand within 2 GiB."""
    op = "packed_attention"
    q, k, v, offsets = lift(query), lift(key), lift(value), lift(offsets)
    for role, t in (("query", q), ("key", k), ("value", v)):
        if not isinstance(t, TracedTensor) or t.ndim != 3:
            raise ValueError(f"{op}: the {role} is not a 3-D [tokens, heads, head_dim] tensor: {t!r}")
    require_float(q, op)
    common_dtype(op, (q, k, v))
    problems = []
    if not q.shape[0] == k.shape[0] == v.shape[0]:
        problems.append("token counts differ")
    if k.shape[1] != v.shape[1]:
        problems.append("key and value head counts differ")
    if q.shape[2] != k.shape[2]:
        problems.append("query and key head dims differ")
    if k.shape[1] == 0 or q.shape[1] % k.shape[1]:
        problems.append("query heads are not a multiple of key/value heads")
    if 0 in (q.shape[2], v.shape[2]):
        problems.append("heads have no elements")
    if problems:
        raise ValueError(f"{op}: query {list(q.shape)}, key {list(k.shape)}, value {list(v.shape)}: " + "; ".join(problems))
    if not isinstance(offsets, TracedTensor) or offsets.ndim != 1 or offsets.dtype not in ("int32", "int64") or not offsets.shape[0]:
        raise ValueError(f"{op}: offsets must be int32 or int64 [sequences + 1], got {offsets!r}")
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[2])
    if isinstance(scale, bool) or not isinstance(scale, (int, float)) or not 0 < scale < math.inf:
        raise ValueError(f"{op}: scale must be a positive number known when the function is compiled, got {scale!r}")
    if not isinstance(is_causal, bool):
        raise ValueError(f"{op}: is_causal must be True or False, got {is_causal!r}")
    return _PackedAttention.apply(q, k, v, offsets, scale=float(scale), causal=is_causal)
