"""The cross entropy of a vocabulary head over its input and weight (``linear_cross_entropy``), beside ``cross_entropy`` over
logits: neither direction ever holds the logits whole."""

from __future__ import annotations

import math

from lumen_amd.autograd.function import Function
from lumen_amd.functional import functions as F
from lumen_amd.functional.cross_entropy import one_hot
from lumen_amd.functional.operators import _operator, _second
from lumen_amd.graph import prims
from lumen_amd.graph.tracer import TracedTensor, accum_dtype, broadcast_to, dot, lift, require_float

_ROWS = (((1,), (1,)), ((), ()))  # [T, K] and [V, K] to [T, V]
REDUCTIONS = ("mean", "sum", "none")


def _logits(h, w):
    acc = accum_dtype(h.dtype)
    return dot(h, w, _ROWS, acc, acc)


def _targets(target, classes, ignore):
    """Each row's class, clamped into the classes, and whether it counts."""
    kept = ~prims.eq(target, prims.full(target.shape, ignore, target.dtype))
    last = prims.full(target.shape, classes - 1, target.dtype)
    zero = prims.full(target.shape, 0, target.dtype)
    cls = F.where(prims.lt(target, zero), zero, F.where(prims.lt(last, target), last, target))
    return cls, kept


def _masked(x, kept):
    return F.where(kept, x, prims.full(x.shape, 0.0, x.dtype))


def _losses(logits, target, ignore):
    """``(losses, lse)``, a value a row."""
    t, v = logits.shape
    cls, kept = _targets(target, v, ignore)
    m = F.amax(logits, -1, keepdim=True)
    lse = m.reshape(t) + F.log(F.sum(F.exp(logits - broadcast_to(m, logits.shape)), -1))
    at = prims.iota("int64", (t,), 0) * v + cls.to("int64")
    picked = prims.gather(logits.reshape(t * v), at, 0)
    return _masked(lse - picked, kept), lse


def _gradients(h, w, target, g, ignore, p=None):
    """``[dh, dw, losses]`` for the losses' cotangents ``g``; ``p``: the probabilities, by default of the logits again."""
    t, v = h.shape[0], w.shape[0]
    acc = accum_dtype(h.dtype)
    logits = _logits(h, w)
    losses, lse = _losses(logits, target, ignore)
    if p is None:
        p = F.exp(logits - broadcast_to(lse.reshape(t, 1), logits.shape))
    cls, kept = _targets(target, v, ignore)
    d = (p - one_hot(cls, v, acc)) * broadcast_to(_masked(g, kept).reshape(t, 1), logits.shape)
    # a row that is ignored counts for nothing whatever its logits are
    d = F.where(broadcast_to(kept.reshape(t, 1), d.shape), d, prims.full(d.shape, 0.0, acc)).to(h.dtype)
    return [dot(d, w, (((1,), (0,)), ((), ())), acc, h.dtype), dot(d, h, (((0,), (0,)), ((), ())), acc, w.dtype), losses]


def _taken(h, w):
    (t, k), v = h.shape, w.shape[0]
    kp, vp = -(-k // 64) * 64, -(-v // 64) * 64  # whole k tiles, and whole blocks of classes as their exponentials are kept

    def launch(m, n):
        return -(-m // 128) * -(-n // 128) < 1 << 24

    return h.dtype in ("bfloat16", "float16") and 0 < kp < 1 << 20 and 0 < vp < 1 << 22 and (v + 256) * kp < (1 << 30) - 1024 \
        and t < 1 << 26 and launch(t, v) and launch(v, k) and launch(t, k)


class _HeadLoss(Function):
    """A loss a row; the gradients' fusion computes the losses again with what it needs of them, and takes this one's place
    where its cotangents do not depend on them (``compiler/operators.py``)."""

    @staticmethod
    def forward(ctx, h, w, target, *, ignore):
        ctx.ignore = ignore
        ctx.save_for_backward(h, w, target)
        (losses,) = _operator("head_loss", _taken(h, w), [h, w, target],
                              lambda h, w, target: [_losses(_logits(h, w), target, ignore)[0]], ignore=ignore)
        return losses

    @staticmethod
    def backward(ctx, g):
        return (*_HeadGradients.apply(g, *ctx.saved_tensors, ignore=ctx.ignore)[:2], None)


class _HeadGradients(Function):
    @staticmethod
    def forward(ctx, g, h, w, target, *, ignore):
        ctx.ignore = ignore
        ctx.save_for_backward(g, h, w, target)
        return _operator("head_loss_backward", _taken(h, w), [h, w, target, g],
                         lambda h, w, target, g: _gradients(h, w, target, g, ignore), ignore=ignore)

    @staticmethod
    def backward(ctx, *cotangents):
        g, h, w, target = ctx.saved_tensors

        def grads(g, h, w):
            return tuple(_gradients(h, w, target, g, ctx.ignore, p=F.softmax(_logits(h, w), -1))[:2])

        return (*_second(grads, (g, h, w), cotangents[:2]), None)


def linear_cross_entropy(input, weight, target, ignore_index=-100, reduction="mean"):
    """``cross_entropy(input @ weight^T, target)`` of a vocabulary head, whose logits never exist whole: ``input`` ``[..., K]``
    and ``weight`` ``[V, K]`` of one float dtype, ``target`` int32 or int64 ``[...]``.

    A row whose target is ``ignore_index`` (a prompt's, padding's) has no loss and no gradient; other targets are clamped into
    the ``V`` classes. ``reduction``: ``"mean"`` over the rows that count (0 of none), ``"sum"``, or ``"none"``, a loss a row
    ``[...]``. Losses and all sums are float32 (float64 of float64 operands). The gradients of the logits are rounded to the
    operands' dtype as operands of the products that give those of ``input`` and ``weight``, which are rounded again. bfloat16
    and float16 (up to 2^26 rows and 2^38 logits, and a weight below 2^30 elements and 2^22 classes) run as kernels of their own,
    which take six products' work for both directions and hold exponentials (the losses alone: maxima and sums of 64 classes each)
    of at most ``config.compiler.head_piece_bytes`` at a time; others run as primitives, over whole logits where there are
    gradients."""
    op = "linear_cross_entropy"
    h, w, target = lift(input), lift(weight), lift(target)
    if not isinstance(h, TracedTensor) or h.ndim < 1:
        raise ValueError(f"{op}: the input is not a tensor of rows: {h!r}")
    require_float(h, op)
    if not isinstance(w, TracedTensor) or w.ndim != 2 or w.shape[1] != h.shape[-1] or not w.shape[0] or not w.shape[1]:
        raise ValueError(f"{op}: the weight must be [classes, {h.shape[-1]}], neither 0, got {w!r}")
    if w.dtype != h.dtype:
        raise TypeError(f"{op}: input is {h.dtype} and weight {w.dtype}: convert them to one with .to(dtype)")
    if not isinstance(target, TracedTensor) or target.dtype not in ("int32", "int64") or target.shape != h.shape[:-1]:
        raise ValueError(f"{op}: the target must be int32 or int64 {list(h.shape[:-1])}, got {target!r}")
    if isinstance(ignore_index, bool) or not isinstance(ignore_index, int):
        raise ValueError(f"{op}: ignore_index must be an integer, got {ignore_index!r}")
    bits = 32 if target.dtype == "int32" else 64
    if not -(1 << (bits - 1)) <= ignore_index < 1 << (bits - 1):
        raise ValueError(f"{op}: ignore_index {ignore_index} is no {target.dtype}")
    if reduction not in REDUCTIONS:
        raise ValueError(f"{op}: reduction must be one of {', '.join(REDUCTIONS)}, got {reduction!r}")
    lead = h.shape[:-1]
    rows = math.prod(lead)
    flat = target.reshape(rows)
    losses = _HeadLoss.apply(h.reshape(rows, h.shape[-1]), w, flat, ignore=ignore_index)
    if reduction == "none":
        return losses.reshape(*lead)
    total = F.sum(losses)
    if reduction == "sum":
        return total
    kept = prims.eq(flat, prims.full(flat.shape, ignore_index, flat.dtype))
    one = prims.full(flat.shape, 1.0, losses.dtype)
    count = F.sum(F.where(kept, prims.full(flat.shape, 0.0, losses.dtype), one))
    return total / F.maximum(count, prims.full((), 1.0, losses.dtype))
