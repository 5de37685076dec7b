"""The transformer's training step on packed documents (packed attention, the head's cross entropy, a clipped AdamW step) by the
oracle, on the CPU, against the same model on each document alone."""

import numpy as np
import pytest

import lumen_amd as L
import lumen_amd.functional as F
from lumen_amd import dtypes as D
from lumen_amd import workloads as W
from lumen_amd.compiler.plan import Plan
from lumen_amd.graph.trace import trace
from oracle import oracle

CFG = W.TransformerConfig(vocab=97, dim=32, heads=2, ffn=48, seq=24, batch=1, layers=2)


def documents(rng, lengths, vocab):
    return [rng.integers(0, vocab, n) for n in lengths]


def values(fn, args, arrays, weights, names):
    traced = trace(fn, args)
    ins = [arrays[k] if kind == "arg" else weights[names[id(traced.weights[k])]] for kind, k in traced.layout]
    return [np.asarray(a, np.float64) for a in oracle.values(traced.graph, ins)]


def _model(cfg):
    model, _ = W.build(cfg)
    weights = W.init_weights(model)
    W.load(model, weights)
    return model, weights, {id(p): n for n, p in model.named_parameters()}


def test_pack():
    ids, places, targets, offsets = W.pack([np.array([5, 6, 7]), np.array([], int), np.array([8]), np.array([9, 3])], 8)
    assert ids.tolist() == [5, 6, 7, 8, 9, 3, 0, 0] and places.tolist() == [0, 1, 2, 0, 0, 1, 0, 0]
    assert targets.tolist() == [6, 7, -100, -100, 3, -100, -100, -100]
    assert offsets.tolist() == [0, 3, 3, 4, 6] and offsets.dtype == np.int32
    with pytest.raises(ValueError, match="7 tokens in 6"):
        W.pack([np.arange(7)], 6)


def test_packed_documents_are_trained_on_as_each_alone():
    """The mean loss, and each gradient, of packed documents are the sums over the documents alone, weighted by their counted
    tokens. Both round every activation and gradient to bfloat16 at the same places; what differs is the sums' order, the place of
    the roundings of a gradient that is summed over documents, and a mean's 1 / t: each bfloat16 product of a chain of some 40
    roundings of 2^-9 is off by sqrt(40) 2^-9 = 1.2e-2 of its size at most in the mean square, and so is a gradient."""
    rng = np.random.default_rng(0)
    model, weights, names = _model(CFG)
    docs = documents(rng, [24, 1, 7, 13, 2], CFG.vocab)
    params = list(model.parameters())

    def packed(model, ids, places, targets, offsets):
        loss = W.packed_loss(model, ids, places, targets, offsets)
        loss.backward()
        return [loss, *(p.grad for p in params)]

    arrays = W.pack(docs, 50)
    got = values(packed, (model, *map(L.from_numpy, arrays)), arrays, weights, names)
    want, count = None, 0
    for doc in docs:
        if len(doc) < 2:
            continue
        one = W.pack([doc], len(doc))
        out = values(packed, (model, *map(L.from_numpy, one)), one, weights, names)
        n, count = len(doc) - 1, count + len(doc) - 1
        want = [n * a for a in out] if want is None else [a + n * b for a, b in zip(want, out)]
    for a, b in zip(got, want):
        b = b / count
        assert np.linalg.norm(a - b) <= 1.2e-2 * np.linalg.norm(b)


def test_the_plan_runs_the_operators():
    """Forward and backward of the attentions, one step for the head's loss and gradients, and one for all weights, whose
    gradients the clip only measures."""
    cfg = W.TransformerConfig(vocab=256, dim=128, heads=2, ffn=256, seq=128, batch=1, layers=2)
    model, _ = W.build(cfg)
    opt = W.adamw(model)
    metas = [L.empty([200], "int64", "meta") for _ in range(3)] + [L.empty([6], "int32", "meta")]
    traced = trace(W.packed_train_step, (model, opt, *metas))
    kinds = [s.kind for s in Plan(traced.graph, build_kernels=False).steps]
    assert [kinds.count(k) for k in ("packed_fwd", "packed_bwd", "head_loss", "adamw", "clip")] == [2, 2, 1, 1, 1]


def _places(program, *metas):
    """The places of each operator step's pointers, by the step's kind."""
    from lumen_amd.compiler import operators

    plan = Plan(L.make_graph(program)(*metas), build_kernels=False)
    return {st.kind: operators.lower(plan, st)[2] for st in plan.steps if st.kind in operators.STEPS}


def test_a_view_off_16_bytes_that_an_adamw_step_reads_too():
    """One value read where it lies (any contiguous place) by one step and from 16 bytes on by another has both."""
    t = 40
    base, state = L.empty([4 + t * 64], "bfloat16", "meta"), L.empty([t, 1, 64], "float32", "meta")
    offsets, target, w = L.empty([3], "int32", "meta"), L.empty([t], "int32", "meta"), L.empty([100, 64], "bfloat16", "meta")

    def attention(base, m, v, offsets):
        x = base[4:4 + t * 64].reshape(t, 1, 64)
        return [F.packed_attention(x, x, x, offsets), F.adamw([x], [x], [m], [v], 1, 0.1)[0][0]]

    def loss(base, m, v, target, w):
        x = base[4:4 + t * 64].reshape(t, 64)
        m, v = m.reshape(t, 64), v.reshape(t, 64)
        return [F.linear_cross_entropy(x, w, target), F.adamw([x], [x], [m], [v], 1, 0.1)[0][0]]

    for places, kind, slots in ((_places(attention, base, state, state, offsets), "packed_fwd", (0, 1, 2)),
                                (_places(loss, base, state, state, target, w), "head_loss", (0,))):
        at = dict(places[kind])
        assert all(at[s].offset * 2 % 16 == 0 for s in slots)
        assert all(loc.contiguous() for _, loc in places["adamw"])
