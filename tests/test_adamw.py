"""adamw on the CPU: what it computes (the oracle on its traced body against plain float64 NumPy), its refusals, the plan it
becomes, the clipping it takes over, and the optimizer built of it."""

import numpy as np
import pytest

import lumen_amd as L
import lumen_amd.functional as F
from lumen_amd import dtypes as D
from lumen_amd import workloads as W
from lumen_amd.compiler.plan import Plan, compile_graph
from lumen_amd.graph.trace import trace
from oracle import oracle
from tests import training_math as M

BETAS, EPS, DECAY = (0.9, 0.99), 1e-6, 0.05


def _meta(a, dtype=None):
    return L.empty(list(np.shape(a)), dtype or np.asarray(a).dtype.name, "meta")


def _weights(rng, shapes, dtype):
    """``[(w, g, m, v)]``, the moments float32 or float64."""
    state = "float64" if dtype == "float64" else "float32"
    out = []
    for s in shapes:
        w, g, m = (rng.standard_normal(s).astype(t) for t in (dtype, dtype, state))
        out.append((w, g, m, np.abs(rng.standard_normal(s)).astype(state)))
    return out


def _program(masters=False, step=None, lr=None):
    def fn(*xs):
        xs = list(xs)
        t = step if step is not None else xs.pop(0)
        rate = lr if lr is not None else xs.pop(0)
        n = len(xs) // (5 if masters else 4)
        p, g, m, v, w = (xs[i * n:(i + 1) * n] for i in range(5))
        p, m, v, w = F.adamw(p, g, m, v, t, rate, betas=BETAS, eps=EPS, weight_decay=DECAY, masters=w if masters else None)
        return [*p, *m, *v, *(w or [])]

    return fn


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("step", [1, 7, 100000])
def test_values(dtype, step, fused):
    """Several shapes, a 0-d weight and an empty one; ``step`` and ``lr`` given with the call, and known ahead."""
    rng = np.random.default_rng(step)
    ws = _weights(rng, [(5, 3), (), (17,), (0, 4)], dtype)
    flat = [x for part in zip(*ws) for x in part]
    for given in (True, False):
        scalars = [np.array(step, np.int32), np.array(3e-3)] if given else []
        fn = _program() if given else _program(step=step, lr=3e-3)
        with L.config.compiler.patch(fused_operators=fused):
            g = L.make_graph(fn)(*(_meta(x) for x in scalars + flat))
        assert [n.params["name"] for n in g.nodes if n.prim == "fusion"] == (["adamw"] if fused and dtype == "float32" else [])
        got = oracle.values(g, scalars + flat)
        for i, (w, gr, m, v) in enumerate(ws):
            want = M.adamw(w, gr, m, v, step, 3e-3, BETAS, EPS, DECAY)
            tol = M.adamw_tolerances(w, gr, m, v, step, 3e-3, BETAS, EPS, DECAY)
            for part in range(3):
                a = np.asarray(got[4 * part + i], np.float64)
                limit = tol[part] if dtype == "float32" else tol[part] * 2.0**-29 + 1e-300
                assert a.shape == want[part].shape and np.all(np.abs(a - want[part]) <= limit), (i, part)


def test_masters():
    """A bfloat16 weight is its stepped master rounded, whatever the weight itself held."""
    rng = np.random.default_rng(3)
    (w, g, m, v), = _weights(rng, [(6, 5)], "float32")
    bits = D.bf16_bits(g)
    graph = L.make_graph(_program(masters=True, step=2, lr=0.1))(_meta(w, "bfloat16"), _meta(g, "bfloat16"), *(_meta(x) for x in (m, v, w)))
    p1, m1, v1, w1 = oracle.values(graph, [np.zeros(w.shape, np.uint16), bits, m, v, w])
    grad = D.bf16_to_f32(bits)
    want = M.adamw(w, grad, m, v, 2, 0.1, BETAS, EPS, DECAY)
    tol = M.adamw_tolerances(w, grad, m, v, 2, 0.1, BETAS, EPS, DECAY)
    for a, b, t in zip((w1, m1, v1), want, tol):
        assert np.all(np.abs(a - b) <= t)
    assert np.array_equal(p1, D.bf16_to_f32(D.bf16_bits(w1)))


def test_refusals():
    p, half = L.empty([4], "float32", "meta"), L.empty([4], "bfloat16", "meta")
    other, ints = L.empty([5], "float32", "meta"), L.empty([4], "int32", "meta")

    def call(*args, **kw):
        L.make_graph(lambda *xs: F.adamw(*[[xs[i] for i in a] for a in args[0]], *args[1:], **kw)[0])(p, half, other, ints)

    good = [[0], [0], [0], [0]]
    call(good, 1, 0.1)
    call(good, 1, 0.1, betas=[0.0, 0.0], eps=0, weight_decay=0)
    for which, error in [([[], [], [], []], ValueError), ([[0, 0], [0], [0, 0], [0, 0]], ValueError), ([[3], [3], [0], [0]], TypeError),
                         ([[0], [2], [0], [0]], TypeError), ([[0], [1], [0], [0]], TypeError), ([[1], [1], [1], [0]], TypeError)]:
        with pytest.raises(error, match="adamw"):
            call(which, 1, 0.1)
    for kw in (dict(betas=(1.0, 0.9)), dict(betas=(0.9,)), dict(betas=(0.9, -0.1)), dict(betas=(True, 0.9)), dict(eps=-1.0),
               dict(eps=float("nan")), dict(weight_decay=-0.1)):
        with pytest.raises(ValueError, match="adamw"):
            call(good, 1, 0.1, **kw)
    for step, lr in ((0, 0.1), (1, -0.1), (True, 0.1), (1, float("inf")), (None, 0.1)):
        with pytest.raises(ValueError, match="adamw"):
            call(good, step, lr)
    with pytest.raises(TypeError, match="masters are of 16-bit"):
        L.make_graph(lambda p: F.adamw([p], [p], [p], [p], 1, 0.1, masters=[p])[0])(p)
    with pytest.raises(TypeError, match="the master"):
        L.make_graph(lambda p, h: F.adamw([h], [h], [p], [p], 1, 0.1, masters=[h])[0])(p, half)
    with pytest.raises(TypeError, match="scalar"):
        L.make_graph(lambda p: F.adamw([p], [p], [p], [p], p, 0.1)[0])(p)
    with pytest.raises(TypeError, match="list"):
        L.make_graph(lambda p: F.adamw(p, p, p, p, 1, 0.1)[0])(p)
    with pytest.raises(NotImplementedError, match="no gradient"):
        L.make_graph(lambda p, g: L.vjp(lambda p: F.adamw([p], [g], [g], [g], 1, 0.1)[0][0], p)[1](g))(p, p)


def test_clipped_gradients_are_scaled_in_the_step():
    """Gradients of one clipping that only the step (and elementwise readers) read come to it as they were, with the scale: the
    same values; a gradient that is returned too, or of two clippings, is not."""
    rng = np.random.default_rng(5)
    (a, g, m, v), (b, h, _, _) = _weights(rng, [(5, 7), (5, 7)], "float32")

    def fn(returned, twice):
        def step(a, b, g, h, m, v):
            clipped, norm = F.clip_grad_norm([g, h], 1.0)
            if twice:
                clipped[1] = F.clip_grad_norm([h], 0.5)[0][0]
            p, m1, v1, _ = F.adamw([a, b], clipped, [m, m], [v, v], 3, 0.1, betas=BETAS, eps=EPS, weight_decay=DECAY)
            return [*p, *m1, *v1] + ([clipped[0]] if returned else [])

        return step

    args = (a, b, g, h, m, v)
    for returned, twice, scaled in ((False, False, True), (True, False, False), (False, True, False)):
        graph = L.make_graph(fn(returned, twice))(*(_meta(x) for x in args))
        compiled, _ = compile_graph(graph)
        assert [n.params["scaled"] for n in compiled.nodes if n.params.get("name") == "adamw"] == [scaled]
        for x, y in zip(oracle.values(graph, list(args)), oracle.values(compiled, list(args))):
            assert np.array_equal(x, y)


def test_the_optimizer_is_one_step_over_its_weights():
    """The 2-layer model's training step with AdamW: one adamw step, every weight, moment and master computed in place."""
    model, _ = W.build(W.TINY)
    opt = W.adamw(model, lr=1e-3)

    def train_step(model, opt, ids, targets):
        loss = W.loss_fn(model, ids, targets)
        loss.backward()
        opt.step(max_norm=1.0)
        return loss

    ids = L.empty([2, 128], "int64", "meta")
    traced = trace(train_step, (model, opt, ids, ids))
    at = {k: i for i, (kind, k) in enumerate(traced.layout) if kind == "weight"}
    donate = {traced.n_returned + j: at[k] for j, k in enumerate(traced.written)}
    plan = Plan(traced.graph, build_kernels=False, donate=donate)
    kinds = [st.kind for st in plan.steps]
    assert kinds.count("adamw") == 1 and kinds.count("clip") == 1
    # the scalar count is not, or is, by its own loop; everything else is
    assert len(donate) == 4 * len(opt.params) + 1
    assert len(plan.in_place_outputs) >= 4 * len(opt.params)


def test_a_result_over_an_operand_that_another_weight_reads_is_not_in_place():
    """Moments of one weight that another weight's step reads too: written apart, since the other may read them later."""
    class Two(L.nn.Module):
        a: L.Tensor
        b: L.Tensor
        m: L.Tensor
        v: L.Tensor

    state = Two(*(L.empty([8], "float32", "meta") for _ in range(4)))

    def step(s, g):
        p, m, v, _ = F.adamw([s.a, s.b], [g, g], [s.m, s.m], [s.v, s.v], 1, 0.1)
        for x, new in zip((s.a, s.b, s.m, s.v), (p[0], p[1], m[0], v[1])):
            x.copy_(new)
        return g * 2.0

    traced = trace(step, (state, L.empty([8], "float32", "meta")))
    at = {k: i for i, (kind, k) in enumerate(traced.layout) if kind == "weight"}
    donate = {traced.n_returned + j: at[k] for j, k in enumerate(traced.written)}
    plan = Plan(traced.graph, build_kernels=False, donate=donate)
    assert sorted(plan.in_place_outputs) == [1, 2]  # the weights
