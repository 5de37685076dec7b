"""linear_cross_entropy on the CPU: what it computes (the oracle on its traced body against plain float64 NumPy), its gradients
against differences, its refusals, and the plan it becomes."""

import ctypes as C

import numpy as np
import pytest

import lumen_amd as L
import lumen_amd.functional as F
from lumen_amd import native as nv
from lumen_amd.compiler.plan import Plan, compile_graph
from lumen_amd.graph import prims
from oracle import oracle
from tests import training_math as M


def _meta(a, dtype=None):
    return L.empty(list(np.shape(a)), dtype or np.asarray(a).dtype.name, "meta")


def _program(reduction, ignore=-100):
    def fn(h, w, target, g):
        loss, pull = L.vjp(lambda h, w: F.linear_cross_entropy(h, w, target, ignore, reduction), h, w)
        return [loss, *pull(g)]

    return fn


def _case(rng, lead, k, v, dtype="float64"):
    h, w = rng.standard_normal((*lead, k)).astype(dtype), rng.standard_normal((v, k)).astype(dtype)
    target = rng.integers(0, v, lead)
    return h, w, np.where(rng.random(lead) < 0.3, -100, target)


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("reduction", F.linear_cross_entropy.__globals__["REDUCTIONS"])
@pytest.mark.parametrize("lead,k,v,target_type", [((9,), 5, 11, "int64"), ((2, 3), 4, 7, "int32"), ((1,), 1, 1, "int64"), ((), 3, 4, "int32")])
def test_values_and_gradients(dtype, reduction, lead, k, v, target_type):
    rng = np.random.default_rng(k + v)
    h, w, target = _case(rng, lead, k, v, dtype)
    target = target.astype(target_type)
    rows, n = int(np.prod(lead)), int((target != -100).sum())
    given = np.asarray(rng.standard_normal(lead if reduction == "none" else ())).astype(dtype)
    g = L.make_graph(_program(reduction))(*(_meta(a) for a in (h, w, target, given)))
    assert not [x for x in g.nodes if x.prim == "fusion"]
    got = oracle.values(g, [h, w, target, given])
    each = given.reshape(rows) if reduction == "none" else np.full(rows, given / (max(n, 1) if reduction == "mean" else 1))
    flat = (h.reshape(rows, k), w, target.reshape(rows), -100, each)
    losses, dh, dw = M.linear_cross_entropy(*flat)
    tl, th, tw = M.linear_cross_entropy_tolerances(*flat, "float32")
    loss, tol = {"none": (losses.reshape(lead), tl.reshape(lead)), "sum": (losses.sum(), tl.sum() + 1e-6 * losses.sum()),
                 "mean": (losses.sum() / max(n, 1), tl.sum() + 1e-6 * losses.sum())}[reduction]
    for a, b, t in zip(got, (loss, dh.reshape(h.shape), dw), (tol, th.reshape(h.shape), tw)):
        assert np.shape(a) == np.shape(b) and np.all(np.abs(a - b) <= (t if dtype == "float32" else t * 2.0**-13 + 1e-14))


def test_gradient_against_differences():
    rng = np.random.default_rng(1)
    h, w, target = _case(rng, (4,), 3, 5)
    x, g = {"h": h, "w": w}, rng.standard_normal(4)
    _, dh, dw = M.linear_cross_entropy(h, w, target, -100, g)
    from tests.operator_math import differences

    for name, grad in (("h", dh), ("w", dw)):
        diff = differences(lambda x: (M.linear_cross_entropy(x["h"], x["w"], target, -100, g)[0] * g).sum(), x, name)
        assert np.abs(diff - grad).max() <= 1e-7


def test_a_gradient_differentiated_again():
    """The float64 derivative of dh along a direction against differences of dh."""
    rng = np.random.default_rng(2)
    h, w, target = _case(rng, (4,), 3, 5)
    u, g = rng.standard_normal(h.shape), rng.standard_normal(4)

    def fn(h, w, target, g, u):
        def along(h):
            _, pull = L.vjp(lambda h: F.linear_cross_entropy(h, w, target, reduction="none"), h)
            return F.sum(pull(g)[0] * u)

        return [L.grad(along)(h)]

    args = [h, w, target, g, u]
    (got,) = oracle.values(L.make_graph(fn)(*(_meta(a) for a in args)), args)
    want = [M.linear_cross_entropy(h + s * 1e-5 * u, w, target, -100, g)[1] for s in (1, -1)]
    assert np.abs(got - (want[0] - want[1]) / 2e-5).max() <= 1e-7


def test_targets_outside_and_another_ignored_value():
    rng = np.random.default_rng(3)
    h, w, _ = _case(rng, (4,), 3, 5)
    target = np.array([2, -1, 7, 3])
    g = L.make_graph(lambda h, w, t: [F.linear_cross_entropy(h, w, t, ignore_index=2, reduction="none")])(*(_meta(a) for a in (h, w, target)))
    (got,) = oracle.values(g, [h, w, target])
    want = M.linear_cross_entropy(h, w, np.array([9, 0, 4, 3]), 9, np.ones(4))[0]
    assert np.abs(got - want).max() <= 1e-12


def test_refusals():
    h, w, t = L.empty([6, 8], "float32", "meta"), L.empty([10, 8], "float32", "meta"), L.empty([6], "int64", "meta")

    def call(h=h, w=w, t=t, **kw):
        L.make_graph(lambda *xs: F.linear_cross_entropy(*xs, **kw))(h, w, t)

    def shaped(*s, dtype="float32"):
        return L.empty(list(s), dtype, "meta")

    call()
    for kw in (dict(w=shaped(10, 7)), dict(w=shaped(80)), dict(w=shaped(0, 8)), dict(h=shaped(6, 0), w=shaped(10, 0)), dict(t=shaped(5, dtype="int64")),
               dict(t=shaped(6)), dict(t=shaped(6, 1, dtype="int64")), dict(reduction="max"), dict(reduction=None), dict(ignore_index=1.0),
               dict(ignore_index=True), dict(ignore_index=1 << 40, t=shaped(6, dtype="int32"))):
        with pytest.raises(ValueError, match="linear_cross_entropy"):
            call(**kw)
    with pytest.raises(TypeError):
        call(w=shaped(10, 8, dtype="bfloat16"))
    with pytest.raises(TypeError):
        call(h=shaped(6, 8, dtype="int32"), w=shaped(10, 8, dtype="int32"))


def _graph(fn, t=300, k=128, v=777, dtype="bfloat16", g=("float32", None)):
    metas = [L.empty([t, k], dtype, "meta"), L.empty([v, k], dtype, "meta"), L.empty([t], "int32", "meta")]
    return L.make_graph(fn)(*metas, *([L.empty([t] if g[1] is None else [], g[0], "meta")] if g else []))


def test_plans():
    """One step for both directions; two where the cotangent depends on the loss; the losses' own where there are no gradients."""
    def kinds(graph):
        return [st.nodes[0].params["name"] for st in Plan(graph, build_kernels=False).steps if st.kind == "head_loss"]

    assert kinds(_graph(_program("none"))) == ["head_loss_backward"]
    assert kinds(_graph(_program("mean"), g=("float32", 0))) == ["head_loss_backward"]

    def forward(h, w, t):
        return [F.linear_cross_entropy(h, w, t, reduction="none")]

    assert kinds(_graph(forward, g=None)) == ["head_loss"]

    def dependent(h, w, t):
        loss, pull = L.vjp(lambda h, w: F.linear_cross_entropy(h, w, t), h, w)
        return [loss, *pull(loss * 2.0)]

    assert kinds(_graph(dependent, g=None)) == ["head_loss", "head_loss_backward"]

    def two(h, w, t):  # two losses of other ignored values, each with its gradients
        a, pa = L.vjp(lambda h, w: F.linear_cross_entropy(h, w, t, 1), h, w)
        b, pb = L.vjp(lambda h, w: F.linear_cross_entropy(h, w, t, 2), h, w)
        return [a, b, *pa(a * 0.0 + 1.0), *pb(a)]

    assert kinds(_graph(two, g=None)) == ["head_loss", "head_loss_backward", "head_loss_backward"]

    def crossed(h, w, t):  # the cotangent of each is the other's loss: one of them comes first
        a, pa = L.vjp(lambda h, w: F.linear_cross_entropy(h, w, t, 1), h, w)
        b, pb = L.vjp(lambda h, w: F.linear_cross_entropy(h, w, t, 2), h, w)
        return [a, b, *pa(b), *pb(a)]

    assert kinds(_graph(crossed, g=None)) == ["head_loss", "head_loss_backward", "head_loss_backward"]

    def chained(h, w, t):  # the second's cotangent depends on the first's loss alone
        a, pa = L.vjp(lambda h, w: F.linear_cross_entropy(h, w, t, 1), h, w)
        b, pb = L.vjp(lambda h, w: F.linear_cross_entropy(h, w, t, 2), h, w)
        return [a * b, *pb(a), *pa(prims.full((), 1.0, "float32"))]

    assert kinds(_graph(chained, g=None)) == ["head_loss_backward"] * 2
    for dtype in ("float32", "float64"):
        assert not kinds(_graph(_program("none"), dtype=dtype, g=(dtype, None)))
    with L.config.compiler.patch(fused_operators=False):
        assert not [n for n in _graph(_program("none")).nodes if n.prim == "fusion"]
    assert not [n for n in _graph(_program("none"), k=1 << 12, v=1 << 18).nodes if n.prim == "fusion"]  # a weight of 2^31 bytes


def test_the_joined_step_keeps_its_values():
    """The graph with one step gives what the one with two gives, evaluated as primitives; values that depend on the loss, and on
    both, come after it."""
    rng = np.random.default_rng(4)
    h, w, target = _case(rng, (9,), 64, 11, "float32")
    bits = [np.asarray(a, np.float32) for a in (h, w)]
    from lumen_amd import dtypes as D

    def fn(h, w, t):
        loss, pull = L.vjp(lambda h, w: F.linear_cross_entropy(h, w, t), h, w)
        dh, dw = pull(F.sum(h.float()) * 0.0 + 1.0)
        return [loss * 3.0, dh, dw.float() * loss]

    def two(h, w, t, crossed):
        a, pa = L.vjp(lambda h, w: F.linear_cross_entropy(h, w, t, 1), h, w)
        b, pb = L.vjp(lambda h, w: F.linear_cross_entropy(h, w, t, 2), h, w)
        late = a * b
        return [late * 2.0, *pb(a), *pa(b if crossed else prims.full((), 1.0, "float32")), late]

    args = [D.bf16_bits(b) for b in bits] + [target]
    for program, names in ((fn, ["head_loss_backward"]), (lambda *xs: two(*xs, False), ["head_loss_backward"] * 2),
                           (lambda *xs: two(*xs, True), ["head_loss", "head_loss_backward", "head_loss_backward"])):
        graph = L.make_graph(program)(_meta(h, "bfloat16"), _meta(w, "bfloat16"), _meta(target))
        compiled, _ = compile_graph(graph)
        assert [n.params["name"] for n in compiled.nodes if n.prim == "fusion"] == names
        for a, b in zip(oracle.values(graph, args), oracle.values(compiled, args)):
            assert np.array_equal(a, b)


def test_workspace_and_pieces():
    """Memory of the gradients: codes of a piece, and of one piece no sums of the weight's gradient."""
    def workspace(rows, piece, gradients=1):
        n = C.c_size_t()
        d = nv.HeadDesc(rows=rows, classes=32000, k=512, h_m=512, w_n=512, ignore_index=-100, piece_bytes=piece, dtype=1, target_dtype=0)
        nv.call("nhip_head_loss_workspace", C.byref(d), gradients, C.byref(n))
        return n.value

    row, sums = 32000 * 2, 32000 * 512 * 4
    assert workspace(8192, 1 << 30) >= 8192 * row
    assert workspace(8192, 256 * row) < 8192 * row / 8 + 2 * sums
    assert workspace(8192, 256 * row) > 256 * row + sums
    assert workspace(8192, 1 << 30, 0) < 8192 * row / 8


def test_a_piece_holds_rows_of_h_within_a_buffer():
    """Few classes and long rows: the codes of 2^18 rows are 2^29 bytes, which one piece may hold, but their rows of h are 2^32, twice
    what the weight gradient's product reaches: three pieces."""
    n = C.c_size_t()
    rows, k, v = 1 << 18, 1 << 13, 1000
    d = nv.HeadDesc(rows=rows, classes=v, k=k, h_m=k, w_n=k, ignore_index=-100, piece_bytes=1 << 29, dtype=1, target_dtype=0)
    nv.call("nhip_head_loss_workspace", C.byref(d), 1, C.byref(n))
    copy, sums, codes = rows * k * 2, v * k * 4, rows * 1024 * 2
    assert copy + sums + codes / 3 < n.value < copy + sums + codes / 2


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("target_type", ["int32", "int64"])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_losses_alone_of_primitives(dtype, target_type, reduction):
    """Compiled and as traced, the same: targets of any type, which are clamped and converted behind the logits' sums."""
    rng = np.random.default_rng(6)
    h, w, target = _case(rng, (9,), 5, 11, dtype)
    args = [h, w, target.astype(target_type)]
    graph = L.make_graph(lambda h, w, t: [F.linear_cross_entropy(h, w, t, reduction=reduction)])(*(_meta(a) for a in args))
    Plan(graph, build_kernels=False)
    compiled, _ = compile_graph(graph)
    assert [n.prim for n in compiled.nodes].count("linear_cross_entropy") == (dtype == "float32")
    (a,), (b,) = oracle.values(graph, args), oracle.values(compiled, args)
    losses = M.linear_cross_entropy(h, w, target, -100, np.ones(9))[0]
    tol = M.linear_cross_entropy_tolerances(h, w, target, -100, np.ones(9), "float32")[0]
    n = (target != -100).sum()
    want = {"none": losses, "sum": losses.sum(), "mean": losses.sum() / n}[reduction]
    limit = {"none": tol, "sum": tol.sum() + 1e-6 * losses.sum(), "mean": tol.sum() + 1e-6 * losses.sum()}[reduction]
    assert np.all(np.abs(a - want) <= limit) and np.all(np.abs(b - want) <= limit)


def test_a_target_that_depends_on_a_loss():
    """A log-sum-exp that the targets of its own cross entropy, or of one whose log-sum-exp its targets take in turn, are computed from
    stays as primitives; one after the other they become a step each. 1e-5: some 20 float32 roundings of values below 8."""
    from lumen_amd.graph.tracer import dot

    def parts(h, w, target):
        t, v = h.shape[0], w.shape[0]
        x = dot(h, w, (((1,), (1,)), ((), ())), "float32", "float32")
        m = F.amax(x, -1, keepdim=True)
        lse = m.reshape(t) + F.log(F.sum(F.exp(x - m), -1))
        return x, lse, lambda target: lse - prims.gather(x.reshape(t * v), prims.iota("int64", [t], 0) * v + target, 0)

    def classes(lse):
        return F.where(prims.lt(lse, prims.full(lse.shape, 2.0, "float32")), prims.full(lse.shape, 1, "int64"), prims.full(lse.shape, 3, "int64"))

    def own(h, w, u, t):
        _, lse, loss = parts(h, w, t)
        return [loss(classes(lse)), lse]

    def crossed(h, w, u, t):
        _, a, loss_a = parts(h, w, t)
        _, b, loss_b = parts(h, u, t)
        return [loss_a(classes(b)), loss_b(classes(a)), a, b]

    def chained(h, w, u, t):
        _, a, loss_a = parts(h, w, t)
        _, b, loss_b = parts(h, u, t)
        return [loss_a(t), loss_b(classes(a)), b]

    rng = np.random.default_rng(7)
    h, w, _ = _case(rng, (9,), 5, 11, "float32")
    args = [h, w, rng.standard_normal((11, 5)).astype(np.float32), rng.integers(0, 11, 9)]
    for program, count in ((own, 0), (crossed, 1), (chained, 2)):
        graph = L.make_graph(program)(*(_meta(a) for a in args))
        compiled, _ = compile_graph(graph)
        assert [n.prim for n in compiled.nodes].count("linear_cross_entropy") == count, program.__name__
        for a, b in zip(oracle.values(graph, args), oracle.values(compiled, args)):
            assert np.abs(a - b).max() <= 1e-5


STRIDED = {  # shapes of the input, weight and target, and what each is read as
    "columns of rows of a batch": ([3, 10, 128], [50, 64], [3, 10], lambda x: x[:, :, 64:], lambda w: w, lambda t: t),
    "columns of the weight": ([30, 64], [50, 128], [30], lambda x: x, lambda w: w[:, 64:], lambda t: t),
    "a permuted weight": ([30, 64], [64, 10, 5], [30], lambda x: x, lambda w: w.permute(1, 2, 0).reshape(50, 64), lambda t: t),
    "one row for all": ([1, 1, 64], [50, 64], [3, 10], lambda x: x.expand(3, 10, 64), lambda w: w, lambda t: t),
    "a column of targets": ([30, 64], [50, 64], [30, 2], lambda x: x, lambda w: w, lambda t: t[:, 1]),
}


@pytest.mark.parametrize("what", STRIDED)
def test_views_as_operands_of_primitives(what):
    """The step that the losses alone become reads contiguous operands: the views that are none are copied."""
    *shapes, of_x, of_w, of_t = STRIDED[what]
    metas = [L.empty(s, d, "meta") for s, d in zip(shapes, ("float32", "float32", "int64"))]
    plan = Plan(L.make_graph(lambda h, w, t: [F.linear_cross_entropy(of_x(h), of_w(w), of_t(t))])(*metas), build_kernels=False)
    (step,) = [st for st in plan.steps if st.kind == "linear_cross_entropy"]
    assert all(plan.loc[v].contiguous() for v in step.nodes[0].inputs)


@pytest.mark.parametrize("classes", [(1 << 22) - 64, (1 << 22) - 63, (1 << 22) - 1, 1 << 22])
def test_the_most_classes_that_the_kernels_take(classes):
    """What the library would refuse is primitives: blocks of 64 classes below 2^22 are the kernels'."""
    g = _graph(lambda h, w, t: [F.linear_cross_entropy(h, w, t)], t=3, k=64, v=classes, g=None)
    kinds = [st.kind for st in Plan(g, build_kernels=False).steps]
    assert ("head_loss" in kinds) == (classes <= (1 << 22) - 64)


def test_what_is_taken_is_what_the_library_takes():
    """The sizes at which the kernels' rule ends, against the library's own check of them."""
    from lumen_amd.functional.linear_cross_entropy import _taken

    class Shaped:
        dtype = "bfloat16"

        def __init__(self, *shape):
            self.shape = shape

    def library(t, k, v):
        n = C.c_size_t()
        d = nv.HeadDesc(rows=t, classes=v, k=k, h_m=k, w_n=k, ignore_index=-100, piece_bytes=1 << 29, dtype=1, target_dtype=0)
        try:
            nv.call("nhip_head_loss_workspace", C.byref(d), 1, C.byref(n))
        except RuntimeError:
            return False
        return True

    seen = set()
    for t, k, v in [(1, 64, (1 << 22) - 64 + i) for i in (-1, 0, 1, 63, 64)] + [((1 << 26) + i, 1, 1) for i in (-1, 0)] \
            + [(1, (1 << 20) - 64 + i, 1) for i in (-1, 0, 1)] + [(1, 1024, (1 << 20) - 257 + i) for i in range(-2, 3)] \
            + [((1 << 19) + i, 64, 128 * 4096) for i in (-128, 1)] + [(1 << 25, 64, 8192 + i) for i in (0, 1)] + [(1 << 25, 8192 + i, 64) for i in (0, 1)] \
            + [(100, 4096, 262144 - 256 - i) for i in range(3)]:
        taken = _taken(Shaped(t, k), Shaped(v, k))
        seen.add(taken)
        assert taken == library(t, k, v), (t, k, v)
    assert seen == {True, False}


def test_rows_as_far_apart_as_the_library_reads_them():
    """The distance up to which rows stay where they lie, against the library's own check of it."""
    from lumen_amd.compiler import operators
    from lumen_amd.compiler.plan import Loc

    n, seen = C.c_size_t(), set()
    for k in (64, 1024, 2048, 8192):
        for stride in [(((1 << 30) - 1024 - k) // 256 + i) // 8 * 8 for i in range(-16, 24, 8)] + [1 << 22, 1 << 30]:
            taken = operators.reads(Loc(("in", 0), 0, (stride, 1), "bfloat16", (300, k)), {operators.WIDE_ROWS})
            d = nv.HeadDesc(rows=300, classes=10, k=k, h_m=stride, w_n=k, ignore_index=-100, piece_bytes=1 << 29, dtype=1, target_dtype=0)
            try:
                nv.call("nhip_head_loss_workspace", C.byref(d), 0, C.byref(n))
                read = True
            except RuntimeError:
                read = False
            seen.add(taken)
            assert read or not taken, (k, stride)
    assert seen == {True, False}


def test_scratch_of_the_losses_alone():
    """Eight bytes a row and 64 classes, of as many rows as fit the piece's bytes: of 2^20 rows and 128256 classes (16.8 GB at once) 2^29."""
    def workspace(rows, classes, piece):
        n = C.c_size_t()
        d = nv.HeadDesc(rows=rows, classes=classes, k=512, h_m=512, w_n=512, ignore_index=-100, piece_bytes=piece, dtype=1, target_dtype=0)
        nv.call("nhip_head_loss_workspace", C.byref(d), 0, C.byref(n))
        return n.value

    assert workspace(1 << 20, 128256, 1 << 29) <= (1 << 29) + (1 << 20)
    assert workspace(100, 128256, 1 << 29) >= 100 * 2004 * 8
    assert 256 * 2004 * 8 <= workspace(1 << 20, 128256, 0) < 256 * 2004 * 8 + 2048
    assert workspace(0, 10, 0) < 1024
