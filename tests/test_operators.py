"""qk_norm_rope, gated_linear and clip_grad_norm on the CPU: what they compute (the oracle on their traced bodies against
plain float64 NumPy), their gradients against the formula's differences, their refusals, and the plans they become."""

import ctypes as C

import numpy as np
import pytest

import lumen_amd as L
import lumen_amd.functional as F
from lumen_amd import dtypes as D
from lumen_amd import native as nv
from lumen_amd.compiler.plan import Plan
from oracle import oracle
from tests import operator_math as M


def _graph(fn, *arrays, dtypes=None):
    metas = [L.empty(list(a.shape), dt or D.canonical(a.dtype), "meta") for a, dt in zip(arrays, dtypes or [None] * len(arrays))]
    return L.make_graph(fn)(*metas)


def _run(fn, *arrays, fused=True):
    """The oracle's outputs of ``fn`` on float32/float64 arrays (their own dtypes)."""
    with L.config.compiler.patch(fused_operators=fused):
        g = _graph(fn, *arrays)
    return [np.asarray(v, np.float64) for v in oracle.values(g, list(arrays))], g


# ---- values and gradients, float64 (traced as primitives) and float32 (one fusion)


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("d,rot,interleaved,weights,positions", [
    (16, 16, False, True, False), (16, 8, True, True, True), (10, 6, False, False, True), (7, 2, True, True, False),
    (8, 0, False, True, True), (1, 0, False, False, False)])
def test_heads_values_and_gradients(dtype, d, rot, interleaved, weights, positions):
    """Both directions against float64 NumPy. float32: about 3 D + 20 roundings of 2^-24 a value, relative to the largest
    value of the tensor; a weight's gradient sums B S N = 18 rows more. float64 the same with 2^-53."""
    rng = np.random.default_rng(d + rot)
    b, s, n, nkv = 2, 3, 3, 1
    x = M.heads_inputs(rng, b, s, n, nkv, d, rot, table=9, dtype=dtype, weights=weights, positions=positions)
    names = list(x)

    def fn(*args):
        t = dict(zip(names, args))
        keep = [m for m in ("q", "k", "wq", "wk") if m in t]

        def f(*leaves):
            v = {**t, **dict(zip(keep, leaves))}
            return F.qk_norm_rope(v["q"], v["k"], v["cos"], v["sin"], v.get("wq"), v.get("wk"), positions=v.get("positions"),
                                  eps=1e-3, interleaved=interleaved)

        out, pull = L.vjp(f, *(t[m] for m in keep))
        return [*out, *pull((t["gq"], t["gk"]))]

    got, g = _run(fn, *x.values())
    fusions = [m.params["name"] for m in g.nodes if m.prim == "fusion"]
    assert fusions == (["qk_norm_rope", "qk_norm_rope_backward"] if dtype == "float32" else [])
    want = M.heads(x, 1e-3, interleaved)
    step = 2.0**-24 if dtype == "float32" else 2.0**-53
    for a, w in zip(got, want):
        assert a.shape == w.shape
        assert np.abs(a - w).max() <= step * (3 * d + 40) * max(1.0, np.abs(w).max())


def test_heads_gradient_against_differences():
    """The float64 gradient of every input against central differences of the value (step 1e-6: 1e-9 from the third
    derivative and 1e-10 from the rounding of the values)."""
    rng = np.random.default_rng(3)
    x = M.heads_inputs(rng, 1, 3, 2, 1, 8, 6, table=5, dtype="float64", weights=True, positions=True)
    want = M.heads(x, 1e-3, False)
    grads = dict(zip(("q", "k", "wq", "wk"), want[2:]))

    def value(x):
        yq, yk = M.heads(x, 1e-3, False)[:2]
        return (yq * x["gq"]).sum() + (yk * x["gk"]).sum()

    for name, g in grads.items():
        assert np.abs(g - M.differences(value, x, name)).max() <= 1e-7, name


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("activation", M.ACTIVATIONS)
def test_gated_values_and_gradients(activation, dtype):
    """float32: sums of K = 11 and F = 6 products (each rounded) and a few more roundings; float64 the same."""
    rng = np.random.default_rng(len(activation))
    x, gate, up, dh = (rng.standard_normal(s).astype(dtype) for s in ((2, 4, 11), (6, 11), (6, 11), (2, 4, 6)))

    def fn(x, gate, up, dh):
        h, pull = L.vjp(lambda x, gate, up: F.gated_linear(x, gate, up, activation=activation), x, gate, up)
        return [h, *pull(dh)]

    got, g = _run(fn, x, gate, up, dh)
    step = 2.0**-24 if dtype == "float32" else 2.0**-53
    for a, w in zip(got, M.gated(x, gate, up, dh, activation)):
        assert a.shape == w.shape
        assert np.abs(a - w).max() <= step * 100 * max(1.0, np.abs(w).max())


@pytest.mark.parametrize("activation", M.ACTIVATIONS)
def test_gated_gradient_against_differences(activation):
    rng = np.random.default_rng(8)
    x = {n: rng.standard_normal(s) for n, s in (("x", (3, 5)), ("gate", (4, 5)), ("up", (4, 5)), ("dh", (3, 4)))}
    grads = M.gated(*x.values(), activation)[1:]
    for name, g in zip(("x", "gate", "up"), grads):
        diff = M.differences(lambda x: (M.gated(*x.values(), activation)[0] * x["dh"]).sum(), x, name)
        assert np.abs(g - diff).max() <= 1e-6, name


def test_gated_16_bit_is_two_fusions_and_ordinary_products():
    g = _graph(lambda x, gate, up, dh: (lambda h, pull: [h, *pull(dh)])(*L.vjp(F.gated_linear, x, gate, up)),
               *(np.zeros(s, np.uint16) for s in ((64, 64), (128, 64), (128, 64), (64, 128))), dtypes=["bfloat16"] * 4)
    assert [n.params["name"] for n in g.nodes if n.prim == "fusion"] == ["gated_linear", "gated_linear_grad",
                                                                                          "gated_input_grad"]
    # tokens and features that are not whole tiles and chunks: the weights' gradients by the operator's own kernel
    ragged = _graph(lambda x, gate, up, dh: (lambda h, pull: [h, *pull(dh)])(*L.vjp(F.gated_linear, x, gate, up)),
                    *(np.zeros(s, np.uint16) for s in ((65, 64), (127, 64), (127, 64), (65, 127))), dtypes=["bfloat16"] * 4)
    assert [n.params["name"] for n in ragged.nodes if n.prim == "fusion"][2:] == ["gated_input_grad", "gated_weight_grad"]
    forward = _graph(F_gated, *(np.zeros(s, np.uint16) for s in ((64, 64), (128, 64), (128, 64))), dtypes=["bfloat16"] * 3)
    plan = Plan(forward, build_kernels=False)
    assert [st.kind for st in plan.steps] == ["gated_fwd"] and len(plan.steps[0].outputs) == 1  # g and u are not stored


def F_gated(x, gate, up):
    return [F.gated_linear(x, gate, up)]


@pytest.mark.parametrize("fused", [True, False])
def test_clip_values(fused):
    """float32 and float64 tensors, a 0-d one and an empty one; over the bound, below it, and with a traced bound."""
    rng = np.random.default_rng(5)
    xs = [rng.standard_normal(s).astype(np.float32) for s in ((5, 3), (), (7,), (0, 4))]
    norm = np.sqrt(sum((x.astype(np.float64)**2).sum() for x in xs))
    for bound in (0.5 * norm, 2 * norm, 0.0):
        got, g = _run(lambda *xs: (lambda c, n: [n, *c])(*F.clip_grad_norm(xs, float(bound))), *xs, fused=fused)
        assert sum(n.prim == "fusion" for n in g.nodes) == fused
        scale = min(1.0, bound / (norm + 1e-6))
        assert abs(got[0] - norm) <= 2.0**-24 * norm
        for a, x in zip(got[1:], xs):
            assert np.abs(a - x * scale).max(initial=0) <= 2.0**-23 * np.abs(x).max(initial=0)
    traced = L.make_graph(lambda bound, *xs: (lambda c, n: [n, *c])(*F.clip_grad_norm(xs, bound)))(
        0.5 * float(norm), *[L.empty(list(x.shape), "float32", "meta") for x in xs])
    tensors = [v for v in traced.inputs if traced.types[v].dtype == "float32"]
    arrays = dict(zip(tensors, xs))
    got = oracle.values(traced, [arrays.get(v, np.array(0.5 * norm)) for v in traced.inputs])
    assert np.abs(got[1] - 0.5 * xs[0]).max() <= 1e-6


def test_clip_of_extreme_values():
    """Squares that overflow and underflow float32, an infinity and a NaN."""
    big = np.array([3e38, -1e38], np.float32)
    tiny = np.array([1e-30, 3e-30], np.float32)
    clip = lambda x: (lambda c, n: [n, *c])(*F.clip_grad_norm([x], 1.0, eps=0.0))  # noqa: E731
    (norm, out), _ = _run(clip, big)
    np.testing.assert_allclose(out, big / np.float64(np.hypot(3e38, 1e38)), rtol=1e-6)
    (norm, out), _ = _run(clip, tiny)
    np.testing.assert_allclose(norm, np.sqrt(10) * 1e-30, rtol=1e-6)
    assert np.array_equal(out, tiny.astype(np.float64))
    (norm, out), _ = _run(clip, np.array([np.inf, 2.0], np.float32))
    assert np.isinf(norm) and np.isnan(out[0]) and out[1] == 0
    (norm, out), _ = _run(clip, np.array([np.nan, 2.0], np.float32))
    assert np.isnan(norm) and np.isnan(out).all()


def test_clip_of_many_tensors():
    """More tensors than a launch's table holds: one step, every result."""
    xs = [np.full((3,), i, np.float32) for i in range(130)]
    got, g = _run(lambda *xs: (lambda c, n: [n, *c])(*F.clip_grad_norm(xs, 1.0)), *xs)
    norm = np.sqrt(3 * sum(i * i for i in range(130)))
    assert abs(got[0] - norm) <= 1e-6 * norm and len(got) == 131
    np.testing.assert_allclose(got[-1], 129 / (norm + 1e-6), rtol=1e-6)


# ---- refusals


def _m(shape, dtype="bfloat16"):
    return L.empty(list(shape), dtype, "meta")


BAD_HEADS = {
    "3-D query": (ValueError, "4-D", dict(q=(2, 3, 8))),
    "head dims differ": (ValueError, "differ in batch", dict(k=(2, 3, 1, 16))),
    "sequences differ": (ValueError, "differ in batch", dict(k=(2, 4, 1, 8))),
    "integer heads": (TypeError, "floating-point", dict(dtype="int32")),
    "16-bit table": (ValueError, "cos is not a float32", dict(table="bfloat16")),
    "table too wide": (ValueError, "do not turn pairs", dict(cos=(9, 5), sin=(9, 5))),
    "tables differ": (ValueError, "do not turn pairs", dict(cos=(9, 4), sin=(9, 3))),
    "short table": (ValueError, "tables of 2 positions", dict(cos=(2, 4), sin=(2, 4))),
    "weight of another size": (TypeError, "query weight must be", dict(wq=(4,))),
    "positions of another shape": (ValueError, "positions must be", dict(positions=(2, 4))),
    "float positions": (ValueError, "positions must be", dict(positions=(2, 3), ptype="float32")),
    "negative eps": (ValueError, "eps must be", dict(eps=-1.0)),
    "eps that is no number": (ValueError, "eps must be", dict(eps=float("nan"))),
}


@pytest.mark.parametrize("name", sorted(BAD_HEADS))
def test_heads_refusals(name):
    error, match, c = BAD_HEADS[name]
    dt = c.get("dtype", "bfloat16")
    args = [_m(c.get("q", (2, 3, 4, 8)), dt), _m(c.get("k", (2, 3, 1, 8)), dt), _m(c.get("cos", (9, 4)), c.get("table", "float32")),
            _m(c.get("sin", (9, 4)), "float32"), _m(c.get("wq", (8,)), dt)]
    if "positions" in c:
        args.append(_m(c["positions"], c.get("ptype", "int32")))
    with pytest.raises(error, match=match):
        L.make_graph(lambda q, k, cos, sin, wq, p=None: list(
            F.qk_norm_rope(q, k, cos, sin, wq, positions=p, eps=c.get("eps"))))(*args)


def test_heads_of_two_dtypes_are_refused():
    with pytest.raises(TypeError, match="convert them to one"):
        L.make_graph(lambda q, k, c, s: list(F.qk_norm_rope(q, k, c, s)))(
            _m((1, 2, 2, 8)), _m((1, 2, 2, 8), "float32"), _m((2, 4), "float32"), _m((2, 4), "float32"))


@pytest.mark.parametrize("x,gate,up,dtypes,activation,error,match", [
    ((4, 8), (6, 7), (6, 8), None, "silu", ValueError, "gate weight must be"),
    ((4, 8), (6, 8), (5, 8), None, "silu", ValueError, "differ"),
    ((4, 8), (6, 8, 1), (6, 8), None, "silu", ValueError, "gate weight must be"),
    ((4, 8), (6, 8), (6, 8), ("bfloat16", "float32", "bfloat16"), "silu", TypeError, "convert them to one"),
    ((4, 8), (6, 8), (6, 8), ("int32",) * 3, "silu", TypeError, "floating-point"),
    ((4, 8), (6, 8), (6, 8), None, "swish", ValueError, "activation must be one of"),
])
def test_gated_refusals(x, gate, up, dtypes, activation, error, match):
    with pytest.raises(error, match=match):
        L.make_graph(lambda x, g, u: F.gated_linear(x, g, u, activation=activation))(
            *(_m(s, d) for s, d in zip((x, gate, up), dtypes or ("bfloat16",) * 3)))


def test_clip_refusals():
    def clip(*args, **kw):
        return lambda x: (lambda c, n: [n, *c])(*F.clip_grad_norm([x], *args, **kw))

    for fn, error, match in [
        (clip(-1.0), ValueError, "max_norm must be at least 0"), (clip(float("nan")), ValueError, "max_norm"),
        (clip("1"), ValueError, "max_norm"), (clip(1.0, eps=-1.0), ValueError, "eps"),
        (lambda x: F.clip_grad_norm(x, 1.0)[1], TypeError, "list or tuple"),
        (lambda x: F.clip_grad_norm([], 1.0)[1], ValueError, "no gradients"),
        (lambda x: F.clip_grad_norm([2.0], 1.0)[1], TypeError, "gradients are tensors"),
        (lambda x: F.clip_grad_norm([x], x)[1], TypeError, "float scalar"),
        (lambda x: L.grad(lambda x: F.clip_grad_norm([x], 1.0)[1])(x), NotImplementedError, "no gradient"),
    ]:
        with pytest.raises(error, match=match):
            L.make_graph(fn)(_m((4,), "float32"))
    with pytest.raises(TypeError, match="floating-point"):
        L.make_graph(clip(1.0))(_m((4,), "int32"))


def test_vjp_of_several_results():
    """A pullback of several results takes as many cotangents and sums what they send back."""
    x = np.array([1.0, 2.0])

    def fn(x):
        out, pull = L.vjp(lambda x: (x * x, x * 3.0), x)
        return [*out, *pull((x, x))]

    got, _ = _run(fn, x)
    assert np.array_equal(got[2], 2 * x * x + 3 * x)
    with pytest.raises(TypeError, match="2 results take as many"):
        L.make_graph(lambda x: list(L.vjp(lambda x: (x * x, x * 3.0), x)[1](x)))(_m((2,), "float32"))


def test_abi_refusals():
    """Bad descriptors are refused before anything is queued (no GPU here: what passes fails for its missing stream)."""
    def heads(**kw):
        d = dict(batch=1, seq=4, heads=2, kv_heads=1, head_dim=64, rot=64, table_rows=4, dtype=1)
        return nv.HeadsDesc(**{**d, **kw})

    n = C.c_size_t()
    for bad, match in [(heads(head_dim=0), "head dim"), (heads(head_dim=1025), "head dim"), (heads(rot=3), "rotated"),
                       (heads(rot=66), "rotated"), (heads(table_rows=0), "empty table"), (heads(dtype=3), "float32, bf16"),
                       (heads(positions=3), "positions"), (heads(seq=1 << 30), "2\\^30"), (heads(batch=-1), "negative")]:
        with pytest.raises(RuntimeError, match=match):
            nv.call("nhip_qk_norm_rope_workspace", C.byref(bad), C.byref(n))
    nv.call("nhip_qk_norm_rope_workspace", C.byref(heads()), C.byref(n))
    assert n.value == 2050 * 64 * 4  # a row of partial sums for each workgroup of the largest launch
    nv.call("nhip_clip_grad_norm_workspace", C.byref(nv.ClipDesc(count=121)), C.byref(n))
    assert n.value == 2 * 1024 * 8
    with pytest.raises(RuntimeError, match="negative count"):
        nv.call("nhip_clip_grad_norm_workspace", C.byref(nv.ClipDesc(count=-1)), C.byref(n))
    for kw, match in [(dict(m=-1), "negative"), (dict(dtype=0), "bf16 or f16"), (dict(activation=4), "activation")]:
        with pytest.raises(RuntimeError, match=match):
            nv.call("nhip_gated_linear_workspace", C.byref(nv.GatedDesc(**{**dict(m=1, n=1, k=1, dtype=1, config=-1), **kw})), C.byref(n))
    for m, k, want in [(64, 515, 0), (65, 512, 0), (65, 515, (65 + 2 * 8) * 520 * 2)]:  # few rows are read as they are
        nv.call("nhip_gated_linear_workspace", C.byref(nv.GatedDesc(m=m, n=8, k=k, x_m=k, w_n=k, dtype=1, config=-1)), C.byref(n))
        assert n.value == want
    for kw, match in [(dict(m=-1), "negative"), (dict(dtype=0), "bf16 or f16"), (dict(n=1 << 21), "2\\^31"),
                      (dict(n=1 << 15, k=1 << 15), "2\\^31")]:
        d = nv.GatedDesc(**{**dict(m=64, n=64, k=64, x_m=64, w_n=64, dtype=1, config=-1), **kw})
        with pytest.raises(RuntimeError, match=match):
            nv.call("nhip_gated_backward_workspace", C.byref(d), C.byref(n))
    for m, n_, k, want in [(64, 64, 64, 0), (64, 63, 64, 2 * 64 * 64 * 2), (65, 64, 63, 2 * 64 * 64 * 2), (4096, 64, 63, 4096 * 64 * 2),
                           (0, 64, 64, 0), (64, 0, 64, 0), (64, 64, 0, 0), (0, 0, 0, 0)]:
        nv.call("nhip_gated_backward_workspace", C.byref(nv.GatedDesc(m=m, n=n_, k=k, x_m=k, w_n=k, dtype=1, config=-1)), C.byref(n))
        assert n.value >= want and (want or not n.value)
    plan = C.c_void_p()
    nv.call("nhip_plan_create", C.byref(plan))
    d = nv.ClipDesc(count=3)
    rr = (nv.Reloc * 1)(nv.Reloc(slot=10))
    with pytest.raises(RuntimeError, match="descriptor of"):
        nv.call("nhip_plan_add_builtin", plan, nv.NHIP_STEP_CLIP, bytes(d), len(bytes(d)), rr, 0)
    full = bytes(d) + bytes((nv.ClipTensor * 3)())
    with pytest.raises(RuntimeError, match="slot"):
        nv.call("nhip_plan_add_builtin", plan, nv.NHIP_STEP_CLIP, full, len(full), rr, 1)
    nv.call("nhip_plan_destroy", plan)


def test_gated_kernels_refuse_rows_of_nothing_and_rows_past_a_buffer():
    """Above 64 rows the kernels read through buffers of at most 2^31 bytes and need a k; the trace holds primitives there."""
    n = C.c_size_t()
    for m, k, taken in [(64, 0, True), (65, 0, False), (65, 1 << 21, False), (64, 1 << 21, True), (65, (1 << 21) - 8, True)]:
        d = nv.GatedDesc(m=m, n=8, k=k, x_m=k, w_n=k, dtype=1, config=-1)
        if taken:
            nv.call("nhip_gated_linear_workspace", C.byref(d), C.byref(n))
        else:
            with pytest.raises(RuntimeError, match="elements a row"):
                nv.call("nhip_gated_linear_workspace", C.byref(d), C.byref(n))
    for k, fusions in [(0, []), (1 << 21, []), (8, ["gated_linear"])]:
        g = L.make_graph(F_gated)(*(_m((rows, k), "bfloat16") for rows in (70, 8, 8)))
        assert [m.params["name"] for m in g.nodes if m.prim == "fusion"] == fusions


def test_heads_past_a_launch_are_primitives():
    def fn(q, k, c, s):
        return list(F.qk_norm_rope(q, k, c, s))

    for heads, fusions in [((1 << 20) - 1, 1), (1 << 20, 0)]:
        g = L.make_graph(fn)(_m((1, 1, heads, 2), "float32"), _m((1, 1, 1, 2), "float32"), *[_m((1, 1), "float32")] * 2)
        assert sum(m.prim == "fusion" for m in g.nodes) == fusions


@pytest.mark.parametrize("g0", [1e25, -1e25])
def test_gelu_gradient_where_the_square_overflows(g0):
    """act(g) is g or 0 and act'(g) 1 or 0: exact, though g g is no float32."""
    x, gate, up, dh = (np.array(v, np.float32) for v in ([[g0, 2.0]], [[1.0, 0.0]], [[0.0, 1.0]], [[3.0]]))

    def fn(x, gate, up, dh):
        h, pull = L.vjp(lambda x, gate, up: F.gated_linear(x, gate, up, activation="gelu"), x, gate, up)
        return [h, *pull(dh)]

    got, _ = _run(fn, x, gate, up, dh)
    g = np.float64(np.float32(g0))
    a, d = (g, 1.0) if g0 > 0 else (0.0, 0.0)
    want = [[[2 * a]], [[6 * d, 3 * a]], [[6 * d * g, 12 * d]], [[3 * a * g, 6 * a]]]
    for v, w in zip(got, want):
        assert np.all(np.abs(v - np.array(w)) <= 2.0**-22 * np.abs(w)) or not np.isfinite(np.float32(w)).all()


def test_an_operand_used_twice():
    """Queries that are the keys, a gate that is the up projection, a gradient listed twice: each use has its part."""
    rng = np.random.default_rng(21)
    x = M.heads_inputs(rng, 1, 4, 2, 2, 8, 8, table=4, dtype="float64", positions=False)
    x["k"], x["wk"] = x["q"], x["wq"]

    def heads(q, w, c, s, gq, gk):
        out, pull = L.vjp(lambda q, w: F.qk_norm_rope(q, q, c, s, w, w, eps=1e-3), q, w)
        return [*out, *pull((gq, gk))]

    got, _ = _run(heads, *(x[n] for n in ("q", "wq", "cos", "sin", "gq", "gk")))
    want = M.heads(x, 1e-3, False)
    want = [want[0], want[1], want[2] + want[3], want[4] + want[5]]
    t, w, dh = rng.standard_normal((3, 5)), rng.standard_normal((4, 5)), rng.standard_normal((3, 4))

    def gated(t, w, dh):
        h, pull = L.vjp(lambda t, w: F.gated_linear(t, w, w), t, w)
        return [h, *pull(dh)]

    got += _run(gated, t, w, dh)[0]
    h, dx, dg, du = M.gated(t, w, w, dh, "silu")
    want += [h, dx, dg + du]
    got += _run(lambda g: (lambda c, n: [n, *c])(*F.clip_grad_norm([g, g], 1.0)), t)[0]
    scale = min(1.0, 1 / (np.sqrt(2 * (t * t).sum()) + 1e-6))
    want += [np.sqrt(2 * (t * t).sum()), t * scale, t * scale]
    for i, (a, b) in enumerate(zip(got, want)):
        # float64 to a few hundred roundings; the tables and the scale are float32
        assert np.abs(a - b).max() <= 2.0**-22 * max(1, np.abs(b).max()), i


# ---- plans


def test_operands_that_are_no_rows_are_copied():
    """A merged projection's heads are read in place through their strides; a transposed operand, whose rows a view would
    not keep contiguous, becomes a copy."""
    def packed(x, cos, sin):
        q, k = x[:, :, :128].reshape(1, 6, 2, 64), x[:, :, 128:192].reshape(1, 6, 1, 64)
        return list(F.qk_norm_rope(q, k, cos, sin))

    plan = Plan(L.make_graph(packed)(_m((1, 6, 256)), _m((8, 32), "float32"), _m((8, 32), "float32")), build_kernels=False)
    kinds = [st.kind for st in plan.steps]
    assert kinds.count("heads_fwd") == 1 and "loop" not in kinds
    plan = Plan(L.make_graph(lambda xt, g, ut: [F.gated_linear(xt.t(), g, ut.t())])(
        _m((64, 32)), _m((48, 64)), _m((64, 48))), build_kernels=False)
    step = plan.steps[-1]
    assert step.kind == "gated_fwd" and [st.kind for st in plan.steps].count("loop") >= 1
    for v in step.nodes[0].inputs:
        assert plan.loc[v].strides[-1] == 1


def test_clipped_gradients_scale_in_the_update_that_reads_them():
    """An update p - lr clipped(g) reads g and the scale: the clipping step writes the norm alone, with the same values."""
    def step(p, q, gp, gq):
        (cp, cq), norm = F.clip_grad_norm([gp, gq], 0.5)
        return [norm, p - 0.1 * cp, q - 0.1 * cq]

    def plan_of():
        g = L.make_graph(step)(*[_m(s) for s in ((8, 16), (5,), (8, 16), (5,))])
        return Plan(g, build_kernels=False), g

    plan, g = plan_of()
    (clip,) = [st for st in plan.steps if st.kind == "clip"]
    assert len(clip.outputs) == 2  # the norm and the scale
    rng = np.random.default_rng(0)
    xs = [D.bf16_bits(rng.standard_normal(s).astype(np.float32)) for s in ((8, 16), (5,), (8, 16), (5,))]
    for a, b in zip(oracle.run(g, xs), oracle.run(plan.graph, xs)):
        assert np.array_equal(a, b)


def test_gradients_of_few_tiles_are_one_step():
    """Few tiles: one step of all three gradients; many, or an input that needs none: the products' own steps."""
    def plan(t, k, n, leaves):
        def fn(x, gate, up, dh):
            h, pull = L.vjp(lambda *w: F.gated_linear(*(w if leaves == 3 else (x, *w))), *(x, gate, up)[3 - leaves:])
            return [h, *pull(dh)]

        return Plan(L.make_graph(fn)(*(_m(s) for s in ((t, k), (n, k), (n, k), (t, n)))), build_kernels=False)

    assert [st.kind for st in plan(777, 520, 1416, 3).steps] == ["gated_fwd", "gated_grad", "gated_both"]
    assert [st.kind for st in plan(777, 520, 1416, 2).steps] == ["gated_fwd", "gated_grad", "gated_weight"]
    assert [st.kind for st in plan(4001, 2048, 8192, 3).steps] == ["gated_fwd", "gated_grad", "gated_weight", "gated_input"]
    steps = plan(130, 67, 333, 3).steps
    n = C.c_size_t()
    nv.call("nhip_gated_backward_workspace", C.byref(nv.GatedDesc(m=130, n=333, k=67, x_m=67, w_n=67, dtype=1, config=-1)), C.byref(n))
    assert steps[-1].kind == "gated_both" and steps[-1].scratch >= n.value


# ---- the tape used again: several backward() calls in one trace, gradients of gradients


def _bits(x, dtype="bfloat16"):
    return np.ascontiguousarray(D.from_values(np.asarray(x, np.float32), dtype))


def _rounded(x, dtype="bfloat16"):
    return np.asarray(D.to_numpy_values(_bits(x, dtype), dtype), np.float64)


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("activation", M.ACTIVATIONS)
@pytest.mark.parametrize("t,k,n", [(16, 16, 16), (5, 11, 6), (64, 16, 24)])
def test_gated_gradients_of_two_micro_batches(t, k, n, activation, fused):
    """``backward()`` after each micro-batch: the weights' gradients are the sums, each input's its own. Two gradients within
    their own bounds, each of them rounded, and their sum's rounding."""
    from tests.test_gpu_operators import _gated_tolerances

    rng = np.random.default_rng(t + n)
    gate, up = (_rounded(rng.standard_normal((n, k)) / np.sqrt(k)) for _ in range(2))
    batches = [tuple(_rounded(rng.standard_normal(s)) for s in ((t, k), (t, n))) for _ in range(2)]

    def fn(x1, x2, gate, up, dy1, dy2):
        for x, dy in ((x1, dy1), (x2, dy2)):
            F.gated_linear(x, gate, up, activation=activation).backward(dy)
        return [x1.grad, x2.grad, gate.grad, up.grad]

    arrays = [_bits(v) for v in (batches[0][0], batches[1][0], gate, up, batches[0][1], batches[1][1])]
    with L.config.compiler.patch(fused_operators=fused):
        g = _graph(fn, *arrays, dtypes=["bfloat16"] * 6)
    got = [np.asarray(v, np.float64) for v in oracle.values(g, arrays)]
    want = [M.gated(x, gate, up, dy, activation) for x, dy in batches]
    tol = [_gated_tolerances(x, gate, up, dy, activation, "bfloat16") for x, dy in batches]
    for i in range(2):
        assert np.all(np.abs(got[i] - want[i][1]) <= tol[i][1]), i
    for i in (2, 3):
        w = want[0][i] + want[1][i]
        each = tol[0][i] + tol[1][i]
        assert np.all(np.abs(got[i] - w) <= each + 2.0**-8 * (np.abs(w) + each)), i


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("s,n,nkv,d", [(4, 4, 4, 4), (3, 3, 1, 10)])
def test_heads_gradients_of_two_micro_batches(s, n, nkv, d, fused):
    """As above: one rounding of the sum more than test_heads_values_and_gradients counts."""
    rng = np.random.default_rng(s)
    x = [M.heads_inputs(rng, 2, s, n, nkv, d, d, table=9) for _ in range(2)]
    for m in ("wq", "wk", "cos", "sin"):
        x[1][m] = x[0][m]
    own = ("q", "k", "gq", "gk", "positions")

    def fn(wq, wk, cos, sin, *rest):
        parts = [dict(zip(own, rest[:5])), dict(zip(own, rest[5:]))]
        for p in parts:
            yq, yk = F.qk_norm_rope(p["q"], p["k"], cos, sin, wq, wk, positions=p["positions"], eps=1e-3)
            F.sum(yq * p["gq"]).backward()
            F.sum(yk * p["gk"]).backward()
        return [wq.grad, wk.grad, *(p[m].grad for p in parts for m in ("q", "k"))]

    got, _ = _run(fn, *(x[0][m] for m in ("wq", "wk", "cos", "sin")), *(p[m] for p in x for m in own), fused=fused)
    a, b = (M.heads(p, 1e-3, False) for p in x)
    for v, w in zip(got, [a[4] + b[4], a[5] + b[5], a[2], a[3], b[2], b[3]]):
        assert np.abs(v - w).max() <= 2.0**-24 * (3 * d + 40) * 4 * max(1.0, np.abs(w).max())


@pytest.mark.parametrize("fused", [True, False])
def test_a_later_loss_that_does_not_use_the_operator(fused):
    """The second backward() walks a tape that holds the first one's nodes: a weight that both losses share has both
    gradients, exactly (a plain product of small integers besides the gated one's bounds)."""
    from tests.test_gpu_operators import _gated_tolerances

    rng = np.random.default_rng(2)
    x, dy = _rounded(rng.standard_normal((16, 16))), _rounded(rng.standard_normal((16, 16)))
    gate, up = (_rounded(rng.standard_normal((16, 16)) / 4) for _ in range(2))
    c = rng.integers(-2, 3, (16, 16)).astype(np.float64)

    def fn(x, gate, up, dy, c):
        F.gated_linear(x, gate, up).backward(dy)
        F.sum(gate.float() * c.float()).backward()
        return [x.grad, gate.grad, up.grad]

    arrays = [_bits(v) for v in (x, gate, up, dy, c)]
    with L.config.compiler.patch(fused_operators=fused):
        g = _graph(fn, *arrays, dtypes=["bfloat16"] * 5)
    got = [np.asarray(v, np.float64) for v in oracle.values(g, arrays)]
    want, tol = M.gated(x, gate, up, dy, "silu")[1:], _gated_tolerances(x, gate, up, dy, "silu", "bfloat16")[1:]
    want[1] = want[1] + c
    for v, w, e in zip(got, want, tol):
        assert np.all(np.abs(v - w) <= e + 2.0**-8 * (np.abs(w) + e))


def _gated_twice(activation, tied=False):
    """A program of the gated gradients' own gradients, by x, gate, up and dh (``tied``: gate is the up projection)."""
    def f(x, gate, up):
        return F.gated_linear(x, gate, up, activation=activation)

    def fn(x, gate, up, dh, cx, cg, cu):
        if tied:
            pull = L.vjp(lambda x, w, dh: L.vjp(lambda x, w: f(x, w, w), x, w)[1](dh), x, gate, dh)[1]
            return list(pull((cx, cg)))
        return list(L.vjp(lambda x, gate, up, dh: L.vjp(f, x, gate, up)[1](dh), x, gate, up, dh)[1]((cx, cg, cu)))

    return fn


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("activation", M.ACTIVATIONS)
def test_gated_gradient_of_the_gradient(activation, tied):
    """float64 against central differences of the first gradient's formula (step 1e-6: 1e-9 from its rounding and less from
    its third derivative), and in bfloat16 the same bits fused and not."""
    rng = np.random.default_rng(len(activation) + tied)
    shapes = dict(x=(3, 5), gate=(4, 5), up=(4, 5), dh=(3, 4), cx=(3, 5), cg=(4, 5), cu=(4, 5))
    x = {n: rng.standard_normal(s) for n, s in shapes.items()}
    if tied:
        x["up"] = x["gate"]

    def value(x):
        up = x["gate"] if tied else x["up"]
        grads = M.gated(x["x"], x["gate"], up, x["dh"], activation)[1:]
        if tied:
            grads = [grads[0], grads[1] + grads[2]]
        return sum((g * x[c]).sum() for g, c in zip(grads, ("cx", "cg", "cu")))

    got, _ = _run(_gated_twice(activation, tied), *x.values())
    for name, g in zip(("x", "gate", "dh") if tied else ("x", "gate", "up", "dh"), got):
        assert np.abs(g - M.differences(value, x, name)).max() <= 1e-6, name
    arrays = [_bits(v) for v in x.values()]
    both = []
    for fused in (True, False):
        with L.config.compiler.patch(fused_operators=fused):
            g = _graph(_gated_twice(activation, tied), *arrays, dtypes=["bfloat16"] * 7)
        both.append(oracle.run(g, arrays))
    assert all(np.array_equal(a, b) for a, b in zip(*both))


@pytest.mark.parametrize("weights", [True, False])
def test_heads_gradient_of_the_gradient(weights):
    """float64 against differences of the first gradient's formula; float32 against the
    float64 values to a few hundred roundings of the largest."""
    rng = np.random.default_rng(5)
    x = M.heads_inputs(rng, 1, 3, 2, 1, 8, 6, table=5, dtype="float64", weights=weights, positions=True)
    leaves = [n for n in ("q", "k", "wq", "wk", "gq", "gk") if n in x]
    shapes = [x[n].shape for n in leaves[:-2]]
    cots = {f"c{i}": rng.standard_normal(s) for i, s in enumerate(shapes)}

    def fn(*args):
        t = dict(zip([*x, *cots], args))

        def first(*ls):
            v = {**t, **dict(zip(leaves, ls))}
            f = lambda *h: F.qk_norm_rope(*h[:2], v["cos"], v["sin"], *h[2:], positions=v["positions"], eps=1e-3)  # noqa: E731
            return L.vjp(f, *(v[n] for n in leaves[:-2]))[1]((v["gq"], v["gk"]))

        return list(L.vjp(first, *(t[n] for n in leaves))[1](tuple(t[c] for c in cots)))

    def value(x):
        return sum((g * c).sum() for g, c in zip(M.heads(x, 1e-3, False)[2:], cots.values()))

    got, _ = _run(fn, *x.values(), *cots.values())
    for name, g in zip(leaves, got):
        assert np.abs(g - M.differences(value, x, name)).max() <= 1e-6, name
    single = {n: v if n in ("cos", "sin", "positions") else v.astype(np.float32) for n, v in {**x, **cots}.items()}
    wide = {n: v if n in ("cos", "sin", "positions") else v.astype(np.float64) for n, v in single.items()}
    near, _ = _run(fn, *wide.values())
    for a, b in zip(_run(fn, *single.values())[0], near):
        assert np.abs(a - b).max() <= 2.0**-24 * 400 * max(1.0, np.abs(b).max())


@pytest.mark.parametrize("fused,dtype,d,rot", [(True, "float64", 16, 16), (True, "float64", 10, 6), (True, "bfloat16", 1030, 64),
                                               (False, "bfloat16", 16, 8), (False, "float32", 16, 16)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_heads_that_are_primitives_have_plans(fused, dtype, d, rot, interleaved):
    """A turn reads a head's norm at other elements than its own, which no kernel computes that holds one row's statistics at
    a time: the plan stores them."""
    def both(q, k, cos, sin, wq, wk, gq, gk):
        out, pull = L.vjp(lambda q, k, wq, wk: F.qk_norm_rope(q, k, cos, sin, wq, wk, interleaved=interleaved), q, k, wq, wk)
        return [*out, *pull((gq, gk))]

    q, k, table, w = _m((2, 5, 4, d), dtype), _m((2, 5, 2, d), dtype), _m((9, rot // 2), "float32"), _m((d,), dtype)
    with L.config.compiler.patch(fused_operators=fused):
        for fn, args in ((lambda *a: both(*a)[:2], (q, k, table, table, w, w, q, k)), (both, (q, k, table, table, w, w, q, k))):
            steps = Plan(L.make_graph(fn)(*args), build_kernels=False).steps
            assert not {"heads_fwd", "heads_bwd"} & {st.kind for st in steps}


def test_a_gradient_of_the_gradient_has_a_plan():
    for dtype in ("bfloat16", "float32"):
        x, w, dh = _m((65, 63), dtype), _m((17, 63), dtype), _m((65, 17), dtype)
        assert Plan(L.make_graph(_gated_twice("gelu"))(x, w, w, dh, x, w, w), build_kernels=False).steps


@pytest.mark.parametrize("heads,kv_heads", [(16, 16), (1, 1), (32, 8), (8, 0), (0, 8), ((1 << 20) - 1, (1 << 20) - 1)])
def test_a_launch_of_heads_stays_below_2_to_the_32_threads(heads, kv_heads):
    """Queries and keys go out in one launch of up to 64 lanes a head; the workspace, 2050 rows a launch, says how many
    launches there are."""
    n = C.c_size_t()
    for tokens in (1 << 19, 1 << 21, (1 << 25) + 3, (1 << 29) + 1):
        d = nv.HeadsDesc(batch=1, seq=tokens, heads=heads, kv_heads=kv_heads, head_dim=132, rot=0, table_rows=1, dtype=1)
        nv.call("nhip_qk_norm_rope_workspace", C.byref(d), C.byref(n))
        launches = n.value // (2050 * 132 * 4)
        rows = -(-tokens // launches) * (heads + kv_heads)
        assert rows * 64 + 2 * 256 < 1 << 32 and (launches == 1 or rows > 1 << 24)


def sigmoid_gradient(g, n):
    """Operands whose gate is ``g`` and whose other factors are 1, of ``n`` equal features, and dx: n s(g) s(-g), n s(g)."""
    x = np.stack([g, np.ones_like(g)], 1)
    gate, up = np.tile([1.0, 0.0], (n, 1)), np.tile([0.0, 1.0], (n, 1))
    return x, gate, up, np.ones((len(g), n)), n * np.stack([1 / ((1 + np.exp(-g)) * (1 + np.exp(g))), 1 / (1 + np.exp(-g))], 1)


@pytest.mark.parametrize("dtype,step", [("float32", 2.0**-24), ("bfloat16", 2.0**-8)])
def test_sigmoid_gradient_of_large_gates(dtype, step):
    """s(g) s(-g) relative to itself on both sides: a rounding of dg, one of dx and 16 of 2^-24 between."""
    g = np.concatenate([np.arange(8.0, 20.5, 0.5), -np.arange(8.0, 20.5, 0.5)])
    x, gate, up, dh, want = sigmoid_gradient(g, 1)

    def fn(x, gate, up, dh):
        return list(L.vjp(lambda x: F.gated_linear(x, gate, up, activation="sigmoid"), x)[1](dh))

    arrays = [v.astype(np.float32) if dtype == "float32" else _bits(v) for v in (x, gate, up, dh)]
    (got,) = oracle.values(_graph(fn, *arrays, dtypes=[dtype] * 4), arrays)
    assert np.all(np.abs(np.asarray(got, np.float64) - want) <= (2.01 * step + 16 * 2.0**-24) * want)


def test_gated_launches_stay_below_2_to_the_32_threads():
    """More workgroups than a launch holds are refused before anything is queued; the trace holds primitives well before."""
    def workspace(name, **sizes):
        d = nv.GatedDesc(**{**dict(dtype=1, config=-1, x_m=sizes["k"], w_n=sizes["k"]), **sizes})
        nv.call(name, C.byref(d), C.byref(C.c_size_t()))

    for m, n, config, taken in [(1, (1 << 27) - 32, -1, True), (1, 1 << 27, -1, False), (33, (1 << 28) - 32, 0, True),
                                (33, 1 << 28, 0, False), (70, (1 << 30) - 128, 2, True), (70, 1 << 30, 2, False),
                                (1 << 19, 1 << 19, 1, False), (1 << 30, 1 << 12, 2, False), (1 << 40, 8, -1, False)]:
        if taken:
            workspace("nhip_gated_linear_workspace", m=m, n=n, k=8, config=config)
        else:
            with pytest.raises(RuntimeError, match="2\\^32 threads"):
                workspace("nhip_gated_linear_workspace", m=m, n=n, k=8, config=config)
    for n, fusions in [((1 << 26) - 1, ["gated_linear"]), (1 << 26, [])]:
        g = L.make_graph(F_gated)(_m((1, 8)), _m((n, 8)), _m((n, 8)))
        assert [m.params["name"] for m in g.nodes if m.prim == "fusion"] == fusions


def test_gated_gradients_of_more_tokens_than_the_kernels_take():
    """Tokens whose rows are past 2^31 bytes in each of 64 parts: the gradients' products are primitives, not an error."""
    for t, kinds in ((4088 << 12, {"gated_input", "gated_weight"}), ((4088 << 12) + 1, set())):
        g = L.make_graph(_gated_all)(*(_m(s) for s in ((t, 4100), (8, 4100), (8, 4100), (t, 8))))
        plan = Plan(g, build_kernels=False)
        assert {st.kind for st in plan.steps} & {"gated_input", "gated_weight", "gated_both"} == kinds
    # either side of the border by the library's own word
    for t, n in ((4088 << 12, 8), (1023 << 12, 8192)):  # rows of 4104 and of 2 * 8192 elements
        size = C.c_size_t()
        for more in (0, 1):
            d = nv.GatedDesc(m=t + more, n=n, k=4100, x_m=4100, w_n=4100, dtype=1, config=-1)
            g = L.make_graph(_gated_all)(*(_m(s) for s in ((t + more, 4100), (n, 4100), (n, 4100), (t + more, n))))
            names = [m.params["name"] for m in g.nodes if m.prim == "fusion"]
            assert ("gated_input_grad" in names) == (not more)
            if more:
                with pytest.raises(RuntimeError, match="2\\^31"):
                    nv.call("nhip_gated_backward_workspace", C.byref(d), C.byref(size))
            else:
                nv.call("nhip_gated_backward_workspace", C.byref(d), C.byref(size))


def _gated_all(x, gate, up, dh):
    h, pull = L.vjp(F.gated_linear, x, gate, up)
    return [h, *pull(dh)]
