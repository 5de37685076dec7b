"""packed_attention on the CPU: what it computes (the oracle on its traced body against plain float64 NumPy), its gradients against
differences, what it keeps out, its refusals and the plan it becomes."""

import ctypes as C

import numpy as np
import pytest

import lumen_amd as L
import lumen_amd.functional as F
from lumen_amd import dtypes as D
from lumen_amd import native as nv
from lumen_amd.compiler.plan import Plan
from oracle import oracle
from tests import training_math as M


def _meta(a, dtype=None):
    return L.empty(list(np.shape(a)), dtype or np.asarray(a).dtype.name, "meta")


def _program(causal, scale=None):
    def fn(q, k, v, offsets, do):
        o, pull = L.vjp(lambda q, k, v: F.packed_attention(q, k, v, offsets, scale=scale, is_causal=causal), q, k, v)
        return [o, *pull(do)]

    return fn


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,first,tokens,n,nkv,d,dv,offsets_type", [
    ([3, 0, 5, 1], 1, 12, 4, 2, 8, 8, "int32"), ([7], 0, 7, 2, 2, 6, 3, "int64"), ([], 0, 4, 2, 1, 4, 4, "int32"),
    ([], 2, 4, 1, 1, 4, 4, "int64"), ([1], 0, 1, 1, 1, 1, 1, "int32"), ([0, 0, 2, 0], 0, 2, 3, 1, 5, 2, "int32")])
def test_values_and_gradients(dtype, causal, lengths, first, tokens, n, nkv, d, dv, offsets_type):
    """Tokens of no sequence hold NaN and infinities. float64: the same bounds at its own roundings."""
    rng = np.random.default_rng(tokens)
    offsets = M.offsets_of(lengths, first).astype(offsets_type)
    x = {k: v.astype(dtype) for k, v in M.packed_inputs(rng, tokens, n, nkv, d, dv).items()}
    for v in x.values():
        v[:first], v[offsets[-1]:] = np.nan, np.inf
    scale = 0.7
    g = L.make_graph(_program(causal, scale))(*(_meta(a) for a in (x["q"], x["k"], x["v"], offsets, x["do"])))
    got = oracle.values(g, [x["q"], x["k"], x["v"], offsets, x["do"]])
    want, tol = M.packed(x, offsets, causal, scale)
    for a, w, t in zip(got, want, tol):
        assert a.shape == w.shape and np.all(np.abs(a - w) <= (t if dtype == "float32" else t * 2.0**-28))


@pytest.mark.parametrize("causal", [True, False])
def test_gradient_against_differences(causal):
    """Central differences of step 1e-6: 1e-9 from the third derivative and 1e-10 from the rounding of the values."""
    rng = np.random.default_rng(4)
    offsets = M.offsets_of([3, 4], 1)
    x = M.packed_inputs(rng, 9, 4, 2, 3, 2)
    (_, *grads), _ = M.packed(x, offsets, causal, 0.5)
    for name, g in zip("qkv", grads):
        for at in [tuple(rng.integers(0, s) for s in x[name].shape) for _ in range(12)]:
            v = []
            for sign in (1, -1):
                moved = {**x, name: x[name].copy()}
                moved[name][at] += sign * 1e-6
                v.append((M.packed(moved, offsets, causal, 0.5)[0][0] * x["do"]).sum())
            assert abs((v[0] - v[1]) / 2e-6 - g[at]) <= 1e-7, (name, at)


def test_a_gradient_differentiated_again():
    """The float64 second derivative along a direction against differences of the gradient."""
    rng = np.random.default_rng(5)
    offsets = M.offsets_of([2, 3])
    x = M.packed_inputs(rng, 5, 2, 1, 3)
    u = rng.standard_normal(x["q"].shape)

    def fn(q, k, v, offsets, do, u):
        def dq_along(q):
            _, pull = L.vjp(lambda q: F.packed_attention(q, k, v, offsets), q)
            return F.sum(pull(do)[0] * u)

        return [L.grad(dq_along)(q)]

    args = [x["q"], x["k"], x["v"], offsets, x["do"], u]
    (got,) = oracle.values(L.make_graph(fn)(*(_meta(a) for a in args)), args)
    step = 1e-5
    want = [(M.packed({**x, "q": x["q"] + s * step * u}, offsets, True, 3**-0.5)[0][1]) for s in (1, -1)]
    assert np.abs(got - (want[0] - want[1]) / (2 * step)).max() <= 1e-7


def test_refusals():
    q, k, v, off = (L.empty(s, t, "meta") for s, t in (([6, 4, 8], "float32"), ([6, 2, 8], "float32"), ([6, 2, 8], "float32"), ([3], "int32")))

    def call(q=q, k=k, v=v, off=off, **kw):
        L.make_graph(lambda *xs: F.packed_attention(*xs, **kw))(q, k, v, off)

    def shaped(*s, dtype="float32"):
        return L.empty(list(s), dtype, "meta")

    call()
    for kw in (dict(q=shaped(6, 32)), dict(k=shaped(5, 2, 8)), dict(k=shaped(6, 1, 8)), dict(k=shaped(6, 2, 4), v=shaped(6, 2, 4)),
               dict(k=shaped(6, 3, 8), v=shaped(6, 3, 8)), dict(k=shaped(6, 0, 8), v=shaped(6, 0, 8)), dict(off=shaped(3)),
               dict(off=shaped(3, 1, dtype="int32")), dict(off=shaped(0, dtype="int32")), dict(scale=0.0), dict(scale=-1.0),
               dict(scale=float("nan")), dict(scale=True), dict(is_causal=1), dict(v=shaped(6, 2, 0))):
        with pytest.raises(ValueError, match="packed_attention"):
            call(**kw)
    with pytest.raises(TypeError):
        call(k=shaped(6, 2, 8, dtype="bfloat16"))
    with pytest.raises(TypeError):
        call(q=shaped(6, 4, 8, dtype="int32"), k=shaped(6, 2, 8, dtype="int32"), v=shaped(6, 2, 8, dtype="int32"))


def _graph(t, n, nkv, d, sequences, dtype="bfloat16", program=None):
    metas = [L.empty(s, dtype, "meta") for s in ([t, n, d], [t, nkv, d], [t, nkv, d])]
    return L.make_graph(program or _program(True))(*metas, L.empty([sequences + 1], "int32", "meta"), L.empty([t, n, d], dtype, "meta"))


def test_plans():
    kinds = [st.kind for st in Plan(_graph(300, 8, 2, 64, 4), build_kernels=False).steps]
    assert kinds == ["packed_fwd", "packed_bwd"]
    for d, dtype in ((60, "bfloat16"), (136, "bfloat16"), (64, "float32")):
        g = _graph(20, 2, 2, d, 2, dtype)
        assert not [n for n in g.nodes if n.prim == "fusion"], (d, dtype)
    with L.config.compiler.patch(fused_operators=False):
        assert not [n for n in _graph(20, 2, 2, 64, 2).nodes if n.prim == "fusion"]

    def only_values(q, k, v, offsets, do):
        return [L.vjp(lambda v: F.packed_attention(q, k, v, offsets), v)[1](do)[0]]

    plan = Plan(_graph(300, 8, 2, 64, 4, program=only_values), build_kernels=False)
    assert [st.kind for st in plan.steps] == ["packed_fwd", "packed_bwd"]
    stored = plan.workspace_bytes
    with L.config.compiler.patch(attention_store_ds=False):
        assert Plan(_graph(300, 8, 2, 64, 4, program=only_values), build_kernels=False).workspace_bytes < stored


def _desc(**kw):
    d = nv.PackedDesc(tokens=100, sequences=3, heads=4, kv_heads=2, head_dim=64, dtype=1, offsets_dtype=1, scale=1.0)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_workspace_and_its_refusals():
    n = C.c_size_t()
    nv.call("nhip_packed_workspace", C.byref(_desc()), 0, C.byref(n))
    assert n.value >= 16 * (100 // 128 + 3 + 2)
    for kw in (dict(tokens=-1), dict(head_dim=60), dict(head_dim=136), dict(value_head_dim=4), dict(dtype=0), dict(kv_heads=3),
               dict(kv_heads=0), dict(offsets_dtype=0), dict(scale=0.0), dict(scale=float("nan")), dict(q_s=4), dict(dv_n=12),
               dict(tokens=(1 << 26) + 1), dict(sequences=(1 << 20) + 1), dict(tokens=1 << 26, sequences=1, heads=16, kv_heads=16),
               dict(tokens=1 << 24, head_dim=40, q_s=1 << 10)):
        with pytest.raises(RuntimeError, match="nhip_packed_workspace"):
            nv.call("nhip_packed_workspace", C.byref(_desc(**kw)), 1, C.byref(n))


def test_tables_and_stored_ds_hold_whatever_the_offsets_are():
    """The bounds that size the tables and dS, restated: blocks of every sequence, of the tokens before and behind them; tiles of 128
    keys and 64 queries."""
    rng = np.random.default_rng(0)
    for _ in range(400):
        tokens, count = int(rng.integers(1, 3000)), int(rng.integers(0, 40))
        cuts = np.sort(rng.integers(0, tokens + 1, count + 1))
        lengths = np.diff(cuts)
        for block in (64, 128, 256):
            used = sum(-(-x // block) for x in [*lengths, cuts[0], tokens - cuts[-1]])
            assert used <= tokens // block + min(count, tokens) + 2
        ds = sum(-(-x // 128) * -(-x // 64) for x in lengths)
        assert ds <= tokens * tokens // 8192 + 3 * tokens // 128 + 1 + min(count, tokens)


def _lowered(program, *metas):
    """``(step kind, PackedDesc, [(pointer slot, place)])`` of each packed step of the program's plan, as the library takes it: the
    descriptor passes the checks that the launches make."""
    from lumen_amd.compiler import operators

    plan = Plan(L.make_graph(program)(*metas), build_kernels=False)
    out = []
    for st in plan.steps:
        if st.kind in ("packed_fwd", "packed_bwd"):
            _, raw, places = operators.lower(plan, st)
            desc, n = nv.PackedDesc.from_buffer_copy(raw), C.c_size_t()
            nv.call("nhip_packed_workspace", C.byref(desc), int(st.kind == "packed_bwd"), C.byref(n))
            out.append((st.kind, desc, places))
    assert out
    return out


UNIT_AXES = {  # a view's shape -> the operand [T, N, 64], whose axes of one element have odd strides
    "a head of two": ([40, 2, 68], lambda x: x[:, 0:1, :64]),
    "a token": ([1, 1, 100], lambda x: x[:, :, :64]),
    "a token of three heads": ([1, 4, 72], lambda x: x[:, :3, :64]),
    "a head by a permutation": ([100 * 64], lambda x: x.reshape(100, 64, 1).permute(0, 2, 1)),
}


@pytest.mark.parametrize("what", UNIT_AXES)
def test_axes_of_one_element_have_any_stride(what):
    shape, view = UNIT_AXES[what]

    def both(q, k, v, offsets, do):
        return _program(True)(view(q), view(k), view(v), offsets, view(do))

    x = L.empty(shape, "bfloat16", "meta")
    for _, desc, places in _lowered(both, x, x, x, L.empty([3], "int32", "meta"), x):
        assert [loc.base[0] for _, loc in places][:3] == ["in"] * 3  # read where they lie
        for name in ("q", "k", "v", "o"):
            assert getattr(desc, f"{name}_s") == 0 or desc.tokens > 1
            assert getattr(desc, f"{name}_n") == 0 or desc.heads > 1


@pytest.mark.parametrize("scale,kernel", [(1e-50, False), (1e-46, False), (2.0**-149, True), (1e-30, True), (3.4e38, True), (3.402e38, False), (1e300, False)])
def test_scales_past_the_kernels_float32(scale, kernel):
    """A positive number is a scale; the library takes those that are one in float32 too."""
    def fn(q, k, v, offsets, do):
        o, pull = L.vjp(lambda q, k, v: F.packed_attention(q, k, v, offsets, scale=scale), q, k, v)
        return [o, *pull(do)]

    kinds = [st.kind for st in Plan(_graph(20, 2, 2, 64, 2, program=fn), build_kernels=False).steps]
    assert (kinds == ["packed_fwd", "packed_bwd"]) == kernel


def test_a_scale_that_float32_rounds_to_zero():
    """Scores of zero: the mean of the values seen."""
    rng = np.random.default_rng(8)
    offsets = M.offsets_of([2, 3])
    x = {k: v.astype(np.float32) for k, v in M.packed_inputs(rng, 5, 2, 1, 8).items()}
    bits = {k: D.bf16_bits(v) for k, v in x.items()}
    g = L.make_graph(lambda q, k, v, o: [F.packed_attention(q, k, v, o, scale=1e-50)])(
        *(_meta(bits[k], "bfloat16") for k in "qkv"), _meta(offsets))
    (got,) = oracle.values(g, [bits["q"], bits["k"], bits["v"], offsets])
    real = {k: D.bf16_to_f32(b).astype(np.float64) for k, b in bits.items()}
    (want, *_), (tol, *_) = M.packed(real, offsets, True, 1e-50, "bfloat16")
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("dtype,tokens,n,nkv,d", [("float32", 0, 2, 1, 8), ("float32", 5, 0, 2, 8), ("bfloat16", 0, 2, 2, 60), ("bfloat16", 5, 0, 2, 60),
                                                  ("bfloat16", 5, 0, 2, 64)])
def test_plans_without_tokens_or_query_heads(dtype, tokens, n, nkv, d):
    kinds = [st.kind for st in Plan(_graph(tokens, n, nkv, d, 2, dtype), build_kernels=False).steps]
    assert ("packed_bwd" in kinds) == (d == 64)
