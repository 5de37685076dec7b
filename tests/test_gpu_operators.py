"""qk_norm_rope, gated_linear and clip_grad_norm on the GPU against plain float64 NumPy (tests/operator_math.py).

Tolerances: a result's one rounding, half a step of its dtype (U), plus what float32 arithmetic can be off by, as a count
of roundings times 2^-24 times the sum of the magnitudes that were added."""

import ctypes as C

import numpy as np
import pytest

import lumen_amd as L
import lumen_amd.functional as F
from lumen_amd import dtypes as D
from lumen_amd import native as nv
from lumen_amd.compiler.plan import Plan
from lumen_amd.nn import Module
from lumen_amd.tensor import DeviceBuffer
from tests import operator_math as M
from tests.hiputil import Dev
from tests.stepcheck import check_steps

pytestmark = pytest.mark.gpu

U = {"float32": 2.0**-24, "bfloat16": 2.0**-8, "float16": 2.0**-11}
F32 = 2.0**-24


def _round(x, dtype):
    """float64 values as ``dtype``'s, in float64."""
    return np.asarray(D.to_numpy_values(D.from_values(np.asarray(x, np.float32), dtype), dtype), np.float64)


def _tensor(x, dtype):
    return L.Tensor(dtype, np.shape(x), "cpu", host=np.array(D.from_values(np.asarray(x, np.float32), dtype)))


def _values(t):
    return np.asarray(L.to_numpy(t), np.float64)


def _near(got, want, tol, what=""):
    assert got.shape == want.shape, what
    bad = ~(np.abs(got - want) <= tol) & ~(np.isnan(got) & np.isnan(want))
    assert not bad.any(), (what, np.abs(got - want)[bad].max(), int(bad.sum()), np.argwhere(bad)[0])


# ---- heads


def _heads_case(seed, b, s, n, nkv, d, rot, dtype, interleaved=False, weights=True, positions=True, table=64):
    rng = np.random.default_rng(seed)
    x = M.heads_inputs(rng, b, s, n, nkv, d, rot, table, weights=weights, positions=positions)
    return {k: v if k in ("cos", "sin", "positions") else _round(v, dtype) for k, v in x.items()}


def _heads_program(names, interleaved, eps):
    def fn(*args):
        t = dict(zip(names, args))
        keep = [m for m in ("q", "k", "wq", "wk") if m in t]

        def f(*leaves):
            v = {**t, **dict(zip(keep, leaves))}
            return F.qk_norm_rope(v["q"], v["k"], v["cos"], v["sin"], v.get("wq"), v.get("wk"),
                                  positions=v.get("positions"), eps=eps, interleaved=interleaved)

        out, pull = L.vjp(f, *(t[m] for m in keep))
        return [*out, *pull((t["gq"], t["gk"]))]

    return fn


def _heads_check(got, x, dtype, eps, interleaved, what=""):
    d = x["q"].shape[3]
    want = M.heads(x, eps, interleaved)
    for i, (a, w) in enumerate(zip(got, want)):
        if i < 4:  # a head: its row's sums of D, about 40 roundings more, of values to 8 times the largest result
            tol = U[dtype] * np.abs(w) + F32 * (d + 40) * 8 * np.abs(w).max(initial=0)
        else:  # a weight's gradient: a sum over every row
            rows = np.prod(x["q" if i == 4 else "k"].shape[:3])
            tol = U[dtype] * np.abs(w) + F32 * (rows + d + 40) * 4 * rows
        _near(a, w, tol, (what, i))


HEADS = [
    # b, s, n, nkv, d, rot, dtype, interleaved, weights, positions
    (16, 1, 16, 16, 128, 128, "bfloat16", False, True, True),
    (2, 37, 16, 4, 64, 32, "float16", True, True, True),
    (1, 200, 16, 16, 128, 128, "bfloat16", False, True, False),
    (3, 33, 6, 2, 80, 40, "float32", False, True, True),
    (1, 1, 1, 1, 8, 8, "bfloat16", False, True, True),
    (2, 19, 3, 1, 36, 18, "bfloat16", True, True, True),
    (2, 19, 3, 3, 36, 36, "float16", False, False, True),
    (1, 9, 2, 1, 7, 2, "bfloat16", False, True, False),
    (1, 5, 2, 1, 1, 0, "float32", False, True, False),
    (2, 40, 8, 2, 96, 48, "bfloat16", False, True, True),
    (1, 30, 4, 4, 256, 256, "float16", True, True, True),
    (1, 6, 2, 2, 1024, 512, "bfloat16", False, True, True),
    (1, 6, 2, 1, 1024, 1024, "float32", True, True, True),
    (1, 3, 2, 1, 1023, 510, "float32", False, True, True),
    (4, 300, 32, 8, 64, 64, "bfloat16", False, False, True),
    (2, 17, 5, 5, 24, 8, "bfloat16", False, True, True),
    (2, 64, 16, 16, 128, 0, "bfloat16", False, True, False),
]


@pytest.mark.parametrize("case", range(len(HEADS)))
def test_heads(hip, case):
    b, s, n, nkv, d, rot, dtype, interleaved, weights, positions = HEADS[case]
    x = _heads_case(case, b, s, n, nkv, d, rot, dtype, interleaved, weights, positions, table=max(64, s))
    f = L.compile(_heads_program(list(x), interleaved, 1e-3), device="hip")
    args = [L.from_numpy(v) if k in ("cos", "sin", "positions") else _tensor(v, dtype) for k, v in x.items()]
    for _ in range(2):
        got = [_values(t) for t in f(*args)]
        _heads_check(got, x, dtype, 1e-3, interleaved)
    assert sorted(st.kind for st in f.plan.steps) == ["heads_bwd", "heads_fwd"]


def test_heads_of_a_merged_projection_in_int64_positions_out_of_the_table(hip):
    """Heads read through the strides of a merged projection; positions below 0 and past the tables are clamped."""
    b, s, n, nkv, d = 2, 21, 4, 2, 64
    rng = np.random.default_rng(1)
    qkv = _round(rng.standard_normal((b, s, (n + 2 * nkv) * d)), "bfloat16")
    x = _heads_case(2, b, s, n, nkv, d, 32, "bfloat16")
    x["q"], x["k"] = qkv[:, :, :n * d].reshape(b, s, n, d), qkv[:, :, n * d:(n + nkv) * d].reshape(b, s, nkv, d)
    pos = rng.integers(-5, 80, (b, s)).astype(np.int64)
    pos[0, :3] = [-2**40, 2**40, 63]

    def fn(qkv, cos, sin, wq, wk, pos):
        q, k = qkv[:, :, :n * d].reshape(b, s, n, d), qkv[:, :, n * d:(n + nkv) * d].reshape(b, s, nkv, d)
        return list(F.qk_norm_rope(q, k, cos, sin, wq, wk, positions=pos, eps=1e-3))

    f = L.compile(fn, device="hip")
    got = [_values(t) for t in f(_tensor(qkv, "bfloat16"), L.from_numpy(x["cos"]), L.from_numpy(x["sin"]),
                                 _tensor(x["wq"], "bfloat16"), _tensor(x["wk"], "bfloat16"), L.from_numpy(pos))]
    assert "loop" not in [st.kind for st in f.plan.steps]
    _heads_check(got, {**x, "positions": pos}, "bfloat16", 1e-3, False)


def test_heads_default_eps_and_rows_that_are_zero_or_not_finite(hip):
    """A row of zeros stays zeros; a NaN or an infinity reaches its own row alone, in both directions."""
    x = _heads_case(4, 1, 12, 2, 1, 64, 64, "bfloat16", positions=False)
    x["q"][0, 3] = 0
    x["q"][0, 5, 1, 7] = np.nan
    x["k"][0, 6, 0, 0] = np.inf
    f = L.compile(_heads_program(list(x), False, None), device="hip")
    got = [_values(t) for t in f(*[L.from_numpy(v) if k in ("cos", "sin") else _tensor(v, "bfloat16") for k, v in x.items()])]
    with np.errstate(invalid="ignore"):
        want = M.heads(x, 2.0**-7, False)
    assert np.all(got[0][0, 3] == 0)
    for a, w, bad in ((got[0], want[0], (0, 5, 1)), (got[2], want[2], (0, 5, 1)), (got[1], want[1], (0, 6, 0)),
                      (got[3], want[3], (0, 6, 0))):
        assert np.isnan(a[bad]).any()
        rest = np.ones(a.shape[:3], bool)
        rest[bad] = False
        _near(a[rest], w[rest], U["bfloat16"] * np.abs(w[rest]) + F32 * 200 * 8 * np.abs(w[rest]).max())
    assert np.isnan(got[4]).any() and np.isnan(got[5]).any()


def test_heads_gradient_of_a_weight_alone_and_of_keys_alone(hip):
    """What nothing differentiates is neither computed nor written: the keys' weight alone, then the keys alone."""
    x = _heads_case(6, 2, 10, 4, 2, 64, 64, "bfloat16", positions=False)
    want = M.heads(x, 1e-3, False)
    args = [L.from_numpy(v) if k in ("cos", "sin") else _tensor(v, "bfloat16") for k, v in x.items()]

    def by(which):
        def fn(q, k, cos, sin, wq, wk, gq, gk):
            leaf = {"wk": wk, "k": k}[which]

            def f(leaf):
                v = {"wk": wk, "k": k, which: leaf}
                return F.qk_norm_rope(q, v["k"], cos, sin, wq, v["wk"], eps=1e-3)

            return list(L.vjp(f, leaf)[1]((gq, gk)))

        return _values(L.compile(fn, device="hip")(*args)[0])

    rows = 2 * 10 * 2
    _near(by("wk"), want[5], U["bfloat16"] * np.abs(want[5]) + F32 * (rows + 104) * 4 * rows)
    _near(by("k"), want[3], U["bfloat16"] * np.abs(want[3]) + F32 * 104 * 8 * np.abs(want[3]).max())


def test_heads_of_no_tokens(hip):
    """An empty batch: no rows, and weight gradients of zeros."""
    x = _heads_case(7, 0, 5, 2, 1, 64, 64, "bfloat16", positions=False)
    f = L.compile(_heads_program(list(x), False, 1e-3), device="hip")
    out = f(*[L.from_numpy(v) if k in ("cos", "sin") else _tensor(v, "bfloat16") for k, v in x.items()])
    assert out[0].shape == (0, 5, 2, 64) and not _values(out[4]).any() and not _values(out[5]).any()


def test_heads_past_32_bit_offsets(hip):
    """Batches 2^31 + 64 elements apart, through the ABI, on the vector and the general kernel."""
    for d in (64, 36):
        far = (1 << 31) + 64
        x = _heads_case(9, 2, 1, 1, 1, d, d, "bfloat16", weights=False)
        q = Dev(nbytes=2 * (far + 64))
        cos, sin, pos = Dev(x["cos"]), Dev(x["sin"]), Dev(x["positions"])
        k, ok, oq = Dev(D.from_values(np.asarray(x["k"], np.float32), "bfloat16")), Dev(nbytes=4 * d), Dev(nbytes=4 * d)
        host = np.ascontiguousarray(D.from_values(np.asarray(x["q"], np.float32), "bfloat16"))
        for i in range(2):
            nv.h2d(q.ptr + 2 * far * i, host[i].ctypes.data, 2 * d)
        desc = nv.HeadsDesc(batch=2, seq=1, heads=1, kv_heads=1, head_dim=d, rot=d, table_rows=64, dtype=1, positions=1, eps=1e-3)
        desc.q_b, desc.q_s, desc.q_n = far, d, d
        for t in ("k", "oq", "ok"):
            setattr(desc, f"{t}_b", d), setattr(desc, f"{t}_s", d), setattr(desc, f"{t}_n", d)
        nv.call("nhip_qk_norm_rope", C.byref(desc), q.ptr, k.ptr, None, None, cos.ptr, sin.ptr, pos.ptr, oq.ptr, ok.ptr)
        got = D.to_numpy_values(oq.get((2, 1, 1, d), np.uint16), "bfloat16").astype(np.float64)
        want = M.heads(x, 1e-3, False)[0]
        _near(got, want, U["bfloat16"] * np.abs(want) + F32 * 8 * (d + 40) * np.abs(want).max())


def test_heads_write_nothing_past_their_rows(hip):
    """Rows behind the last token of the output stay as they were (odd row counts on both kernels, both directions)."""
    for d in (64, 36):
        x = _heads_case(11, 1, 5, 3, 1, d, d, "bfloat16", positions=False)
        bits = {m: np.ascontiguousarray(D.from_values(np.asarray(x[m], np.float32), "bfloat16")) for m in ("q", "k", "gq", "gk", "wq", "wk")}
        dev = {m: Dev(v) for m, v in bits.items()}
        cos, sin = Dev(x["cos"]), Dev(x["sin"])
        desc = nv.HeadsDesc(batch=1, seq=5, heads=3, kv_heads=1, head_dim=d, rot=d, table_rows=64, dtype=1, eps=1e-3)
        for t, heads in (("q", 3), ("k", 1), ("oq", 3), ("ok", 1), ("dq", 3), ("dk", 1)):
            setattr(desc, f"{t}_b", 5 * heads * d), setattr(desc, f"{t}_s", heads * d), setattr(desc, f"{t}_n", d)
        fence = np.full(15 * d + 512, 0x4242, np.uint16)
        outs = {m: Dev(fence) for m in ("oq", "ok", "dq", "dk", "dwq", "dwk")}
        n = C.c_size_t()
        nv.call("nhip_qk_norm_rope_workspace", C.byref(desc), C.byref(n))
        ws = Dev(nbytes=n.value)
        head = [dev["q"].ptr, dev["k"].ptr, dev["wq"].ptr, dev["wk"].ptr, cos.ptr, sin.ptr, None]
        nv.call("nhip_qk_norm_rope", C.byref(desc), *head, outs["oq"].ptr, outs["ok"].ptr)
        nv.call("nhip_qk_norm_rope_bwd", C.byref(desc), *head, dev["gq"].ptr, dev["gk"].ptr, outs["dq"].ptr, outs["dk"].ptr,
                outs["dwq"].ptr, outs["dwk"].ptr, ws.ptr)
        for m, size in (("oq", 15 * d), ("ok", 5 * d), ("dq", 15 * d), ("dk", 5 * d), ("dwq", d), ("dwk", d)):
            got = outs[m].get(fence.shape, np.uint16)
            assert np.all(got[size:] == 0x4242) and not np.all(got[:size] == 0x4242), (d, m)


# ---- gated projections


def _gated_case(seed, t, k, n, dtype):
    rng = np.random.default_rng(seed)
    return (_round(rng.standard_normal((t, k)), dtype), _round(rng.standard_normal((n, k)) / np.sqrt(max(k, 1)), dtype),
            _round(rng.standard_normal((n, k)) / np.sqrt(max(k, 1)), dtype), _round(rng.standard_normal((t, n)), dtype))


def _gated_tolerances(x, gate, up, dh, activation, dtype):
    """What [h, dx, dgate, dup] may be off by: the float32 products g and u by (K + 16) roundings of the sums of their
    terms' magnitudes, dg and du by their own rounding and what that makes of them (|act'| <= 1.2, |act''| <= 1.3), the
    gradients by those times the other operand and by their own sums' roundings."""
    t, k, n = x.shape[0], x.shape[1], gate.shape[0]
    e = F32 * (k + 16)
    g, u = x @ gate.T, x @ up.T
    eg, eu = e * (np.abs(x) @ np.abs(gate).T), e * (np.abs(x) @ np.abs(up).T)
    a, da = M.activation(activation, g)
    few = 32 * F32
    h = a * u
    th = U[dtype] * np.abs(h) + (1.2 * eg + few * np.abs(a)) * np.abs(u) + np.abs(a) * eu
    dg, du = dh * u * da, dh * a
    if activation == "relu":  # where the sum's sign may differ, the derivative may be either
        da_off = np.where(np.abs(g) <= eg, 1.0, 0.0)
    else:
        da_off = 1.3 * eg
    few_g = few * (1 + np.abs(g))
    tdg = U[dtype] * np.abs(dg) + np.abs(dh) * (eu * np.abs(da) + np.abs(u) * (da_off + few_g))
    tdu = U[dtype] * np.abs(du) + np.abs(dh) * (1.2 * eg + few * np.abs(a))
    mags = np.abs(dg) @ np.abs(gate) + np.abs(du) @ np.abs(up)
    dx = dg @ gate + du @ up
    tdx = U[dtype] * np.abs(dx) + tdg @ np.abs(gate) + tdu @ np.abs(up) + F32 * (2 * n + 16) * mags
    out = [th, tdx]
    for d, td in ((dg, tdg), (du, tdu)):
        w = d.T @ x
        out.append(U[dtype] * np.abs(w) + td.T @ np.abs(x) + F32 * (t + 16) * (np.abs(d).T @ np.abs(x)))
    return [1.05 * v + 1e-30 for v in out]


GATED = [
    # tokens, K, F, activation, dtype
    (1, 512, 256, "silu", "bfloat16"),
    (16, 256, 512, "gelu", "bfloat16"),
    (17, 264, 72, "silu", "float16"),
    (33, 64, 96, "relu", "bfloat16"),
    (64, 128, 16, "sigmoid", "float16"),
    (65, 192, 320, "silu", "bfloat16"),
    (300, 128, 200, "gelu", "float16"),
    (520, 64, 1032, "silu", "bfloat16"),
    (129, 100, 65, "silu", "bfloat16"),
    (5, 7, 3, "gelu", "float16"),
    (1, 1, 1, "silu", "bfloat16"),
    (70, 515, 131, "relu", "float16"),
    (128, 64, 128, "silu", "bfloat16"),
    (1000, 32, 36, "gelu", "bfloat16"),
    (90, 1024, 48, "silu", "bfloat16"),
]


def _gated_program(activation):
    def fn(x, gate, up, dh):
        h, pull = L.vjp(lambda x, gate, up: F.gated_linear(x, gate, up, activation=activation), x, gate, up)
        return [h, *pull(dh)]

    return fn


@pytest.mark.parametrize("case", range(len(GATED)))
def test_gated(hip, case):
    t, k, n, activation, dtype = GATED[case]
    x = _gated_case(case, t, k, n, dtype)
    f = L.compile(_gated_program(activation), device="hip")
    got = f(*[_tensor(v, dtype) for v in x])
    for i, (a, w, tol) in enumerate(zip(got, M.gated(*x, activation), _gated_tolerances(*x, activation, dtype))):
        _near(_values(a), w, tol, i)


def _gated_abi(x, gate, up, dtype, activation, config, save, fence=64):
    """nhip_gated_linear through the ABI: (h with ``fence`` elements behind it, g, u)."""
    t, k, n = x.shape[0], x.shape[1], gate.shape[0]
    dx, dg, du = (Dev(np.ascontiguousarray(D.from_values(np.asarray(v, np.float32), dtype))) for v in (x, gate, up))
    h = Dev(np.full(t * n + fence, 0x4242, np.uint16))
    g, u = (Dev(np.full(t * n + fence, 77.0, np.float32)) for _ in range(2))
    desc = nv.GatedDesc(m=t, n=n, k=k, x_m=k, w_n=k, h_m=n, config=config)
    desc.dtype, desc.activation = {"bfloat16": 1, "float16": 2}[dtype], nv.NHIP_ACT[activation]
    size = C.c_size_t()
    nv.call("nhip_gated_linear_workspace", C.byref(desc), C.byref(size))
    ws = Dev(nbytes=size.value)
    nv.call("nhip_gated_linear", C.byref(desc), dx.ptr, dg.ptr, du.ptr, h.ptr, g.ptr if save else None, u.ptr if save else None,
            ws.ptr if size.value else None)
    return h.get((t * n + fence,), np.uint16), g.get((t * n + fence,), np.float32), u.get((t * n + fence,), np.float32)


@pytest.mark.parametrize("t,k,n", [(1, 64, 16), (64, 192, 136), (256, 64, 128), (257, 128, 129), (300, 320, 260), (130, 72, 65),
                                   (61, 515, 70), (290, 131, 64), (2, 3, 5)])
@pytest.mark.parametrize("save", [False, True])
def test_every_gated_kernel(hip, t, k, n, save):
    """Each kernel that takes the shape, by its config: h, g and u, and nothing behind them."""
    x, gate, up, dh = _gated_case(t + n, t, k, n, "bfloat16")
    tol = _gated_tolerances(x, gate, up, dh, "silu", "bfloat16")[0]
    e = F32 * (k + 16)
    count = C.c_int()
    nv.call("nhip_gated_config_count", C.byref(count))
    ran = 0
    for config in range(count.value):
        try:
            h, g, u = _gated_abi(x, gate, up, "bfloat16", "silu", config, save)
        except RuntimeError as err:
            assert "does not take these operands" in str(err) and config == 0 and t > 64
            continue
        ran += 1
        a, _ = M.activation("silu", x @ gate.T)
        got = D.to_numpy_values(h[:t * n], "bfloat16").astype(np.float64).reshape(t, n)
        _near(got, a * (x @ up.T), tol, config)
        assert np.all(h[t * n:] == 0x4242), config
        for s, w in ((g, gate), (u, up)):
            if save:
                _near(s[:t * n].astype(np.float64).reshape(t, n), x @ w.T, e * (np.abs(x) @ np.abs(w).T), config)
            assert np.all(s[t * n if save else 0:] == 77.0), config
    assert ran >= 3
    with pytest.raises(RuntimeError, match="does not take these operands"):
        _gated_abi(x, gate, up, "bfloat16", "silu", count.value, save)


def test_gated_of_three_axes_strided_rows_and_no_features(hip):
    """Rows [B, S, K] that are a slice of wider ones (read in place), and sums over no features: act(0) * 0."""
    rng = np.random.default_rng(3)
    wide = _round(rng.standard_normal((2, 5, 192)), "bfloat16")
    _, gate, up, _ = _gated_case(4, 1, 128, 96, "bfloat16")
    f = L.compile(lambda x, gate, up: [F.gated_linear(x[:, :, 64:], gate, up)], device="hip")
    got = _values(f(_tensor(wide, "bfloat16"), _tensor(gate, "bfloat16"), _tensor(up, "bfloat16"))[0])
    rows = wide[:, :, 64:].reshape(10, 128)
    want = M.gated(rows, gate, up, np.zeros((10, 96)), "silu")[0].reshape(2, 5, 96)
    tol = _gated_tolerances(rows, gate, up, np.zeros((10, 96)), "silu", "bfloat16")[0].reshape(2, 5, 96)
    _near(got, want, tol)
    empty = L.compile(lambda x, gate, up: [F.gated_linear(x, gate, up)], device="hip")
    out = empty(*(_tensor(np.zeros(s), "bfloat16") for s in ((3, 0), (4, 0), (4, 0))))[0]
    assert out.shape == (3, 4) and not _values(out).any()


def test_gated_of_values_that_are_not_finite(hip):
    """A NaN or infinite row of x reaches its own row of h alone."""
    x, gate, up, _ = _gated_case(5, 40, 64, 48, "bfloat16")
    want = M.gated(x, gate, up, np.zeros((40, 48)), "silu")[0]
    tol = _gated_tolerances(x, gate, up, np.zeros((40, 48)), "silu", "bfloat16")[0]
    x[3, 5], x[8, 0] = np.nan, np.inf
    for config in (0, 1, 2, 3):
        h = _gated_abi(x, gate, up, "bfloat16", "silu", config, False)[0][:40 * 48]
        got = D.to_numpy_values(h, "bfloat16").astype(np.float64).reshape(40, 48)
        rest = [i for i in range(40) if i not in (3, 8)]
        assert np.isnan(got[3]).all() and not np.isfinite(got[8]).all()
        _near(got[rest], want[rest], tol[rest], config)


def test_gated_past_32_bit_offsets(hip):
    """Rows of x 2^30 + 64 elements apart: the third is past 2^31. Through the workspace, except the few-row kernel."""
    far = (1 << 30) + 64
    x, gate, up, _ = _gated_case(6, 3, 64, 32, "bfloat16")
    buf = Dev(nbytes=2 * (2 * far + 64))
    host = np.ascontiguousarray(D.from_values(np.asarray(x, np.float32), "bfloat16"))
    for i in range(3):
        nv.h2d(buf.ptr + 2 * far * i, host[i].ctypes.data, 128)
    dg, du = (Dev(np.ascontiguousarray(D.from_values(np.asarray(v, np.float32), "bfloat16"))) for v in (gate, up))
    h = Dev(nbytes=2 * 3 * 32)
    want = M.gated(x, gate, up, np.zeros((3, 32)), "silu")[0]
    tol = _gated_tolerances(x, gate, up, np.zeros((3, 32)), "silu", "bfloat16")[0]
    ws = Dev(nbytes=2 * 64 * (3 + 2 * 32))
    for config in (0, 1, 2, 3):
        desc = nv.GatedDesc(m=3, n=32, k=64, x_m=far, w_n=64, h_m=32, dtype=1, activation=0, config=config)
        size = C.c_size_t()
        nv.call("nhip_gated_linear_workspace", C.byref(desc), C.byref(size))
        assert size.value == (ws.nbytes if config else 0)
        nv.call("nhip_gated_linear", C.byref(desc), buf.ptr, dg.ptr, du.ptr, h.ptr, None, None, ws.ptr)
        _near(D.to_numpy_values(h.get((3, 32), np.uint16), "bfloat16").astype(np.float64), want, tol, config)


@pytest.mark.parametrize("t,k,n,dtype", [(1, 8, 8, "bfloat16"), (130, 64, 64, "float16"), (257, 136, 72, "bfloat16"),
                                         (40, 520, 1416, "float16"), (512, 264, 4096, "bfloat16"), (300, 72, 2056, "bfloat16"),
                                         (929, 167, 333, "bfloat16"), (3000, 65, 130, "float16"), (7, 1, 1, "bfloat16")])
def test_gated_backward_kernels(hip, t, k, n, dtype):
    """dx, d_gate and d_up of [dg | du] through the ABI: whole and in parts, sizes that end inside a tile of k or a chunk,
    one row that is not finite, a d_up left out, and nothing written behind a result."""
    rng = np.random.default_rng(t)
    whole = -(-n // 8) * 8
    x, gate, up, _ = _gated_case(t + k, t, k, n, dtype)
    dg, du = (_round(rng.standard_normal((t, n)), dtype) for _ in range(2))
    dgu = np.zeros((t, 2 * whole))
    dgu[:, :n], dgu[:, whole:whole + n] = dg, du
    bad = dgu.copy()
    bad[t // 2, whole] = np.inf
    bits = lambda v: np.ascontiguousarray(D.from_values(np.asarray(v, np.float32), dtype))  # noqa: E731
    ddgu, dbad, dx_, dgate, dup = (Dev(bits(v)) for v in (dgu, bad, x, gate, up))
    desc = nv.GatedDesc(m=t, n=n, k=k, x_m=k, w_n=k, dtype={"bfloat16": 1, "float16": 2}[dtype], config=-1)
    size = C.c_size_t()
    nv.call("nhip_gated_backward_workspace", C.byref(desc), C.byref(size))
    ws = Dev(nbytes=size.value)

    def outputs(count, rows):
        return [Dev(np.full(rows * k + 64, 0x4242, np.uint16)) for _ in range(count)]

    def values(dev, rows):
        raw = dev.get((rows * k + 64,), np.uint16)
        assert np.all(raw[rows * k:] == 0x4242)
        return D.to_numpy_values(raw[:rows * k].view(D.storage(dtype)), dtype).astype(np.float64).reshape(rows, k)

    for a in (ddgu, dbad):
        (out,) = outputs(1, t)
        nv.call("nhip_gated_input_grad", C.byref(desc), a.ptr, dgate.ptr, dup.ptr, out.ptr, ws.ptr if size.value else None)
        got, want = values(out, t), dg @ gate + du @ up
        rows = [i for i in range(t) if a is ddgu or i != t // 2]
        mags = np.abs(dg) @ np.abs(gate) + np.abs(du) @ np.abs(up)
        _near(got[rows], want[rows], (U[dtype] * np.abs(want) + F32 * (2 * n + 16) * mags)[rows], "dx")
    for with_up in (True, False):
        d_gate, d_up = outputs(2, n)
        nv.call("nhip_gated_weight_grad", C.byref(desc), ddgu.ptr, dx_.ptr, d_gate.ptr, d_up.ptr if with_up else None,
                ws.ptr if size.value else None)
        for out, d in [(d_gate, dg), (d_up, du)][:1 + with_up]:
            want = d.T @ x
            _near(values(out, n), want, U[dtype] * np.abs(want) + F32 * (t + 16) * (np.abs(d).T @ np.abs(x)), "dw")
        if not with_up:
            assert np.all(d_up.get((n * k + 64,), np.uint16) == 0x4242)


def test_gated_gradient_of_one_weight_and_of_no_tokens(hip):
    """The gate's gradient alone, the up projection's alone, and zeros for an empty batch."""
    x, gate, up, dh = _gated_case(12, 100, 72, 56, "bfloat16")
    want, tol = M.gated(x, gate, up, dh, "silu"), _gated_tolerances(x, gate, up, dh, "silu", "bfloat16")
    for i, name in ((2, "gate"), (3, "up")):
        def fn(x, gate, up, dh):
            f = (lambda w: F.gated_linear(x, w, up)) if name == "gate" else (lambda w: F.gated_linear(x, gate, w))
            return list(L.vjp(f, gate if name == "gate" else up)[1](dh))

        got = _values(L.compile(fn, device="hip")(*(_tensor(v, "bfloat16") for v in (x, gate, up, dh)))[0])
        _near(got, want[i], tol[i], name)
    out = L.compile(_gated_program("silu"), device="hip")(*(_tensor(v, "bfloat16") for v in (x[:0], gate, up, dh[:0])))
    assert [tuple(t.shape) for t in out] == [(0, 56), (0, 72), (56, 72), (56, 72)] and not _values(out[2]).any() \
        and not _values(out[3]).any()


# ---- clipping


@pytest.mark.parametrize("scale", [0.4, 3.0])
def test_clip(hip, scale):
    """Tensors of every dtype, of one element to several chunks, misaligned slices among them, over and below the bound."""
    rng = np.random.default_rng(0)
    shapes = [((), "float32"), ((1,), "bfloat16"), ((130, 333), "float32"), ((16384,), "float16"), ((16385,), "bfloat16"),
              ((3, 20000), "bfloat16"), ((0, 5), "float32"), ((7,), "float16")]
    xs = [_round(rng.standard_normal(s), dt) for s, dt in shapes]
    norm = np.sqrt(sum((x**2).sum() for x in xs))
    bound = scale * norm
    f = L.compile(lambda bound, *xs: (lambda c, n: [n, *c])(*F.clip_grad_norm(xs, bound)), device="hip")
    args = [_tensor(x, dt) for x, (_, dt) in zip(xs, shapes)]
    for b in (bound, 2 * bound, bound):  # another bound is another run of the same plan
        got = [_values(t) for t in f(float(b), *args)]
        factor = min(1.0, b / (norm + 1e-6))
        assert abs(got[0] - norm) <= 2 * F32 * norm
        for a, x, (_, dt) in zip(got[1:], xs, shapes):
            _near(a, x * factor, U[dt] * np.abs(x * factor) + 4 * F32 * np.abs(x))
        if factor == 1.0:
            assert all(np.array_equal(a, x) for a, x in zip(got[1:], xs))
    assert [st.kind for st in f.plan.steps] == ["clip"]


def test_clip_of_views_and_of_more_tensors_than_a_table(hip):
    """150 tensors in one step (two launches a pass), a slice that starts at an odd element and a transposed one among
    them; the same bits every run."""
    rng = np.random.default_rng(2)
    xs = [_round(rng.standard_normal(rng.integers(1, 300)), "bfloat16") for _ in range(148)]
    base, square = _round(rng.standard_normal(1001), "bfloat16"), _round(rng.standard_normal((40, 24)), "bfloat16")

    def fn(base, square, *xs):
        clipped, norm = F.clip_grad_norm([base[1:], square.t(), *xs], 2.0)
        return [norm, *clipped]

    f = L.compile(fn, device="hip")
    args = [_tensor(v, "bfloat16") for v in (base, square, *xs)]
    first = [t.raw().copy() for t in f(*args)]
    again = [t.raw() for t in f(*args)]
    assert all(np.array_equal(a, b) for a, b in zip(first, again))
    want = [base[1:], square.T, *xs]
    norm = np.sqrt(sum((x**2).sum() for x in want))
    assert abs(float(first[0]) - norm) <= 2 * F32 * norm
    for a, x in zip(first[1:], want):
        w = x * (2.0 / (norm + 1e-6))
        _near(D.to_numpy_values(a, "bfloat16").astype(np.float64), w, U["bfloat16"] * np.abs(w) + 4 * F32 * np.abs(x))


def test_clip_of_values_that_are_not_finite(hip):
    f = L.compile(lambda x: (lambda c, n: [n, *c])(*F.clip_grad_norm([x], 1.0)), device="hip")
    for bad, check in ((np.inf, lambda o: np.isnan(o[0]) and np.all(o[1:] == 0)), (np.nan, lambda o: np.isnan(o).all())):
        x = np.ones(5000)
        x[0] = bad
        norm, out = (_values(t) for t in f(_tensor(x, "bfloat16")))
        assert (np.isinf(norm) if np.isinf(bad) else np.isnan(norm)) and check(out)
    norm, out = (_values(t) for t in f(_tensor(np.full(5000, 1e38), "float32")))  # its squares are past float32
    assert np.isinf(norm) and np.allclose(out, 1 / np.sqrt(5000), rtol=1e-5)  # the float32 norm, not the scale
    norm, out = (_values(t) for t in f(_tensor(np.zeros(10), "bfloat16")))
    assert norm == 0 and not out.any()


def test_clip_past_32_bits_of_elements(hip):
    """2^31 + 77 bf16 elements of which only the last few are not zero."""
    n = (1 << 31) + 77
    buf, norm, ws = Dev(nbytes=2 * n), Dev(nbytes=256), Dev(nbytes=1 << 16)
    nv.call("nhip_memset", C.c_void_p(buf.ptr), 0, C.c_size_t(2 * n))
    tail = D.from_values(np.array([3.0, 4.0], np.float32), "bfloat16")
    nv.h2d(buf.ptr + 2 * (n - 2), np.ascontiguousarray(tail).ctypes.data, 4)
    t = (nv.ClipTensor * 1)(nv.ClipTensor(in_=buf.ptr, out=buf.ptr, numel=n, dtype=1))
    desc = nv.ClipDesc(count=1, max_norm=2.5, eps=0.0)
    nv.call("nhip_clip_grad_norm", C.byref(desc), t, None, norm.ptr, norm.ptr + 4, ws.ptr)
    assert norm.get((2,), np.float32).tolist() == [5.0, 0.5]
    out = np.empty(2, np.uint16)
    nv.d2h(out.ctypes.data, buf.ptr + 2 * (n - 2), 4)
    assert D.to_numpy_values(out, "bfloat16").tolist() == [1.5, 2.0]


# ---- together, captured


class Layer(Module):
    wq: L.Tensor
    wk: L.Tensor
    wv: L.Tensor
    wo: L.Tensor
    norm_q: L.Tensor
    norm_k: L.Tensor
    gate: L.Tensor
    up: L.Tensor
    down: L.Tensor
    lr: float

    def __call__(self, x, cos, sin, batch, heads):
        t, dim = x.shape
        q, k, v = (F.matmul(x, w.t(), "float32", "bfloat16").reshape(batch, t // batch, heads, -1)
                   for w in (self.wq, self.wk, self.wv))
        q, k = F.qk_norm_rope(q, k, cos, sin, self.norm_q, self.norm_k)
        o = F.flash_attention(q, k, v, is_causal=True)
        x = x + F.matmul(o.reshape(t, dim), self.wo.t(), "float32", "bfloat16")
        return x + F.matmul(F.gated_linear(x, self.gate, self.up), self.down.t(), "float32", "bfloat16")


def _layer(dim, ffn, head_dim, lr):
    w = lambda *s: L.empty(list(s), "bfloat16", "meta")  # noqa: E731
    return Layer(w(dim, dim), w(dim, dim), w(dim, dim), w(dim, dim), w(head_dim), w(head_dim), w(ffn, dim), w(ffn, dim),
                 w(dim, ffn), lr)


def _train(layer, x, dy, cos, sin, batch, heads):
    y = layer(x, batch=batch, heads=heads, cos=cos, sin=sin)
    y.backward(dy)
    params = [p for p in layer.parameters()]
    clipped, norm = F.clip_grad_norm([p.grad for p in params], 0.5)
    for p, g in zip(params, clipped):
        p.copy_(p - layer.lr * g)
    return [y, norm]


def _layer_inputs(rng, t, dim, table, half):
    x, dy = (_round(rng.standard_normal((t, dim)), "bfloat16") for _ in range(2))
    angle = np.arange(table)[:, None] * 10000.0 ** (-np.arange(half) / half)
    return [_tensor(x, "bfloat16"), _tensor(dy, "bfloat16"), L.from_numpy(np.cos(angle).astype(np.float32)),
            L.from_numpy(np.sin(angle).astype(np.float32))]


def _load(layer, rng):
    layer.load_state_dict({n: _tensor(_round(rng.standard_normal(p.shape) * 0.1 + (len(p.shape) == 1), "bfloat16"), "bfloat16")
                           for n, p in layer.named_parameters()})


def test_a_layer_in_training_against_the_oracle(hip):
    """Heads, attention, the gated MLP, the clipped gradients and the update in one plan, every step's values against the
    oracle's: 2e-2 of the value and of the tensor's largest, as the attention and the products are held."""
    from lumen_amd.graph.trace import trace

    rng = np.random.default_rng(0)
    batch, heads, dim, ffn, t = 2, 2, 64, 96, 48
    layer = _layer(dim, ffn, dim // heads, 0.5)
    args = _layer_inputs(rng, t, dim, 32, dim // heads // 2)
    traced = trace(_train, (layer, *args, batch, heads))
    arrays = []
    for kind, k in traced.layout:
        if kind == "arg":
            arrays.append(args[k].raw())
        elif kind == "scalar":
            arrays.append(np.array(0.5, np.float64))
        else:
            w = traced.weights[k]
            arrays.append(D.from_values((rng.standard_normal(w.shape) * 0.1 + (len(w.shape) == 1)).astype(np.float32), "bfloat16"))

    def tolerance(dtype, got, want):
        got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
        off = np.abs(got - want) - 2e-2 * np.abs(want) - 2e-2 * np.abs(want).max(initial=0)
        return None if off.max(initial=-1) <= 0 else f"off by {off.max()}"

    assert check_steps(traced.graph, arrays, tolerance) == []
    kinds = {st.kind for st in Plan(traced.graph, "hip:0").steps}
    assert {"heads_fwd", "heads_bwd", "gated_fwd", "gated_grad", "clip", "flash_fwd", "flash_bwd"} <= kinds


def test_a_layer_in_training_replayed(hip):
    """Six calls, the later ones replays of a captured graph with other inputs, against the same calls run uncaptured:
    outputs and weights bit for bit."""
    runs = []
    for graphs in (True, False):
        rng = np.random.default_rng(1)
        layer = _layer(64, 96, 32, 0.5)
        _load(layer, rng)
        out = []
        with L.config.compiler.patch(hip_graphs=graphs):
            f = L.compile(_train, device="hip")
            for _ in range(6):
                y, norm = f(layer, *_layer_inputs(rng, 48, 64, 32, 16), 2, 2)
                out += [y.raw().copy(), norm.raw().copy()]
                nv.sync(0)
        out += [p.raw().copy() for p in layer.parameters()]
        assert len(f.plan.native_steps) >= f.GRAPH_MIN_STEPS
        runs.append(out)
    for a, b in zip(*runs):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("which", ["heads", "gated", "clip"])
def test_each_operator_captured_by_itself(hip, which):
    """A captured run of the operator alone (the plan is short, so Compiled would not capture it), replayed with other
    inputs in the same memory, against the plain run."""
    rng = np.random.default_rng(3)
    if which == "heads":
        x = _heads_case(0, 2, 16, 4, 2, 64, 64, "bfloat16")
        fn, sets = _heads_program(list(x), False, 1e-3), [_heads_case(i, 2, 16, 4, 2, 64, 64, "bfloat16") for i in range(4)]
        dts = ["float32" if k in ("cos", "sin") else "int32" if k == "positions" else "bfloat16" for k in x]
        sets = [list(s.values()) for s in sets]
    elif which == "gated":
        fn, sets, dts = _gated_program("silu"), [_gated_case(i, 40, 64, 96, "bfloat16") for i in range(4)], ["bfloat16"] * 4
    else:
        fn = lambda *xs: (lambda c, n: [n, *c])(*F.clip_grad_norm(xs, 1.5))  # noqa: E731
        sets = [[rng.standard_normal((300,)), rng.standard_normal((70, 30))] for _ in range(4)]
        dts = ["bfloat16"] * 2
    raws = [[np.ascontiguousarray(np.asarray(v, np.int32) if dt == "int32" else D.from_values(np.asarray(v, np.float32), dt))
             for v, dt in zip(s, dts)] for s in sets]
    graph = L.make_graph(fn)(*[L.empty(list(r.shape), dt, "meta") for r, dt in zip(raws[0], dts)])
    plan = Plan(graph, "hip:0")
    ins, ws = [DeviceBuffer(0, r.nbytes) for r in raws[0]], DeviceBuffer(0, plan.workspace_bytes)

    def put(raw):
        for b, r in zip(ins, raw):
            nv.h2d(b.ptr, r.ctypes.data, r.nbytes)

    def read():
        out = []
        for loc in plan.output_locs:
            a = np.empty(loc.shape, D.storage(loc.dtype))
            nv.d2h(a.ctypes.data, ws.ptr + loc.offset * D.size_of(loc.dtype), a.nbytes)
            out.append(a)
        return out

    plain = []
    for raw in raws:
        put(raw)
        plan.run_in(ws.ptr, [b.ptr for b in ins])
        plain.append(read())
    captured = plan.capture(ws.ptr, [b.ptr for b in ins])
    for raw, want in list(zip(raws, plain)) * 2:
        put(raw)
        captured.launch()
        assert all(np.array_equal(a, b) for a, b in zip(read(), want))


def test_gated_of_no_features_and_many_rows(hip):
    f = L.compile(_gated_program("silu"), device="hip")
    got = f(*(_tensor(np.zeros(s), "bfloat16") for s in ((70, 0), (24, 0), (24, 0), (70, 24))))
    assert [o.shape for o in got] == [(70, 24), (70, 0), (24, 0), (24, 0)] and not _values(got[0]).any()


@pytest.mark.parametrize("t,k,n", [(33, 768, 4104), (64, 776, 4096 + 72), (40, 771, 4104), (64, 760, 4104)])
def test_gated_of_wide_weights_and_few_rows(hip, t, k, n):
    """Both sides of the rule that gives 33 to 64 rows of wide weights to the tiles of 128 rows."""
    x, gate, up, dh = _gated_case(t + k, t, k, n, "bfloat16")
    f = L.compile(lambda x, gate, up: [F.gated_linear(x, gate, up)], device="hip")
    got = _values(f(*(_tensor(v, "bfloat16") for v in (x, gate, up)))[0])
    _near(got, M.gated(x, gate, up, dh, "silu")[0], _gated_tolerances(x, gate, up, dh, "silu", "bfloat16")[0])


@pytest.mark.parametrize("n", [8, 9])
def test_gelu_gradient_where_the_square_overflows(hip, n):
    """Both elementwise kernels: g of 1e25 and -1e25 have a derivative of 1 and 0."""
    x = np.array([[1e25, 2.0], [-1e25, 2.0]])
    gate, up, dh = np.tile([1.0, 0.0], (n, 1)), np.tile([0.0, 1.0], (n, 1)), np.full((2, n), 3.0)
    x = _round(x, "bfloat16")
    f = L.compile(_gated_program("gelu"), device="hip")
    h, dx = (_values(v) for v in f(*(_tensor(v, "bfloat16") for v in (x, gate, up, dh)))[:2])
    g = x[0, 0]
    assert np.all(np.abs(h[0] - 2 * g) <= 2.0**-8 * 2 * g) and not h[1].any()
    want = np.array([[6.0 * n, 3 * g * n], [0.0, 0.0]])
    assert np.all(np.abs(dx - want) <= 1.01 * 2.0**-7 * want)  # du's rounding, then dx's


def test_an_operand_used_twice(hip):
    """Queries that are the keys, a gate that is the up projection, a gradient listed twice."""
    x = _heads_case(31, 2, 9, 2, 2, 64, 64, "bfloat16", positions=False)
    x["k"], x["wk"] = x["q"], x["wq"]

    def heads(q, w, c, s, gq, gk):
        out, pull = L.vjp(lambda q, w: F.qk_norm_rope(q, q, c, s, w, w, eps=1e-3), q, w)
        return [*out, *pull((gq, gk))]

    got = [_values(v) for v in L.compile(heads, device="hip")(*(
        _tensor(x[n], "float32" if n in ("cos", "sin") else "bfloat16") for n in ("q", "wq", "cos", "sin", "gq", "gk")))]
    want = M.heads(x, 1e-3, False)
    _heads_check(got[:2], x, "bfloat16", 1e-3, False)
    for a, parts in ((got[2], want[2:4]), (got[3], want[4:6])):
        rows = np.prod(x["q"].shape[:3])
        tol = U["bfloat16"] * (sum(np.abs(p) for p in parts) + np.abs(sum(parts))) * 1.01 + F32 * (rows + 104) * 8 * rows
        _near(a, sum(parts), tol)
    t, w, _, dh = _gated_case(32, 70, 72, 40, "bfloat16")

    def gated(t, w, dh):
        h, pull = L.vjp(lambda t, w: F.gated_linear(t, w, w), t, w)
        return [h, *pull(dh)]

    got = [_values(v) for v in L.compile(gated, device="hip")(*(_tensor(v, "bfloat16") for v in (t, w, dh)))]
    h, dx, dg, du = M.gated(t, w, w, dh, "silu")
    th, tdx, tdg, tdu = _gated_tolerances(t, w, w, dh, "silu", "bfloat16")
    _near(got[0], h, th)
    _near(got[1], dx, tdx)
    _near(got[2], dg + du, tdg + tdu + U["bfloat16"] * 1.05 * np.abs(dg + du) + U["bfloat16"] * (tdg + tdu))
    clip = L.compile(lambda g: (lambda c, n: [n, *c])(*F.clip_grad_norm([g, g], 1.0)), device="hip")
    out = [_values(v) for v in clip(_tensor(t, "bfloat16"))]
    norm = np.sqrt(2 * (t * t).sum())
    assert abs(out[0] - norm) <= 2 * F32 * norm
    for o in out[1:]:
        _near(o, t / (norm + 1e-6), (U["bfloat16"] + 4 * F32) * np.abs(t / norm))


@pytest.mark.parametrize("flags", [dict(memory_limit=1), dict(schedules=False, update_in_place=False),
                                   dict(merge_dots=False, epilogue_fusion=False)], ids=lambda f: "-".join(f))
def test_a_layer_in_training_under_other_flags(hip, flags):
    """The same layer's two calls with rematerialized values, without donation and without merged
    products: output, norm and weights within 2e-2 of the largest, as the layer is held against the oracle."""
    runs = []
    for patch in ({}, flags):
        rng = np.random.default_rng(9)
        layer = _layer(64, 96, 32, 0.5)
        _load(layer, rng)
        with L.config.compiler.patch(**patch):
            f = L.compile(_train, device="hip")
            out = []
            for _ in range(2):
                out += [_values(v).copy() for v in f(layer, *_layer_inputs(rng, 48, 64, 32, 16), 2, 2)]
        runs.append(out + [_values(p).copy() for p in layer.parameters()])
    for a, b in zip(*runs):
        assert np.abs(a - b).max() <= 2e-2 * max(np.abs(a).max(), 1e-6)


@pytest.mark.parametrize("t,k,n,dtype", [(2901, 2891, 9, "float16"), (70, 2300, 2001, "bfloat16"), (2300, 2307, 77, "bfloat16"),
                                         (65, 1153, 2304, "float16"), (700, 700, 12000, "bfloat16")])
def test_gated_backward_kernels_of_many_tiles(hip, t, k, n, dtype):
    """As above where the products' launches pass one workgroup a CU: tiles of 256 whole (dx; then the weights'), tiles of 128
    in two stages (dx; then the weights'), and tiles of 256 in parts (dx)."""
    test_gated_backward_kernels(hip, t, k, n, dtype)


@pytest.mark.parametrize("t,k,n", [(139, 2056, 72), (70, 1029, 131), (64, 4096, 40), (200, 1088, 260)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_gated_in_parts(hip, t, k, n, dtype):
    """Few tiles of a long k in parts, by default and by the config: k that ends inside a part's tile, odd sizes, g and u, and
    the same bits every run."""
    x, gate, up, dh = _gated_case(t + k, t, k, n, dtype)
    tol, e = _gated_tolerances(x, gate, up, dh, "gelu", dtype)[0], F32 * (k + 16)
    want = M.gated(x, gate, up, dh, "gelu")[0]
    runs = []
    for config in (-1, 4, 4):
        h, g, u = _gated_abi(x, gate, up, dtype, "gelu", config, True)
        _near(D.to_numpy_values(h[:t * n].view(D.storage(dtype)), dtype).astype(np.float64).reshape(t, n), want, tol, config)
        for s, w in ((g, gate), (u, up)):
            _near(s[:t * n].astype(np.float64).reshape(t, n), x @ w.T, e * (np.abs(x) @ np.abs(w).T), config)
            assert np.all(s[t * n:] == 77.0)
        assert np.all(h[t * n:] == 0x4242)
        runs.append((h, g, u))
    assert all(np.array_equal(a, b) for a, b in zip(*runs[1:]))


def test_heads_of_which_one_tensor_has_none(hip):
    """Queries without keys' heads and keys without queries': the other's results as ever, weight gradients of zeros."""
    for n, nkv in ((3, 0), (0, 2)):
        x = _heads_case(40 + n, 2, 7, max(n, 1), max(nkv, 1), 64, 64, "bfloat16", positions=False)
        want = M.heads(x, 1e-3, False)
        empty = ("k", "gk") if nkv == 0 else ("q", "gq")
        for m in empty:
            x[m] = x[m][:, :, :0]
        got = [_values(v) for v in L.compile(_heads_program(list(x), False, 1e-3), device="hip")(
            *(_tensor(v, "float32" if m in ("cos", "sin") else "bfloat16") for m, v in x.items()))]
        full = 0 if nkv == 0 else 1
        rows, d = 2 * 7 * max(n, nkv), 64
        for i in range(6):
            if i % 2 != full:
                assert not got[i].any() and (i >= 4 or got[i].size == 0)
            elif i < 4:
                _near(got[i], want[i], U["bfloat16"] * np.abs(want[i]) + F32 * (d + 40) * 8 * np.abs(want[i]).max())
            else:
                _near(got[i], want[i], U["bfloat16"] * np.abs(want[i]) + F32 * (rows + d + 40) * 4 * rows)


def test_gated_of_one_axis_of_no_outputs_and_of_a_sliced_cotangent(hip):
    """x [K] gives [F]; weights of no features give nothing and gradients of zeros; a cotangent whose rows start off 16 bytes."""
    x, gate, up, dh = _gated_case(50, 5, 48, 40, "bfloat16")
    tol, want = _gated_tolerances(x, gate, up, dh, "gelu", "bfloat16"), M.gated(x, gate, up, dh, "gelu")
    one = L.compile(lambda x, gate, up: [F.gated_linear(x, gate, up, activation="gelu")], device="hip")
    got = _values(one(_tensor(x[2], "bfloat16"), _tensor(gate, "bfloat16"), _tensor(up, "bfloat16"))[0])
    _near(got, want[0][2], tol[0][2])
    out = L.compile(_gated_program("silu"), device="hip")(*(_tensor(np.ones(s), "bfloat16") for s in ((70, 48), (0, 48), (0, 48), (70, 0))))
    assert [o.shape for o in out] == [(70, 0), (70, 48), (0, 48), (0, 48)] and not _values(out[1]).any()
    wide = np.full((5, 51), np.nan)
    wide[:, 3:43] = dh

    def fn(x, gate, up, wide):
        h, pull = L.vjp(lambda x, gate, up: F.gated_linear(x, gate, up, activation="gelu"), x, gate, up)
        return [h, *pull(wide[:, 3:43])]

    got = L.compile(fn, device="hip")(*(_tensor(v, "bfloat16") for v in (x, gate, up, wide)))
    for i, (a, w, t) in enumerate(zip(got, want, tol)):
        _near(_values(a), w, t, i)


def test_clip_of_empty_gradients_and_a_bound_that_is_infinite(hip):
    f = L.compile(lambda *xs: (lambda c, n: [n, *c])(*F.clip_grad_norm(xs, float("inf"))), device="hip")
    x = np.array([3.0, 4.0])
    out = [_values(v) for v in f(_tensor(np.zeros((0, 4)), "float32"), _tensor(x, "bfloat16"), _tensor(np.zeros(0), "float16"))]
    assert out[0] == 5.0 and np.array_equal(out[2], x) and out[1].shape == (0, 4) and out[3].shape == (0,)
    g = L.compile(lambda x: (lambda c, n: [n, *c])(*F.clip_grad_norm([x], 1.0)), device="hip")
    out = [_values(v) for v in g(_tensor(np.zeros((0, 4)), "float32"))]
    assert out[0] == 0.0 and out[1].shape == (0, 4)


def test_heads_of_more_rows_than_a_launch(hip):
    """2^30 + 24 rows of one element (two launches): the last tokens' results, and weight gradients over all rows. x / |x| of
    eps 0 is a sign, so y is the weight and dw the sum of dy; float32 sums of at most 2^17 terms a lane, then of 4096."""
    seq, heads = (1 << 27) + 3, 8
    rows = seq * heads
    x, y, dy, dx = (Dev(nbytes=2 * rows) for _ in range(4))
    nv.call("nhip_memset", C.c_void_p(x.ptr), 0x3c, C.c_size_t(2 * rows))
    nv.call("nhip_memset", C.c_void_p(dy.ptr), 0x3c, C.c_size_t(2 * rows))
    tail = np.random.default_rng(0).choice([-2.0, 0.5, 3.0], 24)
    bits = np.ascontiguousarray(D.from_values(tail.astype(np.float32), "bfloat16"))
    nv.h2d(x.ptr + 2 * (rows - 24), bits.ctypes.data, 48)
    w, table, dw = Dev(np.array([0x4000], np.uint16)), Dev(np.zeros(4, np.float32)), Dev(nbytes=256)  # a weight of 2
    desc = nv.HeadsDesc(batch=1, seq=seq, heads=heads, kv_heads=0, head_dim=1, rot=0, table_rows=1, dtype=1, eps=0.0)
    for m in ("q", "oq", "dq"):
        setattr(desc, m + "_s", heads)
        setattr(desc, m + "_n", 1)
    size = C.c_size_t()
    nv.call("nhip_qk_norm_rope_workspace", C.byref(desc), C.byref(size))
    assert size.value >= 2 * 2048 * 4
    ws = Dev(nbytes=size.value)
    head = [x.ptr, x.ptr, w.ptr, w.ptr, table.ptr, table.ptr, None]
    nv.call("nhip_qk_norm_rope", C.byref(desc), *head, y.ptr, y.ptr)
    nv.call("nhip_qk_norm_rope_bwd", C.byref(desc), *head, dy.ptr, dy.ptr, dx.ptr, dx.ptr, dw.ptr, None, ws.ptr)
    got = np.empty(64, np.uint16)
    for at, want in ((0, np.full(64, 2.0)), (rows - 64, np.r_[np.full(40, 2.0), 2.0 * np.sign(tail)])):
        nv.d2h(got.ctypes.data, y.ptr + 2 * at, 128)
        assert np.array_equal(D.to_numpy_values(got, "bfloat16"), want), at
        nv.d2h(got.ctypes.data, dx.ptr + 2 * at, 128)
        assert np.abs(D.to_numpy_values(got, "bfloat16").astype(np.float64)).max() <= 90 * 0.025 * 8 * F32, at
    one = float(D.to_numpy_values(np.array([0x3c3c], np.uint16), "bfloat16")[0])
    want = one * (rows - 24 + np.sign(tail).sum())
    total = float(D.to_numpy_values(dw.get((1,), np.uint16), "bfloat16")[0])
    assert abs(total - want) <= (U["bfloat16"] + 2 * (1 << 17) * F32) * want


@pytest.mark.parametrize("t,k,n,dtype,paired", [(777, 520, 1416, "float16", True), (130, 67, 333, "bfloat16", True), (5, 1, 9, "bfloat16", True),
                                                (65, 1153, 2304, "bfloat16", False), (17, 128, 1344, "float16", True),
                                                (1500, 70, 72, "bfloat16", True)])
def test_gated_gradients_in_one_call(hip, t, k, n, dtype, paired):
    """dx and the weights' gradients together, with and without d_up, the same bits each time, nothing written behind them."""
    whole = -(-n // 8) * 8
    x, gate, up, _ = _gated_case(t + k, t, k, n, dtype)
    rng = np.random.default_rng(t)
    dg, du = (_round(rng.standard_normal((t, n)), dtype) for _ in range(2))
    dgu = np.zeros((t, 2 * whole))
    dgu[:, :n], dgu[:, whole:whole + n] = dg, du
    dev = [Dev(np.ascontiguousarray(D.from_values(np.asarray(v, np.float32), dtype))) for v in (dgu, gate, up, x)]
    desc = nv.GatedDesc(m=t, n=n, k=k, x_m=k, w_n=k, dtype={"bfloat16": 1, "float16": 2}[dtype], config=-1)
    size, flag = C.c_size_t(), C.c_int()
    nv.call("nhip_gated_backward_workspace", C.byref(desc), C.byref(size))
    nv.call("nhip_gated_backward_paired", C.byref(desc), C.byref(flag))
    assert bool(flag.value) == paired
    ws = Dev(np.full(size.value + 256, 0x42, np.uint8))
    place = ws.ptr if size.value else None
    shapes = [(t, k), (n, k), (n, k)]
    runs = []
    for with_up in (True, False, True):
        outs = [Dev(np.full(a * b + 64, 0x4242, np.uint16)) for a, b in shapes]
        nv.call("nhip_gated_backward", C.byref(desc), *(v.ptr for v in dev), outs[0].ptr, outs[1].ptr,
                outs[2].ptr if with_up else None, place)
        runs.append([o.get((a * b + 64,), np.uint16) for o, (a, b) in zip(outs, shapes)])
    assert all(np.array_equal(a, b) for a, b in zip(runs[0], runs[2]))
    assert all(np.array_equal(a, b) for a, b in zip(runs[0][:2], runs[1][:2])) and np.all(runs[1][2] == 0x4242)
    mags = np.abs(dg) @ np.abs(gate) + np.abs(du) @ np.abs(up)
    want = [(dg @ gate + du @ up, (2 * n + 16) * mags)]
    want += [(d.T @ x, (t + 16) * (np.abs(d).T @ np.abs(x))) for d in (dg, du)]
    for raw, (a, b), (w, roundings) in zip(runs[0], shapes, want):
        assert np.all(raw[a * b:] == 0x4242)
        got = D.to_numpy_values(raw[:a * b].view(D.storage(dtype)), dtype).astype(np.float64).reshape(a, b)
        _near(got, w, U[dtype] * np.abs(w) + F32 * roundings)
    assert np.all(ws.get((size.value + 256,), np.uint8)[size.value:] == 0x42)


def test_heads_of_several_launches_in_sequences_that_end_inside_them(hip):
    """3 sequences of 2^24 + 1 heads of 4 elements: launches end inside a sequence and start there again. Both directions at
    the tokens around every boundary, positions past the table clamped."""
    batch, seq, d, table = 3, (1 << 24) + 1, 4, 64
    rows = batch * seq
    rng = np.random.default_rng(3)
    part = _round(rng.standard_normal((10007, d)) + 2, "bfloat16")
    dpart = _round(rng.standard_normal((10007, d)), "bfloat16")
    dev = [Dev(np.resize(D.from_values(p.astype(np.float32), "bfloat16"), (rows, d))) for p in (part, dpart)]
    y, dx = Dev(nbytes=rows * d * 2), Dev(nbytes=rows * d * 2)
    angle = np.arange(table)[:, None] * np.array([0.1, 0.03])
    cos, sin = (f(angle).astype(np.float32) for f in (np.cos, np.sin))
    dcos, dsin, w, dw = Dev(cos), Dev(sin), Dev(np.array([0x4000] * d, np.uint16)), Dev(nbytes=256)  # weights of 2
    desc = nv.HeadsDesc(batch=batch, seq=seq, heads=1, kv_heads=0, head_dim=d, rot=d, table_rows=table, dtype=1, eps=1e-3)
    for m in ("q", "oq", "dq"):
        for axis, stride in (("b", seq * d), ("s", d), ("n", d)):
            setattr(desc, f"{m}_{axis}", stride)
    size = C.c_size_t()
    nv.call("nhip_qk_norm_rope_workspace", C.byref(desc), C.byref(size))
    ws = Dev(nbytes=size.value)
    head = [dev[0].ptr, dev[0].ptr, w.ptr, w.ptr, dcos.ptr, dsin.ptr, None]
    nv.call("nhip_qk_norm_rope", C.byref(desc), *head, y.ptr, y.ptr)
    nv.call("nhip_qk_norm_rope_bwd", C.byref(desc), *head, dev[1].ptr, dev[1].ptr, dx.ptr, dx.ptr, dw.ptr, None, ws.ptr)
    for at in (0, seq - 40, seq + 20, 1 << 25, (1 << 25) - 80, 2 * seq - 40, rows - 80):
        token = np.arange(at, at + 80)
        s = token % seq
        x = {"q": part[token % 10007].reshape(1, 80, 1, d), "k": np.zeros((1, 80, 0, d)), "wq": np.full(d, 2.0), "wk": np.full(d, 2.0),
             "cos": cos.astype(np.float64), "sin": sin.astype(np.float64), "positions": np.minimum(s, table - 1).reshape(1, 80),
             "gq": dpart[token % 10007].reshape(1, 80, 1, d), "gk": np.zeros((1, 80, 0, d))}
        want = M.heads(x, 1e-3, False)
        for buf, i in ((y, 0), (dx, 2)):
            got = np.empty((80, d), np.uint16)
            nv.d2h(got.ctypes.data, buf.ptr + at * d * 2, got.nbytes)
            ref = want[i].reshape(80, d)
            _near(D.to_numpy_values(got, "bfloat16").astype(np.float64), ref, U["bfloat16"] * np.abs(ref) + F32 * (d + 40) * 8 * np.abs(ref).max(), at)


@pytest.mark.parametrize("t,k,n,dtype", [(16, 16, 16, "bfloat16"), (65, 72, 40, "float16"), (128, 64, 64, "bfloat16")])
def test_gated_gradients_of_two_micro_batches(hip, t, k, n, dtype):
    """``backward()`` after each of two micro-batches: the weights' gradients are the sums of both, each rounded, and rounded
    again; each input's gradient is its own."""
    (x1, gate, up, dy1), (x2, _, _, dy2) = _gated_case(61, t, k, n, dtype), _gated_case(62, t, k, n, dtype)

    def fn(x1, x2, gate, up, dy1, dy2):
        for x, dy in ((x1, dy1), (x2, dy2)):
            F.gated_linear(x, gate, up).backward(dy)
        return [x1.grad, x2.grad, gate.grad, up.grad]

    f = L.compile(fn, device="hip")
    got = [_values(v) for v in f(*(_tensor(v, dtype) for v in (x1, x2, gate, up, dy1, dy2)))]
    want = [M.gated(x, gate, up, dy, "silu") for x, dy in ((x1, dy1), (x2, dy2))]
    tol = [_gated_tolerances(x, gate, up, dy, "silu", dtype) for x, dy in ((x1, dy1), (x2, dy2))]
    assert [st.kind for st in f.plan.steps].count("gated_fwd") == 2
    for i in range(2):
        _near(got[i], want[i][1], tol[i][1], i)
    for i in (2, 3):
        w, each = want[0][i] + want[1][i], tol[0][i] + tol[1][i]
        _near(got[i], w, each + U[dtype] * (np.abs(w) + each), i)


def test_a_layer_of_two_micro_batches(hip):
    """Heads, attention and the gated MLP twice in one plan, ``backward()`` after each: the weights' gradients against the sum
    of two plans of one micro-batch each, 2e-2 of the largest, as the layer is held under other flags."""
    rng = np.random.default_rng(7)
    layer = _layer(64, 96, 32, 0.5)
    _load(layer, rng)
    (x1, dy1, cos, sin), (x2, dy2, _, _) = (_layer_inputs(rng, 48, 64, 32, 16) for _ in range(2))

    def grads(layer, cos, sin, *pairs):
        for x, dy in zip(pairs[::2], pairs[1::2]):
            layer(x, cos, sin, 2, 2).backward(dy)
        return [p.grad for p in layer.parameters()]

    runs = [[_values(v).copy() for v in L.compile(grads, device="hip")(layer, cos, sin, *pairs)]
            for pairs in ((x1, dy1), (x2, dy2), (x1, dy1, x2, dy2))]
    for a, b, both in zip(*runs):
        assert np.abs(both - a - b).max() <= 2e-2 * (np.abs(a) + np.abs(b)).max()


@pytest.mark.parametrize("fused,dtype,d,rot,interleaved", [
    (True, "float64", 16, 16, False), (True, "float64", 10, 6, True), (True, "bfloat16", 1030, 64, True),
    (False, "bfloat16", 16, 8, False), (False, "float32", 64, 64, False)])
def test_heads_that_are_primitives(hip, fused, dtype, d, rot, interleaved):
    """What the head kernels do not take, in both directions, float64 with its own roundings."""
    x = _heads_case(70 + d, 2, 5, 4, 2, d, rot, "float32" if dtype == "float64" else dtype, interleaved)
    exact = ("cos", "sin", "positions")
    args = [L.from_numpy(v if m in exact else v.astype(np.float64)) if m in exact or dtype == "float64" else _tensor(v, dtype)
            for m, v in x.items()]
    with L.config.compiler.patch(fused_operators=fused):
        f = L.compile(_heads_program(list(x), interleaved, 1e-3), device="hip")
        got = [_values(t) for t in f(*args)]
    assert not {"heads_fwd", "heads_bwd"} & {st.kind for st in f.plan.steps}
    if dtype != "float64":
        return _heads_check(got, x, dtype, 1e-3, interleaved)
    step = 2.0**-53
    for i, (a, w) in enumerate(zip(got, M.heads(x, 1e-3, interleaved))):
        rows = np.prod(x["q" if i in (0, 2, 4) else "k"].shape[:3])
        _near(a, w, step * (d + 40) * 8 * np.abs(w).max() if i < 4 else step * (rows + d + 40) * 4 * rows, i)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_a_gradient_of_the_gated_gradient(hip, dtype):
    """The gradients' own gradients against the oracle on the same graph: 2e-2 of the largest in bfloat16, as the layer is
    held, and 2^-24 times 40 sums of 63 terms in float32."""
    from oracle import oracle

    rng = np.random.default_rng(80)
    shapes = [(65, 63), (17, 63), (17, 63), (65, 17), (65, 63), (17, 63), (17, 63)]
    scale = [1, 63**-0.5, 63**-0.5, 1, 1, 1, 1]
    arrays = [_round(rng.standard_normal(s) * c, dtype) for s, c in zip(shapes, scale)]

    def fn(x, gate, up, dh, cx, cg, cu):
        def first(x, gate, up, dh):
            return L.vjp(lambda x, gate, up: F.gated_linear(x, gate, up), x, gate, up)[1](dh)

        return list(L.vjp(first, x, gate, up, dh)[1]((cx, cg, cu)))

    tensors = [_tensor(v, dtype) for v in arrays]
    got = [_values(t) for t in L.compile(fn, device="hip")(*tensors)]
    graph = L.make_graph(fn)(*[L.empty(list(s), dtype, "meta") for s in shapes])
    for a, w in zip(got, oracle.values(graph, [t.raw() for t in tensors])):
        w = np.asarray(w, np.float64)
        assert np.abs(a - w).max() <= (2e-2 if dtype == "bfloat16" else 2.0**-24 * 40 * 63) * np.abs(w).max()


def test_heads_of_as_many_queries_as_keys_past_a_launch(hip):
    """2^21 tokens of 16 + 16 heads of 132 elements, 64 lanes each: 2^32 threads, two launches. The inputs' tokens are 64 that
    repeat (batches that lie on one another), the results' rows at both ends and at the launches' border."""
    batch, seq, n, d = 1 << 15, 64, 16, 132
    x = _heads_case(90, 1, seq, n, n, d, 64, "bfloat16", positions=False)
    dev = {m: Dev(np.ascontiguousarray(D.from_values(np.asarray(x[m], np.float32), "bfloat16"))) for m in ("q", "k", "wq", "wk")}
    cos, sin = Dev(x["cos"]), Dev(x["sin"])
    out = {m: Dev(nbytes=batch * seq * n * d * 2) for m in ("oq", "ok")}
    desc = nv.HeadsDesc(batch=batch, seq=seq, heads=n, kv_heads=n, head_dim=d, rot=64, table_rows=64, dtype=1, eps=1e-3)
    for m in ("q", "k", "oq", "ok"):
        for axis, stride in (("b", seq * n * d if m in out else 0), ("s", n * d), ("n", d)):
            setattr(desc, f"{m}_{axis}", stride)
    nv.call("nhip_qk_norm_rope", C.byref(desc), dev["q"].ptr, dev["k"].ptr, dev["wq"].ptr, dev["wk"].ptr, cos.ptr, sin.ptr, None,
            out["oq"].ptr, out["ok"].ptr)
    got = np.empty((seq, n, d), np.uint16)
    for m, want in zip(("oq", "ok"), M.heads(x, 1e-3, False)):
        for b in (0, batch // 2 - 1, batch // 2, batch - 1):
            nv.d2h(got.ctypes.data, out[m].ptr + b * got.nbytes, got.nbytes)
            _near(D.to_numpy_values(got, "bfloat16").astype(np.float64), want[0],
                  U["bfloat16"] * np.abs(want[0]) + F32 * (d + 40) * 8 * np.abs(want).max(), (m, b))


@pytest.mark.parametrize("n", [8, 9])
@pytest.mark.parametrize("dtype,most", [("bfloat16", 20.0), ("float16", 9.0)])
def test_sigmoid_gradient_of_large_gates(hip, dtype, most, n):
    """Both elementwise kernels, relative to the value on both sides (float16 within its normal numbers): a rounding of dg,
    one of dx and 64 of 2^-24 between (exp(20) as 2^28.9: the exponent's rounding and its factor's are 20 each)."""
    from tests.test_operators import sigmoid_gradient

    g = np.arange(4.0, most + 0.5, 0.5)
    *x, want = sigmoid_gradient(np.concatenate([g, -g]), n)
    dx = _values(L.compile(_gated_program("sigmoid"), device="hip")(*(_tensor(v, dtype) for v in x))[1])
    _near(dx, want, (2.01 * U[dtype] + 64 * F32) * want)


@pytest.mark.parametrize("b,s,n,nkv,d", [(1, 200, 16, 16, 128), (4, 300, 32, 8, 64), (3, 33, 6, 2, 80), (1, 131, 3, 3, 36), (2, 57, 5, 1, 7)])
def test_heads_weight_gradients_hold_every_row_once(hip, b, s, n, nkv, d):
    """float32 heads, so that no rounding of the result hides a row: each term's own error, 40 roundings (a row's sum of squares is
    at most 8 elements a lane and 6 exchanges, its root, mean and factors a dozen more), and at most 161 additions on its way
    (8 rows a lane, 6 exchanges, 3 waves, 2050 partial rows as 129 and 15). A row's share is over twice
    that in some element: of one lost or counted twice more than the tolerance would be left."""
    rot = d // 2 * 2
    x = _heads_case(100 + d, b, s, n, nkv, d, rot, "float32", table=512)
    f = L.compile(_heads_program(list(x), False, 1e-3), device="hip")
    got = [_values(t) for t in f(*[L.from_numpy(v) if m in ("cos", "sin", "positions") else _tensor(v, "float32") for m, v in x.items()])]
    want = M.heads(x, 1e-3, False)
    for i, h, g, w in ((4, "q", "gq", "wq"), (5, "k", "gk", "wk")):
        at = x["positions"].astype(int)
        c, sn = (np.float64(x[t])[at][:, :, None] for t in ("cos", "sin"))
        xhat = x[h] / np.sqrt((x[h] ** 2).mean(-1, keepdims=True) + 1e-3)
        p, q, rest = x[g][..., :rot // 2], x[g][..., rot // 2:rot], x[g][..., rot:]
        dz = np.concatenate([p * c + q * sn, q * c - p * sn, rest], -1)
        terms = (dz * xhat).reshape(-1, d)
        mags = (np.concatenate([np.abs(p) + np.abs(q), np.abs(p) + np.abs(q), np.abs(rest)], -1) * np.abs(xhat)).reshape(-1, d).sum(0)
        assert np.allclose(terms.sum(0), want[i], rtol=1e-10, atol=1e-9)
        tol = U["float32"] * np.abs(want[i]) + F32 * (161 + 40) * mags
        assert np.all((np.abs(terms) / tol).max(1) > 2)
        _near(got[i], want[i], tol, w)


@pytest.mark.parametrize("d", [1, 4])
def test_heads_weight_gradients_hold_every_launch_once(hip, d):
    """2^26 + 24 rows, three launches, on the general and the vector kernel: cotangents of 1, 2, .. 64 in rows at the launches'
    borders, zeros elsewhere. Of heads of equal elements dw is their sum, 127, which bf16 holds: exact."""
    rows = (1 << 26) + 24
    x, dy, dx = (Dev(nbytes=2 * rows * d) for _ in range(3))
    nv.call("nhip_memset", C.c_void_p(x.ptr), 0x3c, C.c_size_t(2 * rows * d))
    nv.call("nhip_memset", C.c_void_p(dy.ptr), 0, C.c_size_t(2 * rows * d))
    for i, row in enumerate((0, 12345, (1 << 25) - 1, 1 << 25, (1 << 26) - 1, 1 << 26, rows - 1)):
        bits = np.ascontiguousarray(D.from_values(np.full(d, 2.0**i, np.float32), "bfloat16"))
        nv.h2d(dy.ptr + 2 * row * d, bits.ctypes.data, 2 * d)
    w, table, dw = Dev(np.full(d, 0x3f80, np.uint16)), Dev(np.zeros(4, np.float32)), Dev(nbytes=256)
    desc = nv.HeadsDesc(batch=1, seq=rows, heads=1, kv_heads=0, head_dim=d, rot=0, table_rows=1, dtype=1, eps=0.0)
    for m in ("q", "oq", "dq"):
        setattr(desc, m + "_s", d)
        setattr(desc, m + "_n", d)
    size = C.c_size_t()
    nv.call("nhip_qk_norm_rope_workspace", C.byref(desc), C.byref(size))
    assert size.value == 3 * 2050 * d * 4
    ws = Dev(nbytes=size.value)
    nv.call("nhip_qk_norm_rope_bwd", C.byref(desc), x.ptr, x.ptr, w.ptr, w.ptr, table.ptr, table.ptr, None, dy.ptr, dy.ptr,
            dx.ptr, dx.ptr, dw.ptr, None, ws.ptr)
    assert D.to_numpy_values(dw.get((d,), np.uint16), "bfloat16").tolist() == [127.0] * d


def test_operands_and_cotangents_that_are_broadcast(hip):
    """One token's row for all rows, one head for all heads (strides of 0), and losses that are plain sums, whose cotangents are
    ones, or take the queries alone, so that the keys' are zeros."""
    x, gate, up, _ = _gated_case(110, 1, 64, 40, "bfloat16")
    for t in (70, 9):
        def gated(x, gate, up, t=t):
            F.sum(F.gated_linear(x.expand(t, 64), gate, up).float()).backward()
            return [F.gated_linear(x.expand(t, 64), gate, up), x.grad, gate.grad, up.grad]

        rows, ones = np.repeat(x, t, 0), np.ones((t, 40))
        want, tol = M.gated(rows, gate, up, ones, "silu"), _gated_tolerances(rows, gate, up, ones, "silu", "bfloat16")
        got = [_values(v) for v in L.compile(gated, device="hip")(*(_tensor(v, "bfloat16") for v in (x, gate, up)))]
        for i in (0, 2, 3):
            _near(got[i], want[i], tol[i], i)
        each = want[1].sum(0, keepdims=True)  # t rounded gradients and their sum's roundings
        _near(got[1], each, tol[1].sum(0, keepdims=True) + (U["bfloat16"] + t * F32) * (np.abs(want[1]) + tol[1]).sum(0), "dx")
    h = _heads_case(111, 2, 9, 1, 1, 64, 64, "bfloat16", positions=False)
    args = [_tensor(h[m], "float32" if m in ("cos", "sin") else "bfloat16") for m in ("q", "k", "cos", "sin", "wq", "wk")]

    def heads(q, k, cos, sin, wq, wk):
        yq, yk = F.qk_norm_rope(q.expand(2, 9, 3, 64), k, cos, sin, wq, wk, eps=1e-3)
        F.sum(yq.float()).backward()
        return [yq, yk, wq.grad, k.grad if k.grad is not None else k * 0.0]

    h["q"], h["gq"], h["gk"] = np.repeat(h["q"], 3, 2), np.ones((2, 9, 3, 64)), np.zeros((2, 9, 1, 64))
    want = M.heads(h, 1e-3, False)
    f = L.compile(heads, device="hip")
    got = [_values(v) for v in f(*args)]
    for a, w in zip(got[:2], want):
        _near(a, w, U["bfloat16"] * np.abs(w) + F32 * 104 * 8 * np.abs(w).max())
    xhat = np.abs(h["q"]) / np.sqrt((h["q"] ** 2).mean(-1, keepdims=True) + 1e-3)
    _near(got[2], want[4], U["bfloat16"] * np.abs(want[4]) + F32 * 201 * 2 * xhat.sum((0, 1, 2)), "dw")
    assert not got[3].any() and {"heads_fwd", "heads_bwd"} <= {st.kind for st in f.plan.steps}
