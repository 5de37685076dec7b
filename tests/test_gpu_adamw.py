"""adamw on the GPU against plain float64 NumPy (tests/training_math.py): float32 results within the roundings counted there, a
16-bit weight within its own rounding of that."""

import ctypes as C

import numpy as np
import pytest

import lumen_amd as L
import lumen_amd.functional as F
from lumen_amd import dtypes as D
from lumen_amd import native as nv
from lumen_amd import workloads as W
from lumen_amd.compiler.plan import Plan
from lumen_amd.tensor import DeviceBuffer
from tests import training_math as M
from tests.hiputil import Dev

pytestmark = pytest.mark.gpu

BETAS, EPS, DECAY = (0.9, 0.99), 1e-6, 0.05
DT = {"float32": 0, "bfloat16": 1, "float16": 2}


def _bits(x, dtype):
    return np.array(D.from_values(np.asarray(x, np.float32), dtype))


def _up(bits, dtype):
    return np.asarray(D.to_numpy_values(bits, dtype), np.float64)


def _weight(rng, shape, dtype, master):
    """Storage of a weight's operands: p, g, m, v and its master or None."""
    w = rng.standard_normal(shape).astype(np.float32)
    m, v = rng.standard_normal(shape).astype(np.float32), np.abs(rng.standard_normal(shape)).astype(np.float32)
    return _bits(w, dtype), _bits(rng.standard_normal(shape), dtype), m, v, w if master else None


def _check(x, got, dtype, step, lr, what, scale=None):
    """``got``: the new p, m, v and master (or None), storage. A gradient times ``scale`` is rounded to float32 and then to its
    type, or at once (the instruction that multiplies and converts): where the float32 product is a tie between two values of the
    type and the exact one is not, these are one step apart, so an element is right if all its results are those of either."""
    p, g, m, v, w = x
    grads = [_up(g, dtype)]
    if scale is not None:
        scale = np.float64(np.float32(scale))
        grads = [_up(_bits(np.float32(grads[0] * scale), dtype), dtype), _up(D.from_values(grads[0] * scale, dtype), dtype)]
    start = _up(p, dtype) if w is None else w
    right = np.zeros(start.shape, bool)
    for grad in grads:
        want = M.adamw(start, grad, m, v, step, lr, BETAS, EPS, DECAY)
        tol = M.adamw_tolerances(start, grad, m, v, step, lr, BETAS, EPS, DECAY)
        tp = tol[0] + (0 if dtype == "float32" else M.U[dtype] * np.abs(want[0]) + M.LOW[dtype])
        ok = np.ones(start.shape, bool)
        for a, b, t in ((_up(got[0], dtype), want[0], tp), (got[1], want[1], tol[1]), (got[2], want[2], tol[2]), (got[3], want[0], tol[0])):
            if a is not None:
                assert a.shape == b.shape
                ok &= np.abs(a - b) <= t
        right |= ok
    assert right.all(), (what, int((~right).sum()))
    if w is not None and got[3] is not None:
        assert np.array_equal(got[0], _bits(got[3], dtype)), what


def _tensor(bits, dtype):
    return L.Tensor(dtype, np.shape(bits), "cpu", host=bits)


@pytest.mark.parametrize("step", [1, 3000])
def test_adamw(hip, step):
    """All types at once, with masters and without, shapes of every alignment, a 0-d and an empty weight, more weights than a
    launch's table; the step and the rate given with each call."""
    rng = np.random.default_rng(step)
    kinds = [("float32", False), ("bfloat16", False), ("float16", False), ("bfloat16", True), ("float16", True)]
    shapes = [(1,), (), (0, 3), (4,), (7, 3), (4096,), (4097,), (129, 65), (3, 5000), (8191,)]
    weights = [(k, _weight(rng, s, *k)) for k in kinds for s in shapes]
    n, at = len(weights), [i for i, (k, _) in enumerate(weights) if k[1]]

    def fn(t, lr, *xs):
        p, g, m, v = (list(xs[i * n:(i + 1) * n]) for i in range(4))
        masters = [None] * n
        for i, w in zip(at, xs[4 * n:]):
            masters[i] = w
        p, m, v, w = F.adamw(p, g, m, v, t, lr, betas=BETAS, eps=EPS, weight_decay=DECAY, masters=masters)
        return [*p, *m, *v, *(w[i] for i in at)]

    f = L.compile(fn, device="hip")
    args = [_tensor(x[i], k[0] if i < 2 else "float32") for i in range(4) for k, x in weights]
    args += [_tensor(weights[i][1][4], "float32") for i in at]
    for lr in (1e-3, 0.3):
        got = [t.raw() for t in f(L.from_numpy(np.array(step, np.int64)), lr, *args)]
        masters = dict(zip(at, got[3 * n:]))
        for i, (k, x) in enumerate(weights):
            _check(x, (got[i], got[n + i], got[2 * n + i], masters.get(i)), k[0], step, lr, (k, x[0].shape))
    assert [st.kind for st in f.plan.steps] == ["adamw"]


def test_results_that_nothing_reads(hip):
    """Only the weights are returned: the moments have no place, and are not written."""
    rng = np.random.default_rng(1)
    x = _weight(rng, (300, 7), "bfloat16", True)
    f = L.compile(lambda p, g, m, v, w: [F.adamw([p], [g], [m], [v], 4, 0.1, BETAS, EPS, DECAY, [w])[0][0]], device="hip")
    (p,) = f(*(_tensor(a, dt) for a, dt in zip(x, ("bfloat16", "bfloat16", "float32", "float32", "float32"))))
    want = M.adamw(x[4], _up(x[1], "bfloat16"), x[2], x[3], 4, 0.1, BETAS, EPS, DECAY)[0]
    tol = M.adamw_tolerances(x[4], _up(x[1], "bfloat16"), x[2], x[3], 4, 0.1, BETAS, EPS, DECAY)[0]
    assert np.all(np.abs(_up(p.raw(), "bfloat16") - want) <= tol + M.U["bfloat16"] * np.abs(want))


@pytest.mark.parametrize("dtype,master", [("float32", False), ("bfloat16", True), ("float16", False)])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_pointers_off_16_bytes_in_place_and_scaled(hip, dtype, master, shift):
    """The C entry point on operands that start `shift` elements into their memory, each result over its operand, the gradients
    times a factor on the device; nothing past the tensors is written."""
    rng = np.random.default_rng(shift)
    n = 5000
    x = _weight(rng, (n,), dtype, master)
    size = D.size_of(dtype)
    devs = []
    for a in x:
        if a is not None:
            pad = np.full(n + 16, 9, a.dtype)
            pad[shift:shift + n] = a
            devs.append(Dev(pad))
    ptr = [d.ptr + shift * (size if i < 2 else 4) for i, d in enumerate(devs)]
    t = (nv.AdamwTensor * 1)(nv.AdamwTensor(param=ptr[0], grad=ptr[1], m=ptr[2], v=ptr[3], param_out=ptr[0], m_out=ptr[2], v_out=ptr[3],
                                            numel=n, dtype=DT[dtype]))
    if master:
        t[0].master = t[0].master_out = ptr[4]
    scalars = Dev(np.array([1e-2, 12.0], np.float64))
    scale = Dev(np.array([0.37], np.float32))
    desc = nv.AdamwDesc(count=1, beta1=BETAS[0], beta2=BETAS[1], eps=EPS, weight_decay=DECAY)
    nv.call("nhip_adamw", C.byref(desc), t, scalars.ptr, scalars.ptr + 8, scale.ptr)
    got = [d.get((n + 16,), a.dtype) for d, a in zip(devs, (a for a in x if a is not None))]
    for i, a in enumerate(got):
        assert np.all(a[:shift] == 9) and np.all(a[shift + n:] == 9)
    cut = [a[shift:shift + n] for a in got]
    assert np.array_equal(cut[1], x[1])
    _check(x, (cut[0], cut[2], cut[3], cut[4] if master else None), dtype, 12, 1e-2, shift, scale=0.37)


def test_refusals_of_the_entry_point(hip):
    one = Dev(np.zeros(64, np.float32))

    def call(desc=None, count=1, **fields):
        given = dict(param=one.ptr, grad=one.ptr, m=one.ptr, v=one.ptr, param_out=one.ptr, m_out=one.ptr, v_out=one.ptr, numel=4, dtype=0)
        given.update(fields)
        t = (nv.AdamwTensor * 1)(nv.AdamwTensor(**given))
        rates = dict(lr=0.1, step=1.0, beta1=0.9, beta2=0.9, eps=1e-8, weight_decay=0.0)
        rates.update(desc or {})
        nv.call("nhip_adamw", C.byref(nv.AdamwDesc(count=count, **rates)), t, None, None, None)

    for kw in (dict(count=-1), dict(desc={"beta1": 1.0}), dict(desc={"beta2": -0.1}), dict(desc={"eps": float("nan")}),
               dict(desc={"step": 0.0}), dict(numel=-1), dict(dtype=3), dict(grad=None), dict(param=None), dict(master=one.ptr),
               dict(master_out=one.ptr, dtype=1)):
        with pytest.raises(RuntimeError, match="nhip_adamw"):
            call(**kw)


def test_values_that_are_not_finite(hip):
    """A NaN or infinite gradient makes NaN of its own element alone; zeros with a second moment of zero stay zero."""
    f = L.compile(lambda p, g, m, v: [x[0] for x in F.adamw([p], [g], [m], [v], 1, 0.1, BETAS, 0.0, 0.0)[:3]], device="hip")
    g = np.ones(9, np.float32)
    g[2], g[5], g[7] = np.nan, np.inf, 0.0
    z = np.zeros(9, np.float32)
    p, m, v = (t.raw() for t in f(*(_tensor(a, "float32") for a in (z, g, z, z))))
    assert np.isnan(p[[2, 5, 7]]).all() and np.allclose(np.delete(p, [2, 5, 7]), -0.1, rtol=1e-6)  # 0 / 0 without an eps
    assert np.isnan(m[2]) and np.isinf(m[5]) and m[7] == 0 and np.isinf(v[5])


def test_past_32_bits_of_elements(hip):
    """2^31 + 77 bf16 weights whose last ones alone are not zero, stepped in place."""
    n = (1 << 31) + 77
    sizes = [2, 2, 4, 4]
    bufs = [Dev(nbytes=s * n) for s in sizes]
    for b, s in zip(bufs, sizes):
        nv.call("nhip_memset", C.c_void_p(b.ptr), 0, C.c_size_t(s * n))
    tail = [_bits([1.0, -2.0], "bfloat16"), _bits([0.5, 0.25], "bfloat16"), np.array([0.1, 0.2], np.float32), np.array([0.3, 0.4], np.float32)]
    for b, s, a in zip(bufs, sizes, tail):
        nv.h2d(b.ptr + s * (n - 2), a.ctypes.data, a.nbytes)
    p, g, m, v = (b.ptr for b in bufs)
    t = (nv.AdamwTensor * 1)(nv.AdamwTensor(param=p, grad=g, m=m, v=v, param_out=p, m_out=m, v_out=v, numel=n, dtype=1))
    desc = nv.AdamwDesc(count=1, lr=0.1, step=2.0, beta1=BETAS[0], beta2=BETAS[1], eps=EPS, weight_decay=DECAY)
    nv.call("nhip_adamw", C.byref(desc), t, None, None, None)
    got = []
    for b, s, a in zip(bufs, sizes, tail):
        out = np.empty_like(a)
        nv.d2h(out.ctypes.data, b.ptr + s * (n - 2), out.nbytes)
        got.append(out)
    _check((*tail, None), (got[0], got[2], got[3], None), "bfloat16", 2, 0.1, "tail")


def test_captured_and_replayed(hip):
    """A captured run replayed with other inputs in the same memory, and other captures of the plan between, against plain runs."""
    rng = np.random.default_rng(7)

    def fn(step, lr, p, g, m, v, w):
        new = F.adamw([p], [g], [m], [v], step, lr, BETAS, EPS, DECAY, [w])
        return [x[0] for x in new]

    dts = ["int32", "float64", "bfloat16", "bfloat16", "float32", "float32", "float32"]
    sets = [[np.array(i + 1, np.int32), np.array(0.1 / (i + 1)), *_weight(rng, (333, 17), "bfloat16", True)] for i in range(4)]
    plan = Plan(L.make_graph(fn)(*[L.empty(list(a.shape), dt, "meta") for a, dt in zip(sets[0], dts)]), "hip:0")
    ins, ws = [DeviceBuffer(0, a.nbytes) for a in sets[0]], DeviceBuffer(0, plan.workspace_bytes)
    ptrs = [b.ptr for b in ins]

    def put(arrays):
        for b, a in zip(ins, arrays):
            nv.h2d(b.ptr, np.ascontiguousarray(a).ctypes.data, a.nbytes)

    def read():
        out = []
        for loc in plan.output_locs:
            a = np.empty(loc.shape, D.storage(loc.dtype))
            nv.d2h(a.ctypes.data, ws.ptr + loc.offset * D.size_of(loc.dtype), a.nbytes)
            out.append(a)
        return out

    plain = []
    for s in sets:
        put(s)
        plan.run_in(ws.ptr, ptrs)
        plain.append(read())
    first, second = plan.capture(ws.ptr, ptrs), plan.capture(ws.ptr, ptrs)
    for i, (s, want) in enumerate(list(zip(sets, plain)) * 2):
        put(s)
        (first if i % 2 else second).launch()
        assert all(np.array_equal(a, b) for a, b in zip(read(), want))


@pytest.mark.parametrize("max_norm", [None, 0.01])
def test_the_optimizer_over_several_steps(hip, max_norm):
    """The small model trained for four steps with AdamW in place: the graph of the whole step captured from the third call on,
    every master, moment and the count as float64 steps from the state before with the gradients that the step returns, every
    weight its master rounded."""
    model, _ = W.build(W.TINY)
    opt = W.adamw(model, lr=2e-3)
    W.load(model, W.init_weights(model))
    W.load_adamw(opt)

    def train_step(model, opt, ids, targets):
        loss = W.loss_fn(model, ids, targets)
        loss.backward()
        grads = [p.grad for p in opt.params]
        kept = F.clip_grad_norm(grads, max_norm)[0] if max_norm else grads
        opt.step(max_norm=max_norm)
        return [loss, *kept]

    step = L.compile(train_step, device="hip")
    ids, targets = (L.from_numpy(a) for a in W.batch(W.TINY))
    state = [opt.params, opt.exp_avgs, opt.exp_avg_sqs, opt.masters]
    before = None
    for t in range(1, 5):
        if before is None:
            before = [[np.array(x.raw()) for x in xs] for xs in state]
        out = step(model, opt, ids, targets)
        grads = [np.array(x.raw()) for x in out[1:]]
        after = [[np.array(x._placed("hip:0").raw()) for x in xs] for xs in state]
        assert int(opt.steps._placed("hip:0").raw()) == t
        for i, g in enumerate(grads):
            start, m, v = before[3][i], before[1][i], before[2][i]
            grad = _up(g, "bfloat16")
            args = (start, grad, m, v, t, 2e-3, W.AdamW.BETAS, W.AdamW.EPS, W.AdamW.WEIGHT_DECAY)
            want, tol = M.adamw(*args), M.adamw_tolerances(*args)
            for a, b, limit in zip((after[3][i], after[1][i], after[2][i]), want, tol):
                assert np.all(np.abs(a - b) <= limit), (t, i)
            assert np.array_equal(after[0][i], _bits(after[3][i], "bfloat16")), (t, i)
        before = after
    assert len(step.plan.in_place_outputs) >= 4 * len(opt.params)
