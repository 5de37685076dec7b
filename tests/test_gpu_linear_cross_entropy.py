"""linear_cross_entropy on the GPU against plain float64 NumPy (tests/training_math.py), with the tolerances derived there."""

import ctypes as C

import numpy as np
import pytest

import lumen_amd as L
import lumen_amd.functional as F
from lumen_amd import dtypes as D
from lumen_amd import native as nv
from lumen_amd.compiler.plan import Plan
from lumen_amd.tensor import DeviceBuffer
from tests import training_math as M
from tests.hiputil import Dev

pytestmark = pytest.mark.gpu

IGNORED = -100


def _round(x, dtype):
    return np.asarray(D.to_numpy_values(D.from_values(np.asarray(x, np.float32), dtype), dtype), np.float64)


def _tensor(x, dtype):
    return L.Tensor(dtype, np.shape(x), "cpu", host=np.array(D.from_values(np.asarray(x, np.float32), dtype)))


def _values(t):
    return np.asarray(L.to_numpy(t), np.float64)


def _near(got, want, tol, what=""):
    assert got.shape == want.shape, what
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (what, np.abs(got - want)[bad].max(), int(bad.sum()), np.argwhere(bad)[0], got[bad][0], want[bad][0])


def _case(seed, t, k, v, dtype, ignored=0.2, std=1.0):
    rng = np.random.default_rng(seed)
    h, w = _round(rng.standard_normal((t, k)) * std, dtype), _round(rng.standard_normal((v, k)) * 1.5 * max(k, 1)**-0.5, dtype)
    target = np.where(rng.random(t) < ignored, IGNORED, rng.integers(0, v, t))
    return h, w, target, rng.standard_normal(t).astype(np.float32)


def _program(reduction="none"):
    def fn(h, w, target, g):
        losses, pull = L.vjp(lambda h, w: F.linear_cross_entropy(h, w, target, IGNORED, reduction), h, w)
        return [losses, *pull(g)]

    return fn


def _check(got, h, w, target, g, dtype, what=""):
    want = M.linear_cross_entropy(h, w, target, IGNORED, g)
    tol = M.linear_cross_entropy_tolerances(h, w, target, IGNORED, g, dtype)
    for name, a, b, t in zip(("losses", "dh", "dw"), got, want, tol):
        if a is not None:
            _near(a, b, t, (what, name))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_cotangents_of_ignored_rows_are_not_read_into_others(hip, dtype):
    """However large, or NaN: the largest cotangent of the rows that count sets the gradients' scale."""
    h, w, target, g = _case(21, 200, 64, 300, dtype)
    target[:4] = IGNORED
    f = L.compile(_program(), device="hip")
    args = [_tensor(h, dtype), _tensor(w, dtype), L.from_numpy(target)]
    want = [_values(a) for a in f(*args, L.from_numpy(np.where(target == IGNORED, 0, g).astype(np.float32)))]
    _check(want, h, w, target, g, dtype)
    for bad in (1e30, np.inf, np.nan):
        odd = np.where(target == IGNORED, bad, g).astype(np.float32)
        for a, b in zip(f(*args, L.from_numpy(odd)), want):
            assert np.array_equal(_values(a), b)


def test_rows_far_apart(hip):
    """Rows of a view whose rows lie 2^21 elements apart, of whole k tiles (read in place where they are near) and not."""
    for i, k in enumerate((64, 40)):
        h, w, target, g = _case(22 + i, 9, k, 300, "bfloat16")
        wide = np.zeros((9, 1 << 21), np.uint16)
        wide[:, :k] = D.from_values(h.astype(np.float32), "bfloat16")

        def fn(x, w, target, g):
            h = x[:, :k]
            losses, pull = L.vjp(lambda h, w: F.linear_cross_entropy(h, w, target, IGNORED, "none"), h, w)
            return [losses, *pull(g)]

        x = L.Tensor("bfloat16", wide.shape, "cpu", host=wide)
        for program in (fn, lambda *xs: [F.linear_cross_entropy(xs[0][:, :k], xs[1], xs[2], IGNORED, "none")]):
            out = L.compile(program, device="hip")(x, _tensor(w, "bfloat16"), L.from_numpy(target), L.from_numpy(g))
            _check([_values(a) for a in out], h, w, target, g, "bfloat16", k)


def test_rows_of_more_than_a_buffer(hip):
    """140000 rows of 8192 are 2^31 bytes and more: the weight's gradient is that of the few rows that are not zero, at both ends and
    around the boundary; a row of zeros has the loss log V."""
    t, k, v = 140000, 8192, 64
    at = np.array([0, 1, 69999, 70000, 131070, 131071, 131072, 139998, 139999])
    h, w, target, g = _case(20, len(at), k, v, "bfloat16", ignored=0.0)
    whole, targets, gs = np.zeros((t, k), np.uint16), np.zeros(t, np.int64), np.ones(t, np.float32)
    whole[at], targets[at], gs[at] = D.from_values(h.astype(np.float32), "bfloat16"), target, g

    def fn(h, w, target, g):
        losses, pull = L.vjp(lambda w: F.linear_cross_entropy(h, w, target, IGNORED, "none"), w)
        return [losses, *pull(g)]

    f = L.compile(fn, device="hip")
    x = L.Tensor("bfloat16", whole.shape, "cpu", host=whole)
    losses, dw = (_values(a) for a in f(x, _tensor(w, "bfloat16"), L.from_numpy(targets), L.from_numpy(gs)))
    want = M.linear_cross_entropy(h, w, target, IGNORED, g)
    tol = M.linear_cross_entropy_tolerances(h, w, target, IGNORED, g, "bfloat16")
    _near(losses[at], want[0], tol[0], "losses")
    _near(dw, want[2], tol[2], "dw")
    rest = np.delete(losses, at)
    assert np.abs(rest - np.log(v)).max() <= 4 * 2.0**-24 * np.log(v) + 64 * 2.0**-24


CASES = [
    # rows, k, classes, dtype: one row, one class, one element; ragged ones; tiles of 128 and of 256 rows; parts of k
    (1, 64, 64, "bfloat16"), (1, 8, 1, "float16"), (5, 1, 3, "bfloat16"), (3, 64, 5003, "bfloat16"), (777, 520, 5003, "float16"),
    (300, 128, 1000, "bfloat16"), (513, 191, 4097, "bfloat16"), (64, 256, 65, "float16"), (4096, 64, 4160, "bfloat16"),
    (4100, 128, 4090, "float16"), (129, 64, 20001, "bfloat16"), (2000, 72, 63, "bfloat16"),
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_both_directions(hip, case):
    t, k, v, dtype = CASES[case]
    h, w, target, g = _case(case, t, k, v, dtype)
    f = L.compile(_program(), device="hip")
    args = [_tensor(h, dtype), _tensor(w, dtype), L.from_numpy(target.astype(np.int32 if case % 2 else np.int64)), L.from_numpy(g)]
    for _ in range(2):
        _check([_values(a) for a in f(*args)], h, w, target, g, dtype)
    assert [st.kind for st in f.plan.steps] == ["head_loss"]
    forward = L.compile(lambda h, w, target: [F.linear_cross_entropy(h, w, target, IGNORED, "none")], device="hip")
    _check([_values(forward(*args[:3])[0]), None, None], h, w, target, g, dtype)


@pytest.mark.parametrize("dtype,rows,k,v", [("bfloat16", 1100, 64, 700), ("float16", 1300, 65, 333), ("bfloat16", 4096, 64, 4100)])
def test_pieces(hip, dtype, rows, k, v):
    """Rows in pieces whose weight gradients add up, and rows of one piece: the same losses and input gradients, bit for bit."""
    h, w, target, g = _case(rows, rows, k, v, dtype)
    args = [_tensor(h, dtype), _tensor(w, dtype), L.from_numpy(target), L.from_numpy(g)]
    got = []
    for size in (1, 600 * 2 * (-(-v // 64) * 64), 1 << 30):
        with L.config.compiler.patch(head_piece_bytes=size):
            f = L.compile(_program(), device="hip")
            got.append([_values(a) for a in f(*args)])
        _check(got[-1], h, w, target, g, dtype, size)
    for other in got[1:]:
        assert np.array_equal(got[0][0], other[0])


@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("dtype,scale", [("bfloat16", 1.0), ("float16", 4096.0)])
def test_reductions_with_a_scaled_loss(hip, reduction, dtype, scale):
    """The mean and the sum over the rows that count, with a runtime scale as their cotangent."""
    h, w, target, _ = _case(5, 333, 128, 777, dtype)

    def fn(h, w, target, scale):
        loss, pull = L.vjp(lambda h, w: F.linear_cross_entropy(h, w, target, IGNORED, reduction), h, w)
        return [loss, *pull(scale.to("float32"))]

    f = L.compile(fn, device="hip")
    n = (target != IGNORED).sum()
    g = np.full(len(h), scale / (n if reduction == "mean" else 1))
    got = [_values(a) for a in f(_tensor(h, dtype), _tensor(w, dtype), L.from_numpy(target), scale)]
    losses = M.linear_cross_entropy(h, w, target, IGNORED, g)[0]
    tol = M.linear_cross_entropy_tolerances(h, w, target, IGNORED, g, dtype)[0]
    total, limit = losses.sum(), tol.sum() + M.F32 * len(h) * losses.sum()
    assert abs(got[0] - (total / n if reduction == "mean" else total)) <= (limit / n if reduction == "mean" else limit)
    _check([None, *got[1:]], h, w, target, g * (1 + 0.0), dtype)
    assert [st.kind for st in f.plan.steps].count("head_loss") == 1


def test_no_row_counts(hip):
    h, w, target, _ = _case(6, 70, 64, 100, "bfloat16", ignored=1.1)
    f = L.compile(_program("mean"), device="hip")
    loss, dh, dw = (_values(a) for a in f(_tensor(h, "bfloat16"), _tensor(w, "bfloat16"), L.from_numpy(target), L.from_numpy(np.float32(1))))
    assert loss == 0 and not dh.any() and not dw.any()


def test_ignored_rows_of_anything_and_targets_outside(hip):
    """Ignored rows of NaN and infinities change nothing, bit for bit; a target below 0 or past the classes is clamped."""
    h, w, target, g = _case(7, 400, 128, 500, "bfloat16")
    f = L.compile(_program(), device="hip")

    def run(h, target):
        return [np.array(a.raw()) for a in f(_tensor(h, "bfloat16"), _tensor(w, "bfloat16"), L.from_numpy(target), L.from_numpy(g))]

    clean = run(h, target)
    bad = h.copy()
    bad[target == IGNORED] = np.where(np.arange(h.shape[1]) % 2, np.nan, np.inf)
    for a, b in zip(clean, run(bad, target)):
        assert np.array_equal(a, b)
    kept = np.flatnonzero(target != IGNORED)
    outside, inside = target.copy(), target.copy()
    outside[kept[:3]], inside[kept[:3]] = [-1, 500, 1 << 40], [0, 499, 499]
    for a, b in zip(run(h, outside), run(h, inside)):
        assert np.array_equal(a, b)


def test_logits_far_apart(hip):
    """A row whose largest logit is 200 above the rest, and one far below its target: losses of nothing and of 200, gradients of the
    target's class alone that do not cancel."""
    k, v = 64, 300
    w = np.zeros((v, k))
    w[:, 0] = -100.0
    w[7, 0] = 100.0
    w[:, 1] = np.arange(v) % 2
    h = np.zeros((3, k))
    h[:, 0] = 1.0
    h[2, :2] = [0.0, 1.0]
    target, g = np.array([7, 9, 4]), np.array([1.0, -2.0, 0.5], np.float32)
    f = L.compile(_program(), device="hip")
    got = [_values(a) for a in f(_tensor(h, "bfloat16"), _tensor(w, "bfloat16"), L.from_numpy(target), L.from_numpy(g))]
    _check(got, h, w, target, g, "bfloat16")
    assert got[0][0] == 0 and got[0][1] == 200


def test_cotangents_of_any_size_in_float16(hip):
    """Cotangents of 1e-7 and of 3 (a mean over many rows, a scaled sum): the rounding of the logits' gradients is relative to
    the largest."""
    for size in (1e-7, 1.0, 3.0):
        h, w, target, g = _case(8, 200, 64, 900, "float16")
        g = (g * size).astype(np.float32)
        f = L.compile(_program(), device="hip")
        got = [_values(a) for a in f(_tensor(h, "float16"), _tensor(w, "float16"), L.from_numpy(target), L.from_numpy(g))]
        _check(got, h, w, target, g, "float16", size)


def test_views_and_one_gradient(hip):
    """Rows read through a view's strides, a row broadcast to all, and gradients of which one is read."""
    rng = np.random.default_rng(9)
    base, w = _round(rng.standard_normal((200, 192)), "bfloat16"), _round(rng.standard_normal((300, 128)) / 8, "bfloat16")
    target = rng.integers(0, 300, 200)
    g = rng.standard_normal(200).astype(np.float32)

    def only(which):
        def fn(base, w, target, g):
            _, pull = L.vjp(lambda h, w: F.linear_cross_entropy(h, w, target, reduction="none"), base[:, 64:], w)
            return [pull(g)[which]]

        return fn

    want = M.linear_cross_entropy(base[:, 64:], w, target, IGNORED, g)
    tol = M.linear_cross_entropy_tolerances(base[:, 64:], w, target, IGNORED, g, "bfloat16")
    args = [_tensor(base, "bfloat16"), _tensor(w, "bfloat16"), L.from_numpy(target), L.from_numpy(g)]
    for which in (0, 1):
        (got,) = L.compile(only(which), device="hip")(*args)
        _near(_values(got), want[1 + which], tol[1 + which], which)

    row = base[:1, 64:]

    def spread(row, w, target):
        return [F.linear_cross_entropy(row.expand(200, 128), w, target, reduction="none")]

    (got,) = L.compile(spread, device="hip")(_tensor(row, "bfloat16"), *args[1:3])
    all_rows = np.repeat(row, 200, 0)
    _near(_values(got), M.linear_cross_entropy(all_rows, w, target, IGNORED, g)[0],
          M.linear_cross_entropy_tolerances(all_rows, w, target, IGNORED, g, "bfloat16")[0])


def test_a_cotangent_that_depends_on_the_loss(hip):
    """Two steps: the losses first, then the gradients for twice the mean."""
    h, w, target, _ = _case(10, 150, 64, 200, "bfloat16")

    def fn(h, w, target):
        loss, pull = L.vjp(lambda h, w: F.linear_cross_entropy(h, w, target), h, w)
        return [loss, *pull(loss * 2.0)]

    f = L.compile(fn, device="hip")
    loss, dh, dw = (_values(a) for a in f(_tensor(h, "bfloat16"), _tensor(w, "bfloat16"), L.from_numpy(target)))
    n = (target != IGNORED).sum()
    g = np.full(len(h), 2 * float(loss) / n)
    _check([None, dh, dw], h, w, target, g, "bfloat16")
    assert [st.kind for st in f.plan.steps].count("head_loss") == 2


def test_captured_and_replayed(hip):
    """One capture replayed with other operands in the same memory, a second capture of the plan between, against plain runs."""
    dts = ["float16", "float16", "int64", "float32"]
    sets = []
    for seed in range(4):
        h, w, target, g = _case(seed, 300, 96, 500, "float16")
        sets.append([D.from_values(h.astype(np.float32), "float16"), D.from_values(w.astype(np.float32), "float16"), target, g])
    with L.config.compiler.patch(head_piece_bytes=1):
        plan = Plan(L.make_graph(_program())(*[L.empty(list(a.shape), dt, "meta") for a, dt in zip(sets[0], dts)]), "hip:0")
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


def test_refusals_of_the_entry_point(hip):
    one = Dev(nbytes=1 << 16)

    def call(h=one.ptr, g=one.ptr, dh=one.ptr, ws=one.ptr, **kw):
        fields = dict(rows=2, classes=3, k=64, h_m=64, w_n=64, ignore_index=-100, piece_bytes=1 << 20, dtype=1, target_dtype=0)
        fields.update(kw)
        nv.call("nhip_head_loss", C.byref(nv.HeadDesc(**fields)), h, one.ptr, one.ptr, g, None, dh, None, ws)

    for kw in (dict(rows=-1), dict(classes=0), dict(k=0), dict(dtype=0), dict(target_dtype=2), dict(w_n=63), dict(h_m=-64), dict(piece_bytes=-1),
               dict(classes=1 << 22), dict(classes=1 << 21, k=1 << 10, w_n=1 << 10, h_m=1 << 10), dict(g=None), dict(ws=None),
               dict(ws=one.ptr + 16), dict(dh=one.ptr + 2), dict(g=None, dh=None, h=one.ptr + 2), dict(rows=1 << 31), dict(h=None)):
        with pytest.raises(RuntimeError, match="nhip_head_loss"):
            call(**kw)


@pytest.mark.parametrize("given", [True, False])
def test_losses_alone_stay_within_the_workspace_of_the_call(hip, given):
    """With cotangents and neither gradient wanted the workspace is the gradients', which holds the maxima and sums of one piece's
    rows and is smaller than those of all rows. What lies behind it is left as it was."""
    t, k, v = 20000, 64, 3000
    h, w, target, g = _case(31, t, k, v, "bfloat16")
    d = nv.HeadDesc(rows=t, classes=v, k=k, h_m=k, w_n=k, ignore_index=IGNORED, piece_bytes=1, dtype=1, target_dtype=1)
    size = C.c_size_t()
    nv.call("nhip_head_loss_workspace", C.byref(d), int(given), C.byref(size))
    blocks = -(-v // 64)
    assert not given or size.value < t * blocks * 8
    behind = t * blocks * 8
    ws = Dev(np.full(size.value + behind, 0x5a, np.uint8))
    dev = [Dev(np.array(D.from_values(x.astype(np.float32), "bfloat16"))) for x in (h, w)] + [Dev(target.astype(np.int64)), Dev(g)]
    out = Dev(np.full(t, np.nan, np.float32))
    nv.call("nhip_head_loss", C.byref(d), dev[0].ptr, dev[1].ptr, dev[2].ptr, dev[3].ptr if given else None, out.ptr, None, None, ws.ptr)
    losses = out.get(t, np.float32)
    for lo in range(0, t, 4000):
        part = (h[lo:lo + 4000], w, target[lo:lo + 4000], IGNORED, g[lo:lo + 4000])
        _near(losses[lo:lo + 4000], M.linear_cross_entropy(*part)[0], M.linear_cross_entropy_tolerances(*part, "bfloat16")[0])
    assert np.all(ws.get(size.value + behind, np.uint8)[size.value:] == 0x5a)


@pytest.mark.parametrize("classes,bad", [(65, [64]), (64, [5]), (500, [130]), (9000, range(4096)), (9000, [8999])])
def test_a_nan_among_the_weights_reaches_every_loss(hip, classes, bad):
    """Wherever its class lies: alone in the last block of 64, among others, in every block that a wavefront adds up."""
    t, k = 40, 64
    h, w, target, g = _case(41, t, k, classes, "bfloat16")
    target[:3] = [IGNORED, 1, 2]
    w[list(bad), 7] = np.nan
    args = [_tensor(h, "bfloat16"), _tensor(w, "bfloat16"), L.from_numpy(target)]
    forward = L.compile(lambda h, w, target: [F.linear_cross_entropy(h, w, target, IGNORED, "none")], device="hip")
    both = L.compile(_program(), device="hip")(*args, L.from_numpy(g))
    kept = target != IGNORED
    for losses in (forward(*args)[0], both[0]):
        losses = _values(losses)
        assert np.isnan(losses[kept]).all() and not losses[~kept].any()
    assert np.isnan(_values(both[1])[kept]).all() and np.isnan(_values(both[2])).all()


def test_classes_of_minus_infinity_count_for_nothing(hip):
    """Logits of -inf, alone in the last block of 64 and throughout a wavefront's: the losses of the other classes."""
    k = 64
    h, w, target, g = _case(42, 40, k, 4160, "bfloat16")
    h[:, 7] = _round(np.abs(h[:, 7]) + 0.5, "bfloat16")
    target %= 64
    forward = L.compile(lambda h, w, target: [F.linear_cross_entropy(h, w, target, IGNORED, "none")], device="hip")
    for classes in (65, 4160):
        some = w[:classes].copy()
        some[64:, 7] = -np.inf
        (losses,) = forward(_tensor(h, "bfloat16"), _tensor(some, "bfloat16"), L.from_numpy(target))
        _check([_values(losses), None, None], h, w[:64], target, g, "bfloat16")


@pytest.mark.parametrize("target_type", ["int32", "int64"])
def test_float32_losses_with_and_without_gradients(hip, target_type):
    """As primitives, whose losses alone are the step of an eval loss over a product."""
    h, w, target, g = _case(51, 70, 33, 130, "float32")
    h, w = h.astype(np.float32), w.astype(np.float32)
    args = [L.from_numpy(a) for a in (h, w, target.astype(target_type))]
    forward = L.compile(lambda h, w, target: [F.linear_cross_entropy(h, w, target, IGNORED, "none")], device="hip")
    _check([_values(forward(*args)[0]), None, None], h, w, target, g, "float32")
    assert "linear_cross_entropy" in [st.kind for st in forward.plan.steps]
    _check([_values(a) for a in L.compile(_program(), device="hip")(*args, L.from_numpy(g))], h, w, target, g, "float32")


def test_float32_losses_of_views(hip):
    rng = np.random.default_rng(52)
    base, wide = rng.standard_normal((3, 10, 96)).astype(np.float32), rng.standard_normal((130, 80)).astype(np.float32)
    target = rng.integers(0, 130, (3, 10))
    f = L.compile(lambda x, w, t: [F.linear_cross_entropy(x[:, :, 32:], w[:, 16:], t, reduction="none")], device="hip")
    (got,) = f(*(L.from_numpy(a) for a in (base, wide, target)))
    rows = (base[:, :, 32:].reshape(30, 64), wide[:, 16:], target.reshape(30), IGNORED, np.ones(30))
    _near(_values(got).reshape(30), M.linear_cross_entropy(*rows)[0], M.linear_cross_entropy_tolerances(*rows, "float32")[0])
    assert "linear_cross_entropy" in [st.kind for st in f.plan.steps]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_no_rows(hip, dtype):
    """No loss, and gradients of zeros: of a step that nothing but the cotangent goes into, and of a mean."""
    h, w, target, g = np.zeros((0, 24)), _round(np.ones((50, 24)), dtype), np.zeros(0, np.int64), np.zeros(0, np.float32)
    args = [_tensor(h, dtype), _tensor(w, dtype), L.from_numpy(target)]
    for out in (L.compile(_program(), device="hip")(*args, L.from_numpy(g)), L.compile(_program("mean"), device="hip")(*args, L.from_numpy(np.array(2.0, np.float32)))):
        losses, dh, dw = (_values(a) for a in out)
        assert losses.size in (0, 1) and not losses.any() and dh.shape == h.shape and dw.shape == w.shape and not dw.any()
    (mean,) = L.compile(lambda h, w, t: [F.linear_cross_entropy(h, w, t)], device="hip")(*args)
    assert float(_values(mean)) == 0.0
