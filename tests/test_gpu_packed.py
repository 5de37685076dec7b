"""packed_attention on the GPU against plain float64 NumPy (tests/training_math.py), with the tolerances derived there."""

import ctypes as C

import numpy as np
import pytest

import lumen_amd as L
import lumen_amd.functional as F
from lumen_amd import dtypes as D
from lumen_amd import native as nv
from lumen_amd.graph import prims
from tests import training_math as M
from tests.hiputil import Dev

pytestmark = pytest.mark.gpu


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


def _program(causal, scale=None):
    def fn(q, k, v, offsets, do):
        o, pull = L.vjp(lambda q, k, v: F.packed_attention(q, k, v, offsets, scale=scale, is_causal=causal), q, k, v)
        return [o, *pull(do)]

    return fn


CASES = [
    # lengths, first, tokens, n, nkv, d, dv, causal, dtype
    ([1], 0, 1, 1, 1, 8, 8, True, "bfloat16"),
    ([1], 0, 1, 2, 1, 64, 64, False, "float16"),
    ([61, 17, 19], 0, 97, 4, 2, 64, 64, True, "bfloat16"),
    ([64, 128, 63, 129, 1, 0, 65], 3, 460, 2, 2, 64, 64, True, "float16"),
    ([64, 128, 63, 129, 1, 0, 65], 3, 460, 2, 1, 128, 128, True, "bfloat16"),
    ([64, 128, 63, 129, 1, 0, 65], 3, 460, 2, 2, 128, 128, False, "float16"),
    ([0, 0, 300, 0], 0, 300, 8, 8, 32, 32, True, "bfloat16"),
    ([700], 5, 800, 3, 3, 80, 80, False, "bfloat16"),
    ([33, 257, 255, 256], 0, 801, 8, 2, 64, 128, True, "bfloat16"),
    ([33, 257, 255, 256], 1, 803, 4, 4, 128, 40, False, "float16"),
    ([2, 3, 1, 1, 5, 8] * 20, 0, 420, 2, 2, 64, 64, True, "bfloat16"),
    ([], 0, 70, 2, 2, 64, 64, True, "bfloat16"),
    ([0], 70, 70, 2, 2, 64, 64, False, "bfloat16"),
    ([1100, 40], 0, 1140, 2, 2, 128, 128, True, "bfloat16"),
]


@pytest.mark.parametrize("store", [True, False])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_packed(hip, case, store):
    """Both directions, dS stored for dQ and computed again."""
    lengths, first, tokens, n, nkv, d, dv, causal, dtype = CASES[case]
    rng = np.random.default_rng(case)
    x = {k: _round(v, dtype) for k, v in M.packed_inputs(rng, tokens, n, nkv, d, dv).items()}
    offsets = M.offsets_of(lengths, first)
    want, tol = M.packed(x, offsets, causal, d**-0.5, dtype)
    args = [_tensor(x[k], dtype) for k in "qkv"] + [L.from_numpy(offsets.astype(np.int32 if case % 2 else np.int64)), _tensor(x["do"], dtype)]
    with L.config.compiler.patch(attention_store_ds=store):
        f = L.compile(_program(causal), device="hip")
        for _ in range(2):
            for name, a, w, t in zip(("o", "dq", "dk", "dv"), f(*args), want, tol):
                _near(_values(a), w, t, name)
    assert [st.kind for st in f.plan.steps] == ["packed_fwd", "packed_bwd"]


def test_nothing_of_another_sequence_or_of_none(hip):
    """NaN and infinities in the tokens of no sequence and in whole sequences: every other sequence's results are, bit for bit,
    those without them."""
    rng = np.random.default_rng(2)
    lengths = [70, 1, 64, 200, 30, 129]
    offsets = M.offsets_of(lengths, 9)
    t = int(offsets[-1]) + 40
    x = M.packed_inputs(rng, t, 4, 2, 64)
    f = L.compile(_program(True), device="hip")

    def run(x):
        args = [_tensor(x[k], "bfloat16") for k in "qkv"] + [L.from_numpy(offsets.astype(np.int32)), _tensor(x["do"], "bfloat16")]
        return [np.array(o.raw()) for o in f(*args)]

    clean = run(x)
    bad = {k: v.copy() for k, v in x.items()}
    for v in bad.values():
        v[:9], v[offsets[-1]:] = np.nan, np.inf
        v[offsets[1]:offsets[2]], v[offsets[3]:offsets[4]] = np.inf, np.nan
    kept = np.ones(t, bool)
    kept[offsets[1]:offsets[2]] = kept[offsets[3]:offsets[4]] = False
    for a, b in zip(clean, run(bad)):
        assert np.array_equal(a[kept], b[kept])
        assert not a[:9].any() and not a[offsets[-1]:].any()


def test_heads_of_a_merged_projection(hip):
    """Queries, keys and values read in place through a merged projection's strides, and gradients joined again."""
    rng = np.random.default_rng(3)
    t, n, nkv, d = 333, 8, 2, 64
    offsets = M.offsets_of([100, 200, 30])
    qkv, do = (_round(rng.standard_normal(s), "bfloat16") for s in ((t, (n + 2 * nkv) * d), (t, n, d)))

    def heads(qkv):
        return (qkv[:, lo * d:hi * d].reshape(t, hi - lo, d) for lo, hi in ((0, n), (n, n + nkv), (n + nkv, n + 2 * nkv)))

    def fn(qkv, offsets, do):
        o, pull = L.vjp(lambda qkv: F.packed_attention(*heads(qkv), offsets), qkv)
        return [o, pull(do)[0]]

    f = L.compile(fn, device="hip")
    o, dqkv = (_values(a) for a in f(_tensor(qkv, "bfloat16"), L.from_numpy(offsets), _tensor(do, "bfloat16")))
    q, k, v = (a for a in heads(qkv))
    want, tol = M.packed({"q": q, "k": k, "v": v, "do": do}, offsets, True, d**-0.5, "bfloat16")
    _near(o, want[0], tol[0], "o")
    for name, a, w, tt in zip("qkv", heads(dqkv), want[1:], tol[1:]):
        _near(a, w, tt, name)
    assert [st.kind for st in f.plan.steps if st.kind != "view"][:2] == ["packed_fwd", "packed_bwd"]  # nothing is copied for them


@pytest.mark.parametrize("limit", [40, 60])
def test_ds_that_does_not_fit(hip, limit):
    """The workspace holds `limit` dS tiles of a head: the offsets on the device decide whether they are stored or computed again;
    the same compiled function with offsets of which all fit and of which they do not."""
    rng = np.random.default_rng(limit)
    t, n, d = 1024, 2, 64
    x = {k: _round(v, "bfloat16") for k, v in M.packed_inputs(rng, t, n, n, d).items()}
    with L.config.compiler.patch(attention_ds_max_bytes=limit * n * 128 * 64 * 2):
        f = L.compile(_program(True), device="hip")
        for lengths in ([1024, 0, 0, 0], [256, 256, 256, 256], [100, 500, 300, 100], [1, 2, 3, 4]):
            offsets = M.offsets_of(lengths)
            want, tol = M.packed(x, offsets, True, d**-0.5, "bfloat16")
            args = [_tensor(x[k], "bfloat16") for k in "qkv"] + [L.from_numpy(offsets), _tensor(x["do"], "bfloat16")]
            for name, a, w, tt in zip(("o", "dq", "dk", "dv"), f(*args), want, tol):
                _near(_values(a), w, tt, (lengths, name))


@pytest.mark.parametrize("lengths,n,nkv,d,dtype,causal", [
    ([700, 1, 385, 214], 32, 16, 64, "bfloat16", True), ([129, 900, 0, 300], 16, 16, 128, "float16", True),
    ([129, 130, 0, 300, 257], 64, 16, 64, "bfloat16", False), ([513, 1, 0, 200, 64], 48, 24, 128, "bfloat16", True)])
@pytest.mark.parametrize("limit", [0, 60, 1000])
def test_heads_enough_for_whole_key_blocks(hip, lengths, n, nkv, d, dtype, causal, limit):
    """So many key blocks that none is done in parts: dS computed again, stored if it fits (it does not), and stored. With the most
    heads the forward's workgroups do not all run at once, and a table orders them."""
    rng = np.random.default_rng(12)
    offsets = M.offsets_of(lengths, 2)
    t = int(offsets[-1]) + 131
    x = {k: _round(v, dtype) for k, v in M.packed_inputs(rng, t, n, nkv, d).items()}
    want, tol = M.packed(x, offsets, causal, d**-0.5, dtype)
    args = [_tensor(x[k], dtype) for k in "qkv"] + [L.from_numpy(offsets), _tensor(x["do"], dtype)]
    with L.config.compiler.patch(attention_ds_max_bytes=limit * n * 128 * 64 * 2, attention_store_ds=limit > 0):
        f = L.compile(_program(causal), device="hip")
        for name, a, w, tt in zip(("o", "dq", "dk", "dv"), f(*args), want, tol):
            _near(_values(a), w, tt, name)


def test_rows_far_apart_within_a_sequence(hip):
    """A sequence whose rows span more than 2^31 bytes, read in place through a view's strides; a padded head dim, whose loads reach
    2^31 bytes, is refused."""
    t, d, wide = 1200, 64, 1 << 20
    rng = np.random.default_rng(14)
    x = {k: _round(v, "bfloat16") for k, v in M.packed_inputs(rng, t, 1, 1, d).items()}
    offsets = M.offsets_of([1150, 50])
    base = np.zeros((t, wide), np.uint16)
    for i, k in enumerate("qkv"):
        base[:, i * d:(i + 1) * d] = D.from_values(x[k].reshape(t, d).astype(np.float32), "bfloat16")
    base = L.Tensor("bfloat16", base.shape, "cpu", host=base).to(device="hip")

    def program(d):
        def fn(base, offsets, do):
            q, k, v = (base[:, i * d:(i + 1) * d].reshape(t, 1, d) for i in range(3))
            o, pull = L.vjp(lambda q, k, v: F.packed_attention(q, k, v, offsets), q, k, v)
            return [o, *pull(do)]

        return fn

    want, tol = M.packed(x, offsets, True, d**-0.5, "bfloat16")
    f = L.compile(program(d), device="hip")
    for name, a, w, tt in zip(("o", "dq", "dk", "dv"), f(base, L.from_numpy(offsets), _tensor(x["do"], "bfloat16")), want, tol):
        _near(_values(a), w, tt, name)
    with pytest.raises(RuntimeError, match="2 GiB"):
        L.compile(program(40), device="hip")(base, L.from_numpy(offsets), _tensor(x["do"][:, :, :40], "bfloat16"))


def test_no_tokens_broadcasts_and_single_gradients(hip):
    """No tokens at all; keys and values broadcast over the heads and a cotangent of one number; each gradient alone."""
    offsets = np.array([0, 0, 0], np.int32)
    none = np.zeros((0, 2, 64))
    out = L.compile(_program(True), device="hip")(*(_tensor(none, "bfloat16") for _ in range(3)), L.from_numpy(offsets), _tensor(none, "bfloat16"))
    assert [_values(a).shape for a in out] == [none.shape] * 4

    rng = np.random.default_rng(15)
    t, n, d = 150, 4, 64
    x = {k: _round(v, "bfloat16") for k, v in M.packed_inputs(rng, t, n, 1, d).items()}
    x["do"] = np.full((t, n, d), 0.5)
    offsets = M.offsets_of([100, 47])
    whole = dict(x, k=np.repeat(x["k"], n, 1), v=np.repeat(x["v"], n, 1))
    want, tol = M.packed(whole, offsets, True, d**-0.5, "bfloat16")
    args = [_tensor(x[k], "bfloat16") for k in "qkv"] + [L.from_numpy(offsets)]

    def gradients(q, k, v, offsets):
        def loss(q, k, v):
            return F.sum(F.packed_attention(q, k, v, offsets).float()) * 0.5

        _, pull = L.vjp(loss, q, k.expand(t, n, d), v.expand(t, n, d))
        return list(pull(prims.full((), 1.0, "float32")))

    for name, a, w, tt in zip(("dq", "dk", "dv"), L.compile(gradients, device="hip")(*args), want[1:], tol[1:]):
        _near(_values(a), w, tt, name)
    for i in range(3):
        (a,) = L.compile(lambda *xs: [gradients(*xs)[i]], device="hip")(*args)
        _near(_values(a), want[1 + i], tol[1 + i], i)


def test_gradients_of_short_sequences_take_o_whole(hip):
    """Rounding is off by a step's half at most, evenly: of values whose logarithms are spread evenly 2^-8 sqrt(0.541 / 3) =
    1.66e-3 in the mean square (the mean of 1 / m^2 for a mantissa m of [1, 2) being 0.541). Of dQ and dK the result, dS and the
    forward's P are rounded: sqrt(3) of it. O's own rounding, the same in every dS of a row, would add more than one of them."""
    rng = np.random.default_rng(13)
    offsets = M.offsets_of([2, 3, 4, 5, 6, 7, 8] * 20)
    t, n, d = int(offsets[-1]), 4, 64
    x = {k: _round(v, "bfloat16") for k, v in M.packed_inputs(rng, t, n, n, d).items()}
    want, _ = M.packed(x, offsets, True, d**-0.5, "bfloat16")
    f = L.compile(_program(True), device="hip")
    got = f(*[_tensor(x[k], "bfloat16") for k in "qkv"], L.from_numpy(offsets), _tensor(x["do"], "bfloat16"))
    for name, a, w in list(zip(("o", "dq", "dk", "dv"), got, want))[1:3]:
        assert np.sqrt(((_values(a) - w) ** 2).sum() / (w**2).sum()) < 3**0.5 * 1.66e-3, name


def test_more_sequences_than_a_pass_of_the_builder(hip):
    """2500 sequences, mostly of a few tokens, some empty, some longer than eight blocks: 1024 of them a pass."""
    rng = np.random.default_rng(8)
    lengths = rng.integers(0, 4, 2500)
    lengths[[5, 1023, 1024, 2100]] = [1500, 200, 1100, 64]
    offsets = M.offsets_of(lengths, 2)
    t = int(offsets[-1]) + 3
    x = {k: _round(v, "float16") for k, v in M.packed_inputs(rng, t, 1, 1, 64).items()}
    want, tol = M.packed(x, offsets, True, 0.125, "float16")
    f = L.compile(_program(True), device="hip")
    args = [_tensor(x[k], "float16") for k in "qkv"] + [L.from_numpy(offsets.astype(np.int32)), _tensor(x["do"], "float16")]
    for name, a, w, tt in zip(("o", "dq", "dk", "dv"), f(*args), want, tol):
        _near(_values(a), w, tt, name)


def test_offsets_that_decrease_or_leave_the_tokens_are_clamped(hip):
    """Each offset is read as clamped into [the one before, tokens]."""
    rng = np.random.default_rng(9)
    t = 150
    x = {k: _round(v, "bfloat16") for k, v in M.packed_inputs(rng, t, 2, 2, 64).items()}
    f = L.compile(_program(False), device="hip")
    for given, read in (([-5, 60, 40, 90, 1 << 30, 7], [0, 60, 60, 90, 150, 150]), ([300, 0, 0, 0, 0, 0], [150] * 6),
                        ([10, 5, 5, -9, 20, 30], [10, 10, 10, 10, 20, 30])):
        want, tol = M.packed(x, read, False, 0.125, "bfloat16")
        args = [_tensor(x[k], "bfloat16") for k in "qkv"] + [L.from_numpy(np.array(given, np.int32)), _tensor(x["do"], "bfloat16")]
        for name, a, w, tt in zip(("o", "dq", "dk", "dv"), f(*args), want, tol):
            _near(_values(a), w, tt, (given, name))


@pytest.mark.parametrize("lengths,tokens,n,nkv,d", [([3000, 5, 1091], 4096, 4, 2, 128), ([2048] * 4, 8192, 2, 2, 64)])
def test_long_sequences_against_flash_attention_of_each(hip, lengths, tokens, n, nkv, d):
    """Each sequence's results are those of flash_attention on it alone, up to their roundings: both within the same tolerance of
    float64, so within twice it (as 4 U of the largest value here) of one another; the same bits in every call."""
    rng = np.random.default_rng(10)
    x = {k: _round(v, "bfloat16") for k, v in M.packed_inputs(rng, tokens, n, nkv, d).items()}
    offsets = M.offsets_of(lengths)
    f = L.compile(_program(True), device="hip")
    args = [_tensor(x[k], "bfloat16") for k in "qkv"] + [L.from_numpy(offsets.astype(np.int32)), _tensor(x["do"], "bfloat16")]
    first = [np.array(a.raw()) for a in f(*args)]
    again = [np.array(a.raw()) for a in f(*args)]
    assert all(np.array_equal(a, b) for a, b in zip(first, again))
    got = [np.asarray(D.to_numpy_values(a, "bfloat16"), np.float64) for a in first]

    def alone(q, k, v, do):
        o, pull = L.vjp(lambda q, k, v: F.flash_attention(q, k, v, is_causal=True), q, k, v)
        return [o, *pull(do)]

    g = L.compile(alone, device="hip")
    for lo, hi in zip(offsets, offsets[1:]):
        one = g(*(_tensor(x[k][None, lo:hi], "bfloat16") for k in ("q", "k", "v", "do")))
        for name, a, b in zip(("o", "dq", "dk", "dv"), got, one):
            b = _values(b)[0]
            assert np.abs(a[lo:hi] - b).max() <= 4 * M.U["bfloat16"] * max(1.0, np.abs(b).max()), (name, lo)


def test_captured_and_replayed(hip):
    """One capture replayed with other offsets and operands in the same memory, a second capture of the plan between, against plain
    runs of each."""
    from lumen_amd.compiler.plan import Plan
    from lumen_amd.tensor import DeviceBuffer

    rng = np.random.default_rng(11)
    t, n, nkv, d = 260, 4, 2, 64
    dts = ["bfloat16"] * 3 + ["int32", "bfloat16"]
    sets = []
    for lengths in ([260, 0, 0], [100, 100, 50], [1, 0, 200], [64, 64, 128]):
        x = M.packed_inputs(rng, t, n, nkv, d)
        sets.append([D.from_values(x[k].astype(np.float32), "bfloat16") for k in "qkv"] +
                    [M.offsets_of(lengths).astype(np.int32), D.from_values(x["do"].astype(np.float32), "bfloat16")])
    plan = Plan(L.make_graph(_program(True))(*[L.empty(list(a.shape), dt, "meta") for a, dt in zip(sets[0], dts)]), "hip:0")
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


def test_refusals_of_the_entry_points(hip):
    one = Dev(nbytes=4096)

    def desc(**kw):
        d = nv.PackedDesc(tokens=2, sequences=1, heads=1, kv_heads=1, head_dim=8, dtype=1, offsets_dtype=1, scale=1.0)
        for name, v in kw.items():
            setattr(d, name, v)
        return C.byref(d)

    with pytest.raises(RuntimeError, match="16 bytes"):
        nv.call("nhip_packed_fwd", desc(), one.ptr + 2, one.ptr, one.ptr, one.ptr, one.ptr, None, None, one.ptr)
    with pytest.raises(RuntimeError, match="workspace"):
        nv.call("nhip_packed_fwd", desc(), one.ptr, one.ptr, one.ptr, one.ptr, one.ptr, None, None, None)
    with pytest.raises(RuntimeError, match="workspace"):
        nv.call("nhip_packed_bwd", desc(), *[one.ptr] * 11, None)
    with pytest.raises(RuntimeError, match="head dim"):
        nv.call("nhip_packed_fwd", desc(head_dim=12), one.ptr, one.ptr, one.ptr, one.ptr, one.ptr, None, None, one.ptr)
    for at in range(5):
        with pytest.raises(RuntimeError, match="without memory"):
            nv.call("nhip_packed_fwd", desc(), *[None if i == at else one.ptr for i in range(5)], None, None, one.ptr)
    for at in (0, 1, 2, 3, 4, 6, 7, 8, 9, 10):  # all but the rest of o
        with pytest.raises(RuntimeError, match="without memory"):
            nv.call("nhip_packed_bwd", desc(), *[None if i == at else one.ptr for i in range(11)], one.ptr)
    nv.call("nhip_packed_fwd", desc(tokens=0), None, None, None, None, None, None, None, None)  # nothing to do


@pytest.mark.parametrize("sequences", [2, 300])
def test_key_heads_without_a_query_head(hip, sequences):
    """Nothing adds to their gradients, which are zeros and not what the memory held: of tables by either builder, a sequence's tokens
    and those of none."""
    t, nkv, d = 400, 2, 64
    offsets = np.concatenate([[3], np.sort(np.random.default_rng(3).integers(3, 390, sequences))]).astype(np.int32)
    desc = nv.PackedDesc(tokens=t, sequences=sequences, heads=0, kv_heads=nkv, head_dim=d, dtype=1, causal=1, offsets_dtype=1, scale=1.0,
                         ds_bytes=1 << 20, k_s=nkv * d, k_n=d, v_s=nkv * d, v_n=d, dk_s=nkv * d, dk_n=d, dv_s=nkv * d, dv_n=d)
    size = C.c_size_t()
    nv.call("nhip_packed_workspace", C.byref(desc), 1, C.byref(size))
    ones = Dev(np.full(t * nkv * d, 0x3f80, np.uint16))
    dk, dv, at, ws = Dev(np.full(t * nkv * d, 0x3f80, np.uint16)), Dev(np.full(t * nkv * d, 0x3f80, np.uint16)), Dev(offsets), Dev(nbytes=size.value)
    nv.call("nhip_packed_bwd", C.byref(desc), None, ones.ptr, ones.ptr, at.ptr, None, None, None, None, None, dk.ptr, dv.ptr, ws.ptr)
    for x in (dk, dv):
        assert not x.get(t * nkv * d, np.uint16).any()
    q, kv = np.zeros((t, 0, d)), np.ones((t, nkv, d))
    out = L.compile(_program(True), device="hip")(_tensor(q, "bfloat16"), _tensor(kv, "bfloat16"), _tensor(kv, "bfloat16"), L.from_numpy(offsets),
                                                  _tensor(q, "bfloat16"))
    assert [_values(a).shape for a in out] == [q.shape, q.shape, kv.shape, kv.shape] and not any(_values(a).any() for a in out)


@pytest.mark.parametrize("shape,view,t,n", [
    ([40, 2, 68], lambda x: x[:, 0:1, :64], 40, 1), ([1, 1, 100], lambda x: x[:, :, :64], 1, 1), ([1, 4, 72], lambda x: x[:, :3, :64], 1, 3),
    ([100 * 64], lambda x: x.reshape(100, 64, 1).permute(0, 2, 1) if isinstance(x, L.graph.tracer.TracedTensor) else x.reshape(100, 1, 64), 100, 1)])
def test_axes_of_one_element_have_any_stride(hip, shape, view, t, n):
    """One head and one token of views whose stride there is no multiple of 8 elements, read where they lie."""
    rng = np.random.default_rng(t + n)
    base = {name: _round(rng.standard_normal(shape), "bfloat16") for name in ("q", "k", "v", "do")}

    def both(q, k, v, offsets, do):
        return _program(True)(view(q), view(k), view(v), offsets, view(do))

    offsets = np.array([0, t // 3, t])
    want, tol = M.packed({name: view(x) for name, x in base.items()}, offsets, True, 0.125, "bfloat16")
    f = L.compile(both, device="hip")
    got = f(*(_tensor(base[name], "bfloat16") for name in "qkv"), L.from_numpy(offsets.astype(np.int32)), _tensor(base["do"], "bfloat16"))
    for name, a, w, tt in zip(("o", "dq", "dk", "dv"), got, want, tol):
        assert w.shape == (t, n, 64)
        _near(_values(a), w, tt, name)
    assert [st.kind for st in f.plan.steps if st.kind != "view"] == ["packed_fwd", "packed_bwd"]


@pytest.mark.parametrize("tokens,n,nkv", [(0, 2, 1), (5, 0, 2), (0, 0, 1)])
def test_primitives_without_tokens_or_query_heads(hip, tokens, n, nkv):
    """float32: gradients of zeros, and results of no elements."""
    q, kv = np.zeros((tokens, n, 8), np.float32), np.ones((tokens, nkv, 8), np.float32)
    args = [L.from_numpy(a) for a in (q, kv, kv, np.array([0, tokens // 2, tokens], np.int32), q)]
    out = [_values(a) for a in L.compile(_program(True), device="hip")(*args)]
    assert [a.shape for a in out] == [q.shape, q.shape, kv.shape, kv.shape] and not any(a.any() for a in out)


def test_sums_over_nothing(hip):
    """Of every axis, the first, the last, and both around one that is kept."""
    f = L.compile(lambda x, y, z: [F.sum(x, 0), F.sum(y, 1), F.sum(z, (0, 2)), F.sum(x)], device="hip")
    got = [_values(a) for a in f(*(L.from_numpy(np.zeros(s, np.float32)) for s in ((0, 300), (7, 0), (3, 5, 0))))]
    assert [a.shape for a in got] == [(300,), (7,), (5,), ()] and not any(a.any() for a in got)
