"""The transformer's training step on packed documents on the GPU: packed attention, the head's cross entropy with its gradients,
the clip and AdamW together, as ``workloads.packed_train_step`` runs them."""

import numpy as np
import pytest

import lumen_amd as L
import lumen_amd.functional as F
from lumen_amd import dtypes as D
from lumen_amd import workloads as W
from lumen_amd.graph import prims
from oracle import oracle
from tests import training_math as M
from tests.test_packed_step import documents, values

pytestmark = pytest.mark.gpu

TOKENS = 256


def _model(lr=2e-3):
    model, _ = W.build(W.TINY)
    weights = W.init_weights(model)
    W.load(model, weights)
    opt = W.adamw(model, lr)
    W.load_adamw(opt)
    return model, opt, weights


def _batches(rng, count):
    lengths = ([128, 64, 1, 0, 60], [70, 128, 3, 55, 0], [1, 1, 2, 0, 100], [128, 128, 0, 0, 0], [33, 65, 97, 31, 30])
    return [W.pack(documents(rng, lengths[i % 5], W.TINY.vocab), TOKENS) for i in range(count)]


def _state(opt):
    return [np.array(x._placed("hip:0").raw()) for xs in (opt.params, opt.masters, opt.exp_avgs, opt.exp_avg_sqs) for x in xs]


def _float64(weights, arrays):
    """The loss and the gradients by name, each document alone, in float64 primitives run by the oracle."""
    cfg, names = W.TINY, list(weights)
    w64 = [D.bf16_to_f32(weights[n]).astype(np.float64) for n in names]

    def matmul(x, y):
        return F.matmul(x, y, "float64", "float64")

    def norm(x, weight):
        return F.rms_norm(x, cfg.dim, weight, 2.0**-23)  # the float32 one's epsilon

    def losses(ids, places, targets, *ws):
        """The sum of a document's losses, the last token's left out."""
        w = dict(zip(names, ws))
        n = ids.shape[0]
        x = w["embed.tokens"][ids] + w["embed.positions"][places]
        ahead = prims.lt(prims.iota("int64", (n, n), 0), prims.iota("int64", (n, n), 1))
        for i in range(cfg.layers):
            at = {k.split(".", 2)[2]: t for k, t in w.items() if k.startswith(f"layers.{i}.")}
            y, heads = norm(x, at["attn.norm"]), []
            for h in range(cfg.heads):
                lo, hi = h * cfg.head_dim, (h + 1) * cfg.head_dim
                q, k, v = (matmul(y, at[f"attn.{m}"][lo:hi].t()) for m in ("wq", "wk", "wv"))
                s = matmul(q, k.t()) * cfg.head_dim**-0.5
                heads.append(matmul(F.softmax(F.where(ahead, prims.full(s.shape, -np.inf, "float64"), s), -1), v))
            x = x + matmul(F.cat(heads, 1), at["attn.wo"].t())
            x = x + matmul(F.gelu(matmul(norm(x, at["mlp.norm"]), at["mlp.w1"].t())), at["mlp.w2"].t())
        logits = matmul(norm(x, w["norm"]), w["head"].t())
        return F.sum(F.cross_entropy(logits[:n - 1], targets[:n - 1]))

    def step(ids, places, targets, *ws):
        loss, pull = L.vjp(lambda *ws: losses(ids, places, targets, *ws), *ws)
        return [loss, *pull(prims.full((), 1.0, "float64"))]

    ids, places, targets, offsets = arrays
    out, counted = 0.0, int((targets != -100).sum())
    for lo, hi in zip(offsets, offsets[1:]):
        if hi > lo + 1:
            ins = [ids[lo:hi], places[lo:hi], targets[lo:hi], *w64]
            metas = [L.empty(list(a.shape), str(a.dtype), "meta") for a in ins]
            out = out + np.array([np.asarray(v, np.float64) for v in oracle.values(L.make_graph(step)(*metas), ins)], object)
    return float(out[0]) / counted, {n: g / counted for n, g in zip(names, out[1:])}


def test_gradients_match_float64_and_the_oracle(hip):
    """Against float64, the loss and every gradient are off by what the oracle's run of the same graph is off by: it rounds the
    same values to bfloat16, some of them the other way, so that both errors are alike in the mean square; 1.5 times allows for the
    gradients of few elements (a norm's 128). Element by element both lie within the bound of the unpacked step's test
    (test_gpu_transformer.py) of the float64 gradient, so within twice it of one another."""
    model, _, weights = _model()
    names = {id(p): n for n, p in model.named_parameters()}

    def grads(model, ids, places, targets, offsets):
        loss = W.packed_loss(model, ids, places, targets, offsets)
        loss.backward()
        return [loss, *(p.grad for p in model.parameters())]

    f = L.compile(grads, device="hip")
    for arrays in _batches(np.random.default_rng(1), 3):
        args = (model, *map(L.from_numpy, arrays))
        got = [np.asarray(L.to_numpy(t), np.float64) for t in f(*args)]
        rounded = values(grads, args, arrays, weights, names)
        loss, want = _float64(weights, arrays)
        assert abs(got[0] - loss) <= 1e-3 * loss
        for name, a, b in zip(names.values(), got[1:], rounded[1:]):
            w = want[name]
            assert np.linalg.norm(a - w) <= 1.5 * np.linalg.norm(b - w), name
            assert np.all(np.abs(a - b) <= 2 * (2e-2 * np.abs(w) + 1e-2 * np.abs(w).max())), name


def _steps(count, **patches):
    """The losses and the state after each of `count` steps on different documents."""
    model, opt, _ = _model()
    with L.config.compiler.patch(**patches):
        step = L.compile(W.packed_train_step, device="hip")
        out = []
        for arrays in _batches(np.random.default_rng(2), count):
            loss = float(L.to_numpy(step(model, opt, *map(L.from_numpy, arrays))))
            out.append((loss, _state(opt)))
    kinds = [s.kind for s in step.plan.steps]
    assert [kinds.count(k) for k in ("packed_fwd", "packed_bwd", "head_loss", "adamw", "clip")] == [2, 2, 1, 1, 1]
    assert len(step.plan.in_place_outputs) >= 4 * len(opt.params)
    return out, step


def test_replayed_steps_are_the_bits_of_plain_ones(hip):
    """Six steps on other documents each, the whole step replayed from a captured graph from the third on, against the same steps
    launched one by one."""
    plain, _ = _steps(6, hip_graphs=False)
    replayed, step = _steps(6, hip_graphs=True)
    assert step._graphs[id(step.plan)]
    for t, ((a, x), (b, y)) in enumerate(zip(plain, replayed)):
        assert a == b and np.isfinite(a), t
        assert all(np.array_equal(i, j) for i, j in zip(x, y)), t
    assert not np.array_equal(plain[0][1][0], plain[5][1][0])


def test_the_clip_within_adamw_is_the_clip_ahead_of_it(hip):
    """A step whose clipped gradients nothing else reads (AdamW takes them times the clip's factor, rounded as the clip would)
    leaves the bits that it leaves where they are results too, which the clip then writes."""
    def written(model, opt, ids, places, targets, offsets):
        loss = W.packed_loss(model, ids, places, targets, offsets)
        loss.backward()
        kept, norm = F.clip_grad_norm([p.grad for p in opt.params], 1.0)
        opt.step(max_norm=1.0)
        return [loss, norm, *kept]

    within, _ = _steps(3)
    model, opt, _ = _model()
    step = L.compile(written, device="hip")
    for (loss, state), arrays in zip(within, _batches(np.random.default_rng(2), 3)):
        out = step(model, opt, *map(L.from_numpy, arrays))
        assert float(L.to_numpy(out[0])) == loss and float(L.to_numpy(out[1])) > 1.0
        assert all(np.array_equal(a, b) for a, b in zip(state, _state(opt)))


def test_a_view_off_16_bytes_that_an_adamw_step_reads_too(hip):
    """Its 8 bytes suit the AdamW step and not the attention or the head's loss, which have a copy of it."""
    rng = np.random.default_rng(6)
    t = 40
    base = np.array(D.bf16_bits(rng.standard_normal(4 + t * 64).astype(np.float32)))
    x = D.bf16_to_f32(base)[4:].astype(np.float64)
    w = np.array(D.bf16_bits(rng.standard_normal((100, 64)).astype(np.float32) / 8))
    target, offsets = rng.integers(0, 100, t), np.array([0, 13, t])
    state = [np.zeros((t, 1, 64), np.float32), np.zeros((t, 1, 64), np.float32)]

    def fn(base, m, v, offsets, target, w):
        x = base[4:4 + t * 64].reshape(t, 1, 64)
        rows = x.reshape(t, 64)
        stepped = F.adamw([x, rows], [x, rows], [m, m.reshape(t, 64)], [v, v.reshape(t, 64)], 1, 0.1, weight_decay=0.0)[0]
        return [F.packed_attention(x, x, x, offsets), F.linear_cross_entropy(rows, w, target, reduction="none"), *stepped]

    args = [L.Tensor("bfloat16", base.shape, "cpu", host=base), *(L.from_numpy(a) for a in state), L.from_numpy(offsets), L.from_numpy(target),
            L.Tensor("bfloat16", w.shape, "cpu", host=w)]
    o, losses, *stepped = (np.asarray(L.to_numpy(a), np.float64) for a in L.compile(fn, device="hip")(*args))
    heads = {name: x.reshape(t, 1, 64) for name in ("q", "k", "v", "do")}
    want, tol = M.packed(heads, offsets, True, 0.125, "bfloat16")
    assert np.all(np.abs(o - want[0]) <= tol[0])
    row = (x.reshape(t, 64), D.bf16_to_f32(w).astype(np.float64), target, -100, np.ones(t))
    assert np.all(np.abs(losses - M.linear_cross_entropy(*row)[0]) <= M.linear_cross_entropy_tolerances(*row, "bfloat16")[0])
    zero = np.zeros(x.shape)
    new, tw = M.adamw(x, x, zero, zero, 1, 0.1, (0.9, 0.999), 1e-8, 0.0)[0], M.adamw_tolerances(x, x, zero, zero, 1, 0.1, (0.9, 0.999), 1e-8, 0.0)[0]
    for a in stepped:
        assert np.all(np.abs(a.reshape(-1) - new) <= tw + 2.0**-8 * (np.abs(new) + tw))


def test_weights_of_two_launches_in_place_and_clipped(hip):
    """More weights than a launch of AdamW's table holds (44), written over their own memory with the clip's factor taken within the step,
    leave the bits of the same step into other memory."""
    cfg = W.TransformerConfig(vocab=97, dim=64, heads=2, ffn=96, seq=24, batch=1, layers=6)
    rng = np.random.default_rng(9)
    batches = [W.pack([rng.integers(0, cfg.vocab, n) for n in lengths], 64) for lengths in ([24, 1, 20], [7, 0, 24, 24], [3, 3])]
    states = []
    for in_place in (True, False):
        model, _ = W.build(cfg)
        W.load(model, W.init_weights(model))
        opt = W.adamw(model, 1e-2)
        W.load_adamw(opt)
        assert len(opt.params) > 44
        with L.config.compiler.patch(update_in_place=in_place):
            step = L.compile(W.packed_train_step, device="hip")
            losses = [float(L.to_numpy(step(model, opt, *map(L.from_numpy, b)))) for b in batches]
        assert [st.kind for st in step.plan.steps].count("adamw") == 1
        assert (len(step.plan.in_place_outputs) >= 4 * len(opt.params)) == in_place
        states.append((losses, _state(opt)))
    (a, x), (b, y) = states
    assert a == b and np.isfinite(a).all()
    assert all(np.array_equal(i, j) for i, j in zip(x, y))
