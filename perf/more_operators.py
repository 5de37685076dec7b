"""Three operators that a training step on packed documents calls, as cases that can be timed and checked:

* ``F.packed_attention``: self attention of tokens whose sequences lie one after another, each within its own;
* ``F.linear_cross_entropy``: the loss of a vocabulary head over the tokens that have a target, without its logits;
* ``F.adamw``: an AdamW step over every weight of a model.

The first two in both directions. With ``own`` false ``run`` computes them from elementary torch operations in float32;
with ``own`` true it calls the compiled functions that a program of this framework makes of them.
"""

import functools
import math
import random

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16, "int32": torch.int32}
NAMES = {v: k for k, v in DTYPES.items()}
IGNORED = -100  # the target of a token without one
BETAS, ADAM_EPS, DECAY = (0.9, 0.95), 1e-8, 0.1


def listed():
    return [
        # three short prompts read together: the smallest call, latency counts
        dict(name="packed_short", kind="packed", train=False, lengths="61,17,19", tokens=97, n=16, nkv=4, d=64, causal=True,
             dtype="bfloat16"),
        # prompts of any length read together, grouped key heads, tokens behind the last prompt unused
        dict(name="packed_prefill", kind="packed", train=False,
             lengths="2048,1777,1213,900,701,512,333,256,129,64,33,1", tokens=8192, n=16, nkv=4, d=128, causal=True,
             dtype="bfloat16"),
        # a batch of documents packed into the 12-layer model's tokens, in training
        dict(name="packed_train", kind="packed", train=True, lengths="4096,3811,2600,2222,1777,1033,500,281", tokens=16384,
             n=16, nkv=16, d=128, causal=True, dtype="bfloat16"),
        # the 2-layer model's heads over many short documents, in training
        dict(name="packed_train_short", kind="packed", train=True,
             lengths="512,500,451,400,390,333,300,277,256,250,200,190,160,128,127,126,90,77,64,63,33,31,16,15,8,7,1,1",
             tokens=5120, n=8, nkv=8, d=64, causal=True, dtype="bfloat16"),
        # an encoder's pieces of odd lengths, some empty, a head dim that is no power of two, float16
        dict(name="packed_train_odd", kind="packed", train=True, lengths="331,0,1,254,97,0,129", tokens=901, n=6, nkv=2, d=80,
             causal=False, dtype="float16"),
        # evaluation of a few sentences by the 2-layer model's head: a loss a token
        dict(name="loss_eval", kind="loss", train=False, tokens=512, dim=512, vocab=32000, ignored=0.1, scale=1.0,
             dtype="bfloat16"),
        # a ragged batch of odd sizes with a scaled loss, float16, a third of the tokens a prompt's
        dict(name="loss_train_odd", kind="loss", train=True, tokens=777, dim=520, vocab=5003, ignored=0.33, scale=2048.0,
             dtype="float16"),
        # the 2-layer model's batch in training
        dict(name="loss_train", kind="loss", train=True, tokens=8192, dim=512, vocab=32000, ignored=0.05, scale=1.0,
             dtype="bfloat16"),
        # the 12-layer model's batch in training: the largest
        dict(name="loss_train_large", kind="loss", train=True, tokens=16384, dim=2048, vocab=32000, ignored=0.05, scale=1.0,
             dtype="bfloat16"),
        # a few float32 weights of odd sizes: launches count
        dict(name="adamw_small", kind="adamw", dim=130, ffn=333, vocab=517, seq=33, layers=1, masters=False, dtype="float32"),
        # one layer, embeddings and head at the 2-layer model's sizes, bfloat16 weights with float32 masters
        dict(name="adamw_step", kind="adamw", dim=512, ffn=2048, vocab=32000, seq=512, layers=1, masters=True,
             dtype="bfloat16"),
        # the same at the 12-layer model's sizes: 190 million weights
        dict(name="adamw_large", kind="adamw", dim=2048, ffn=8192, vocab=32000, seq=4096, layers=1, masters=True,
             dtype="bfloat16"),
    ]


# ---- drawn cases


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size of the range: mostly a multiple of 64, now and then of 8, now and then any."""
    n, q = _log(rng, lo, hi), rng.choice([64, 64, 64, 8, 8, 1])
    return max(q, n // q * q)


def _draw_packed(rng, train):
    tokens = _log(rng, 48, 16384)
    count = min(_log(rng, 1, 64), tokens)
    spread = [rng.uniform(0.05, 1.0) ** rng.choice([1, 2]) for _ in range(count)]
    used = tokens if rng.random() < 0.5 else int(tokens * rng.uniform(0.7, 1.0))
    lengths = [int(used * s / sum(spread)) for s in spread]
    for i in range(count):
        if lengths[i] > 1 and rng.random() < 0.08:
            lengths[i] = rng.choice([0, 1])
    n = rng.choice([2, 4, 6, 8, 16])
    return dict(kind="packed", train=train, lengths=",".join(map(str, lengths)), tokens=tokens, n=n,
                nkv=n // rng.choice([1, 1, 2]), d=rng.choice([64, 64, 128, 128, 32, 80, 96]), causal=rng.random() < 0.8,
                dtype=rng.choice(["bfloat16", "bfloat16", "float16"]))


def _draw(rng):
    kind = rng.choice(["packed", "packed_train", "packed_train", "loss", "loss_train", "loss_train", "adamw"])
    if kind.startswith("packed"):
        return _draw_packed(rng, kind == "packed_train")
    if kind.startswith("loss"):
        half = rng.random() < 0.3
        return dict(kind="loss", train=kind == "loss_train", tokens=_log(rng, 16, 16384), dim=_size(rng, 128, 4096),
                    vocab=_size(rng, 256, 65536), ignored=round(rng.choice([0.0, rng.uniform(0.0, 0.6)]), 2),
                    scale=2048.0 if half else 1.0, dtype="float16" if half else "bfloat16")
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    return dict(kind="adamw", dim=_size(rng, 32, 2048), ffn=_size(rng, 64, 8192), vocab=_log(rng, 100, 32000),
                seq=_log(rng, 16, 4096), layers=1, masters=dtype != "float32" and rng.random() < 0.7, dtype=dtype)


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 300)


def _room(case):
    """The scores or logits that the plain form holds at once."""
    if case["kind"] == "packed":
        lengths = _lengths(case)
        return len(lengths) * max(lengths) ** 2 * case["n"]
    return case["tokens"] * case["vocab"] if case["kind"] == "loss" else 0


def draw(rng):
    """A case of the same kinds and ranges that costs no more, and holds no more, than the largest listed one."""
    most, room = max(_cost(c) for c in listed()), max(_room(c) for c in listed())
    while True:
        c = _draw(rng)
        if _cost(c) <= most and _room(c) <= room and (c["kind"] != "packed" or max(_lengths(c)) > 0):
            return c


# ---- inputs


def _normal(g, shape, dtype, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=g, device="cuda") * std + mean).to(DTYPES[dtype])


def _lengths(case):
    return [int(x) for x in case["lengths"].split(",")]


def _weight_shapes(case):
    """The weights of a decoder, in the order that its modules list them."""
    d, f = case["dim"], case["ffn"]
    layer = [(d,), (d, d), (d, d), (d, d), (d, d), (d,), (f, d), (d, f)]
    return [(case["vocab"], d), (case["seq"], d)] + layer * case["layers"] + [(d,), (case["vocab"], d)]


def _inputs(case, seed):
    """The case's inputs by name, torch tensors on the GPU, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind, dt = case["kind"], case["dtype"]
    if kind == "packed":
        t, n, nkv, d = case["tokens"], case["n"], case["nkv"], case["d"]
        lengths = _lengths(case)
        random.Random(seed).shuffle(lengths)  # the documents in another order
        offsets = [0]
        for length in lengths:
            offsets.append(offsets[-1] + length)
        x = {"q": _normal(g, (t, n, d), dt), "k": _normal(g, (t, nkv, d), dt), "v": _normal(g, (t, nkv, d), dt),
             "offsets": torch.tensor(offsets, dtype=torch.int32, device="cuda")}
        if case["train"]:
            x["do"] = _normal(g, (t, n, d), dt)
        return x
    if kind == "loss":
        t, d, v = case["tokens"], case["dim"], case["vocab"]
        # a head some way into training: rows of unit scale, logits of a few units
        x = {"h": _normal(g, (t, d), dt), "w": _normal(g, (v, d), dt, std=1.5 * d**-0.5)}
        target = torch.randint(0, v, (t,), generator=g, device="cuda")
        unused = torch.rand((t,), generator=g, device="cuda") < case["ignored"]
        x["target"] = torch.where(unused, IGNORED, target).to(torch.int32)
        return x
    x = {}
    for i, shape in enumerate(_weight_shapes(case)):
        master = torch.randn(shape, generator=g, device="cuda") * 0.02
        x[f"p{i}"] = master.to(DTYPES[dt])
        x[f"g{i}"] = _normal(g, shape, dt, std=0.01)
        x[f"m{i}"] = torch.randn(shape, generator=g, device="cuda") * 0.003
        x[f"v{i}"] = (torch.randn(shape, generator=g, device="cuda") * 0.01).square() + 1e-7
        if case["masters"]:
            x[f"w{i}"] = master
    x["step"] = torch.randint(1, 1000, (), generator=g, device="cuda").to(torch.int32)
    return x


def _rate(seed):
    """A learning rate of a schedule."""
    return 1e-3 * random.Random(seed).uniform(0.1, 1.0)


def prepare(case, seed):
    state = {"case": dict(case), "x": _inputs(case, seed), "rate": _rate(seed)}
    if own:
        _own_state(state)
    return state


# ---- the plain forms


def _padded(case, x):
    """Each sequence's tokens in a row of the longest one's length: their indices, and which of them there are."""
    start, end = x["offsets"][:-1, None].long(), x["offsets"][1:, None].long()
    at = start + torch.arange(max(_lengths(case)), device="cuda")
    there = at < end
    return torch.where(there, at, 0), there


def _rows(t, at, there):
    """``t``'s rows of each sequence, float32 ``[sequences, heads, longest, d]``, zeros past its end."""
    return (t[at].float() * there[:, :, None, None]).permute(0, 2, 1, 3)


def _back(t, at, there, like):
    """Padded rows as packed ones, zeros for the tokens of no sequence."""
    out = torch.zeros(like.shape, device="cuda")
    out[at[there]] = t.permute(0, 2, 1, 3)[there]
    return out.to(like.dtype)


def _packed_plain(case, x):
    at, there = _padded(case, x)
    group, scale = case["n"] // case["nkv"], case["d"] ** -0.5
    q, k, v = (_rows(x[name], at, there) for name in "qkv")
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    pos = torch.arange(at.shape[1], device="cuda")
    seen = there[:, None, None, :]
    if case["causal"]:
        seen = seen & (pos[None, :] <= pos[:, None])
    s = (q @ k.transpose(2, 3) * scale).masked_fill(~seen, -math.inf)
    top = s.amax(3, keepdim=True)
    p = torch.exp(s - torch.where(torch.isfinite(top), top, 0.0))
    total = p.sum(3, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    del s
    o = p @ v
    out = [_back(o, at, there, x["q"])]
    if not case["train"]:
        return out
    do = _rows(x["do"], at, there)
    dv = p.transpose(2, 3) @ do
    ds = p * (do @ v.transpose(2, 3) - (do * o).sum(3, keepdim=True)) * scale
    dq, dk = ds @ k, ds.transpose(2, 3) @ q
    b, n, length, d = dk.shape
    dk, dv = (t.reshape(b, case["nkv"], group, length, d).sum(2) for t in (dk, dv))
    return out + [_back(dq, at, there, x["q"]), _back(dk, at, there, x["k"]), _back(dv, at, there, x["v"])]


def _loss_plain(case, x):
    h, w, target = x["h"].float(), x["w"].float(), x["target"].long()
    valid = target != IGNORED
    count = valid.sum().clamp(min=1)
    cls = torch.where(valid, target, 0)
    logits = h @ w.t()
    top = logits.amax(1, keepdim=True)
    e = torch.exp(logits - top)
    total = e.sum(1, keepdim=True)
    lse = (top + torch.log(total))[:, 0]
    picked = logits.gather(1, cls[:, None])[:, 0]
    losses = torch.where(valid, lse - picked, 0.0)
    if not case["train"]:
        return [losses]
    d = e / total
    d[torch.arange(len(cls), device="cuda"), cls] -= 1
    d = d * torch.where(valid, case["scale"] / count, 0.0)[:, None]
    return [losses.sum() / count, (d @ w).to(x["h"].dtype), (d.t() @ h).to(x["w"].dtype)]


def _adamw_plain(case, x, rate):
    b1, b2 = BETAS
    t = x["step"].double()
    c1, c2 = (1 - b1**t).float(), (1 - b2**t).float()
    params, masters, ms, vs = [], [], [], []
    for i in range(len(_weight_shapes(case))):
        g = x[f"g{i}"].float()
        w = x[f"w{i}"] if case["masters"] else x[f"p{i}"].float()
        m = b1 * x[f"m{i}"] + (1 - b1) * g
        v = b2 * x[f"v{i}"] + (1 - b2) * g * g
        w = w * (1 - rate * DECAY) - rate * (m / c1) / (torch.sqrt(v / c2) + ADAM_EPS)
        params.append(w.to(x[f"p{i}"].dtype))
        masters += [w] if case["masters"] else []
        ms.append(m)
        vs.append(v)
    return params + masters + ms + vs


def run(state):
    if own:
        return _own_run(state)
    case = state["case"]
    if case["kind"] == "packed":
        return _packed_plain(case, state["x"])
    if case["kind"] == "loss":
        return _loss_plain(case, state["x"])
    return _adamw_plain(case, state["x"], state["rate"])


# ---- the framework's programs


def _packed_program(q, k, v, offsets, causal):
    import lumen_amd.functional as F

    return [F.packed_attention(q, k, v, offsets, is_causal=causal)]


def _packed_train_program(q, k, v, offsets, causal, do):
    import lumen_amd as L
    import lumen_amd.functional as F

    o, pullback = L.vjp(lambda q, k, v: F.packed_attention(q, k, v, offsets, is_causal=causal), q, k, v)
    return [o, *pullback(do)]


def _loss_program(h, w, target):
    import lumen_amd.functional as F

    return [F.linear_cross_entropy(h, w, target, ignore_index=IGNORED, reduction="none")]


def _loss_train_program(h, w, target, scale):
    import lumen_amd as L
    import lumen_amd.functional as F

    loss, pullback = L.vjp(lambda h, w: F.linear_cross_entropy(h, w, target, ignore_index=IGNORED), h, w)
    return [loss, *pullback(scale.to("float32"))]


def _adamw_program(rate, step, masters, *tensors):
    import lumen_amd.functional as F

    n = len(tensors) // (5 if masters else 4)
    p, g, m, v, w = (list(tensors[i * n:(i + 1) * n]) for i in range(5))
    p, m, v, w = F.adamw(p, g, m, v, step, rate, betas=BETAS, eps=ADAM_EPS, weight_decay=DECAY, masters=w if masters else None)
    return [*p, *(w or []), *m, *v]


@functools.lru_cache(maxsize=None)
def _program(fn):
    """A program's compiled function, kept as a program keeps it: one plan for each shape it is called with."""
    import lumen_amd as L

    return L.compile(fn, device="hip")


def _device(t):
    """A tensor of the framework's on the device with ``t``'s values."""
    import lumen_amd as L
    from lumen_amd import native

    out = L.empty(tuple(t.shape), NAMES[t.dtype], "hip")
    native.d2d(out.data_ptr(), t.data_ptr(), out.nbytes)
    return out


def _own_state(state):
    """The compiled function and its arguments on the framework's device, in place of torch's tensors."""
    from lumen_amd import native

    torch.cuda.synchronize()
    native.set_device(0)
    case = state["case"]
    x = {name: _device(t) for name, t in state.pop("x").items()}
    native.sync()
    if case["kind"] == "packed":
        fn, args = _packed_program, [x["q"], x["k"], x["v"], x["offsets"], case["causal"]]
        if case["train"]:
            fn, args = _packed_train_program, [*args, x["do"]]
    elif case["kind"] == "loss":
        fn, args = _loss_program, [x["h"], x["w"], x["target"]]
        if case["train"]:
            fn, args = _loss_train_program, [*args, case["scale"]]
    else:
        count = len(_weight_shapes(case))
        names = "pgmvw" if case["masters"] else "pgmv"
        fn = _adamw_program
        args = [state["rate"], x["step"], case["masters"], *(x[f"{name}{i}"] for name in names for i in range(count))]
    state.update(program=_program(fn), args=args, views={})


class _Memory:
    """A device tensor's memory for torch, which keeps this object (and so the memory) as long as its view."""

    def __init__(self, t):
        self.tensor = t
        self.__cuda_array_interface__ = {"shape": tuple(t.shape), "data": (t.data_ptr(), False), "version": 2,
                                         "typestr": {"float32": "<f4", "bfloat16": "<i2", "float16": "<f2"}[t.dtype]}


def _view(views, t):
    """``t`` as a torch tensor over the same memory (made once for each place an output is written)."""
    key = (t.data_ptr(), t.dtype, t.shape)
    v = views.get(key)
    if v is None:
        v = views[key] = torch.as_tensor(_Memory(t), device="cuda").view(DTYPES[t.dtype])
    return v


def _own_run(state):
    return [_view(state["views"], t) for t in state["program"](*state["args"])]


# ---- what a pass cannot do without


def work(case):
    kind, size = case["kind"], 4 if case["dtype"] == "float32" else 2
    if kind == "packed":
        lengths = _lengths(case)
        used, d = sum(lengths), case["d"]
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lengths)
        q, kv = used * case["n"] * d * size, used * case["nkv"] * d * size
        rest = 4 * (len(lengths) + 1) + case["tokens"] * case["n"] * d * size - q  # the zeros of unused tokens
        if not case["train"]:
            return {"bytes": 2 * q + 2 * kv + rest, "flops": 4 * case["n"] * d * pairs}
        rest += case["tokens"] * (case["n"] + 2 * case["nkv"]) * d * size - q - 2 * kv
        return {"bytes": 4 * q + 4 * kv + rest, "flops": 14 * case["n"] * d * pairs}
    if kind == "loss":
        t, d, v = case["tokens"], case["dim"], case["vocab"]
        operands = size * (t * d + v * d)
        if not case["train"]:
            return {"bytes": operands + 8 * t, "flops": 2 * t * d * v}
        return {"bytes": 2 * operands + 4 * t, "flops": 6 * t * d * v}
    count = sum(math.prod(s) for s in _weight_shapes(case))
    return {"bytes": count * (3 * size + 16 + (8 if case["masters"] else 0)), "flops": 0}


# ---- the same in 64 bits


def _packed64(case, x):
    """One sequence after another, the gradients by torch's differentiation."""
    leaves = [x[n].double().requires_grad_(case["train"]) for n in "qkv"]
    q, k, v = leaves
    group = case["n"] // case["nkv"]
    rows, at = [], [int(t) for t in x["offsets"]]
    for lo, hi in zip(at, at[1:]):
        s = torch.matmul(q[lo:hi].transpose(0, 1), k[lo:hi].permute(1, 2, 0).repeat_interleave(group, 0)) / math.sqrt(case["d"])
        if case["causal"]:
            s = s + torch.full((hi - lo, hi - lo), -math.inf, dtype=torch.float64, device="cuda").triu(1)
        rows.append(torch.matmul(torch.softmax(s, 2), v[lo:hi].transpose(0, 1).repeat_interleave(group, 0)).transpose(0, 1))
    rows.append(torch.zeros((case["tokens"] - at[-1], case["n"], case["d"]), dtype=torch.float64, device="cuda"))
    o = torch.cat(rows)
    if not case["train"]:
        return [o]
    return [o.detach(), *torch.autograd.grad(o, leaves, x["do"].double())]


def _loss64(case, x):
    h, w = (x[n].double().requires_grad_(case["train"]) for n in "hw")
    kept = torch.nonzero(x["target"] != IGNORED)[:, 0]
    logits = h[kept] @ w.t()
    losses = torch.logsumexp(logits, 1) - logits[torch.arange(len(kept), device="cuda"), x["target"][kept].long()]
    if not case["train"]:
        return [torch.zeros(case["tokens"], dtype=torch.float64, device="cuda").index_put((kept,), losses)]
    loss = losses.sum() / max(len(kept), 1)
    return [loss.detach(), *torch.autograd.grad(loss * case["scale"], [h, w])]


def _adamw64(case, x, rate):
    (b1, b2), t = BETAS, int(x["step"])
    new = {"p": [], "w": [], "m": [], "v": []}
    for i in range(len(_weight_shapes(case))):
        g, m, v = (x[f"{n}{i}"].double() for n in "gmv")
        w = x[f"w{i}" if case["masters"] else f"p{i}"].double()
        m.add_((g - m) * (1 - b1))
        v.add_((g.square() - v) * (1 - b2))
        w = w - rate * DECAY * w - rate / (1 - b1**t) * m / ((v / (1 - b2**t)).sqrt() + ADAM_EPS)
        new["p"].append(w)
        new["w"] += [w] if case["masters"] else []
        new["m"].append(m)
        new["v"].append(v)
    return new["p"] + new["w"] + new["m"] + new["v"]


def exact(case, seed):
    x = _inputs(case, seed)
    if case["kind"] == "packed":
        return _packed64(case, x)
    if case["kind"] == "loss":
        return _loss64(case, x)
    return _adamw64(case, x, _rate(seed))
