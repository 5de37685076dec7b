"""Three operators that a training step or a decoding step of a decoder calls beside its products and attention, as
cases that can be timed and checked:

* ``F.qk_norm_rope``: the RMS norm of each query and key head and its rotation by position, ahead of attention;
* ``F.gated_linear``: the gate and up projections of a gated MLP, the activation and their product;
* ``F.clip_grad_norm``: the 2-norm over every gradient of a model, and the gradients scaled by it.

Each in both directions where it has two. With ``own`` false ``run`` computes them from elementary torch operations
in float32; with ``own`` true it calls the compiled functions that a program of this framework makes of them.
"""

import functools
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16, "int32": torch.int32}
NAMES = {v: k for k, v in DTYPES.items()}
EPS = 2.0**-20  # added to a head's mean square
CLIP_EPS = 1e-6  # added to the norm that a bound is divided by


def listed():
    return [
        # one new token of each of 16 sequences at positions of their own: latency counts
        dict(name="heads_decode", kind="heads", train=False, b=16, s=1, n=16, nkv=16, d=128, rot=128, table=32768,
             positions=True, packed=False, interleaved=False, dtype="bfloat16"),
        # a prompt of odd length with grouped key heads, read in place from the merged projection, half of each head
        # rotated, neighbouring elements paired
        dict(name="heads_prefill", kind="heads", train=False, b=2, s=1777, n=16, nkv=4, d=64, rot=32, table=2048,
             positions=True, packed=True, interleaved=True, dtype="float16"),
        # a layer of the 12-layer model in training: both directions, gradients of the norms' weights too
        dict(name="heads_train", kind="heads", train=True, b=4, s=4096, n=16, nkv=16, d=128, rot=128, table=4096,
             positions=False, packed=False, interleaved=False, dtype="bfloat16"),
        # float32, a head dim and a rotated part that are no powers of two, a ragged sequence
        dict(name="heads_train_odd", kind="heads", train=True, b=3, s=331, n=6, nkv=2, d=80, rot=40, table=512,
             positions=True, packed=False, interleaved=False, dtype="float32"),
        # one token through the 2-layer model's sizes: the smallest call
        dict(name="gated_token", kind="gated", train=False, tokens=1, dim=512, ffn=2048, activation="silu",
             dtype="bfloat16"),
        # one new token of each of 16 sequences: the weights read once
        dict(name="gated_decode", kind="gated", train=False, tokens=16, dim=2048, ffn=8192, activation="silu",
             dtype="bfloat16"),
        # a whole batch of prompts at the 12-layer model's sizes
        dict(name="gated_prefill", kind="gated", train=False, tokens=16384, dim=2048, ffn=8192, activation="silu",
             dtype="bfloat16"),
        # one sequence in training: the product and the gradients of the input and both weights
        dict(name="gated_train", kind="gated", train=True, tokens=4096, dim=2048, ffn=8192, activation="silu",
             dtype="bfloat16"),
        # a ragged batch of small odd sizes, float16, GELU
        dict(name="gated_train_odd", kind="gated", train=True, tokens=777, dim=520, ffn=1416, activation="gelu",
             dtype="float16"),
        # a few float32 gradients of odd sizes below their bound: launches count
        dict(name="clip_small", kind="clip", dim=130, ffn=333, vocab=517, seq=33, layers=1, clips=False, dtype="float32"),
        # the 2-layer model's gradients, over their bound
        dict(name="clip_step", kind="clip", dim=512, ffn=2048, vocab=32000, seq=512, layers=2, clips=True,
             dtype="bfloat16"),
        # five layers, embeddings and head at the 12-layer model's sizes: 475 million gradients
        dict(name="clip_large", kind="clip", dim=2048, ffn=8192, vocab=32000, seq=4096, layers=5, clips=True,
             dtype="bfloat16"),
    ]


# ---- drawn cases


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size of the range: mostly a multiple of 64, now and then of 8, now and then any."""
    n, q = _log(rng, lo, hi), rng.choice([64, 64, 64, 8, 8, 1])
    return max(q, n // q * q)


def _draw(rng):
    kind = rng.choice(["heads", "heads_train", "gated", "gated", "gated_train", "clip"])
    if kind.startswith("heads"):
        train = kind == "heads_train"
        d = rng.choice([64, 64, 128, 128, 256, 32, 80, 96, 36])
        n = rng.choice([2, 4, 6, 8, 16, 32])
        s = _log(rng, 33, 8192) if train or rng.random() < 0.5 else 1
        return dict(kind="heads", train=train, b=_log(rng, 1, 64) if s == 1 else _log(rng, 1, 8), s=s, n=n,
                    nkv=n // rng.choice([1, 1, 2]), d=d, rot=rng.choice([d, d, d // 2 // 2 * 2]),
                    table=s + _log(rng, 1, 32768), positions=rng.random() < 0.5 or s == 1,
                    packed=not train and rng.random() < 0.5, interleaved=rng.random() < 0.5,
                    dtype=rng.choice(["bfloat16", "bfloat16", "float16", "float32"]))
    if kind.startswith("gated"):
        return dict(kind="gated", train=kind == "gated_train", tokens=_log(rng, 1, 16384), dim=_size(rng, 128, 4096),
                    ffn=_size(rng, 256, 16384), activation=rng.choice(["silu", "silu", "gelu", "relu", "sigmoid"]),
                    dtype=rng.choice(["bfloat16", "bfloat16", "float16"]))
    return dict(kind="clip", dim=_size(rng, 32, 2048), ffn=_size(rng, 64, 8192), vocab=_log(rng, 100, 32000),
                seq=_log(rng, 16, 4096), layers=rng.choice([1, 2, 3, 5]), clips=rng.random() < 0.6,
                dtype=rng.choice(["bfloat16", "bfloat16", "float16", "float32"]))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 300)


def draw(rng):
    """A case of the same kinds and ranges that costs no more than the largest listed one."""
    most = max(_cost(c) for c in listed())
    while True:
        c = _draw(rng)
        if _cost(c) <= most:
            return c


# ---- inputs


def _normal(g, shape, dtype, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=g, device="cuda") * std + mean).to(DTYPES[dtype])


def _angles(case):
    """The cosines and sines of a rotary table, float32 of 64-bit angles: [positions, rot / 2]."""
    half = case["rot"] // 2
    freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / max(half, 1))
    angle = torch.arange(case["table"], dtype=torch.float64, device="cuda")[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _gradient_shapes(case):
    """The weights of a decoder with gated MLPs and normed heads, in the order that its modules list them."""
    d, f = case["dim"], case["ffn"]
    layer = [(d,), (d, d), (d, d), (d, d), (d, d), (64,), (64,), (d,), (f, d), (f, d), (d, f)]
    return [(case["vocab"], d), (case["seq"], d)] + layer * case["layers"] + [(d,), (case["vocab"], d)]


def _inputs(case, seed):
    """The case's inputs by name, torch tensors on the GPU, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind, dt = case["kind"], case["dtype"]
    if kind == "heads":
        b, s, n, nkv, d = case["b"], case["s"], case["n"], case["nkv"], case["d"]
        x = {}
        if case["packed"]:  # the merged projection of queries, keys and values
            x["qkv"] = _normal(g, (b, s, (n + 2 * nkv) * d), dt, std=1.5)
        else:
            x["q"], x["k"] = _normal(g, (b, s, n, d), dt, std=1.5), _normal(g, (b, s, nkv, d), dt, std=1.5)
        x["cos"], x["sin"] = _angles(case)
        x["wq"], x["wk"] = (_normal(g, (d,), dt, std=0.1, mean=1.0) for _ in range(2))
        if case["positions"]:  # documents of any length one after another, or the next position of a sequence
            start = torch.randint(0, case["table"] - s + 1, (b, 1), generator=g, device="cuda")
            x["positions"] = (start + torch.arange(s, device="cuda")).to(torch.int32)
        if case["train"]:
            x["dq"], x["dk"] = _normal(g, (b, s, n, d), dt), _normal(g, (b, s, nkv, d), dt)
        return x
    if kind == "gated":
        t, d, f = case["tokens"], case["dim"], case["ffn"]
        x = {"x": _normal(g, (t, d), dt), "gate": _normal(g, (f, d), dt, std=d**-0.5), "up": _normal(g, (f, d), dt, std=d**-0.5)}
        if case["train"]:
            x["dh"] = _normal(g, (t, f), dt)
        return x
    shapes = _gradient_shapes(case)
    return {f"g{i}": _normal(g, shape, dt, std=0.01) for i, shape in enumerate(shapes)}


def _bound(case):
    """The norm's bound: three tenths of what the gradients have on average, or twice that much."""
    count = sum(math.prod(s) for s in _gradient_shapes(case))
    return 0.01 * math.sqrt(count) * (0.3 if case["clips"] else 2.0)


def prepare(case, seed):
    x = _inputs(case, seed)
    state = {"case": dict(case), "x": x, "bound": _bound(case) if case["kind"] == "clip" else None}
    if own:
        _own_state(state)
    return state


# ---- the plain forms


def _split(case, x):
    """Queries and keys, as views of the merged projection where that is what there is."""
    if not case["packed"]:
        return x["q"], x["k"]
    b, s, n, nkv, d = case["b"], case["s"], case["n"], case["nkv"], case["d"]
    return x["qkv"][:, :, :n * d].reshape(b, s, n, d), x["qkv"][:, :, n * d:(n + nkv) * d].reshape(b, s, nkv, d)


def _rows(x, s):
    """The table's rows of each position, [b or 1, s, 1, rot / 2]."""
    if "positions" in x:
        at = x["positions"].long()
        return x["cos"][at][:, :, None], x["sin"][at][:, :, None]
    return x["cos"][None, :s, None], x["sin"][None, :s, None]


def _pairs(x, rot, interleaved):
    if interleaved:
        return x[..., 0:rot:2], x[..., 1:rot:2]
    return x[..., :rot // 2], x[..., rot // 2:rot]


def _joined(a, b, rest, interleaved):
    pairs = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((pairs, rest), -1)


def _rotated(x, cos, sin, rot, interleaved):
    a, b = _pairs(x, rot, interleaved)
    return _joined(a * cos - b * sin, b * cos + a * sin, x[..., rot:], interleaved)


def _heads_plain(case, x):
    rot, inter = case["rot"], case["interleaved"]
    cos, sin = _rows(x, case["s"])
    dtype = DTYPES[case["dtype"]]
    out, grads, weights = [], [], []

    def both(h, w, dy):
        h, w = h.float(), w.float()
        inv = torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
        xhat = h * inv
        out.append(_rotated(xhat * w, cos, sin, rot, inter).to(dtype))
        if dy is not None:
            dz = _rotated(dy.float(), cos, -sin, rot, inter)  # the rotation back
            dxhat = dz * w
            grads.append((inv * (dxhat - xhat * (dxhat * xhat).mean(-1, keepdim=True))).to(dtype))
            weights.append((dz * xhat).sum((0, 1, 2)).to(dtype))

    q, k = _split(case, x)
    both(q, x["wq"], x.get("dq"))
    both(k, x["wk"], x.get("dk"))
    return out + grads + weights


def _activation(name, g):
    """act(g) and its derivative."""
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if name == "sigmoid":
        s = torch.sigmoid(g)
        return s, s * (1 - s)
    if name == "relu":
        return torch.clamp(g, min=0), (g > 0).to(g.dtype)
    c = 0.7978845608
    t = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)


def _gated_plain(case, x):
    dtype = DTYPES[case["dtype"]]
    rows, gate, up = x["x"].float(), x["gate"].float(), x["up"].float()
    g, u = rows @ gate.t(), rows @ up.t()
    a, da = _activation(case["activation"], g)
    out = [(a * u).to(dtype)]
    if case["train"]:
        dh = x["dh"].float()
        du, dg = dh * a, dh * u * da
        out += [(dg @ gate + du @ up).to(dtype), (dg.t() @ rows).to(dtype), (du.t() @ rows).to(dtype)]
    return out


def _clip_plain(x, bound):
    squares = torch.stack([g.float().square().sum() for g in x.values()]).double()
    norm = squares.sum().sqrt().float()
    scale = torch.clamp(bound / (norm + CLIP_EPS), max=1.0)
    return [norm] + [(g.float() * scale).to(g.dtype) for g in x.values()]


def run(state):
    if own:
        return _own_run(state)
    case = state["case"]
    if case["kind"] == "heads":
        return _heads_plain(case, state["x"])
    if case["kind"] == "gated":
        return _gated_plain(case, state["x"])
    return _clip_plain(state["x"], state["bound"])


# ---- the framework's programs


def _heads(q, k, cos, sin, wq, wk, positions, interleaved):
    import lumen_amd.functional as F

    return F.qk_norm_rope(q, k, cos, sin, wq, wk, positions=positions, eps=EPS, interleaved=interleaved)


def _heads_program(q, k, cos, sin, wq, wk, positions, interleaved):
    return list(_heads(q, k, cos, sin, wq, wk, positions, interleaved))


def _heads_packed_program(qkv, cos, sin, wq, wk, positions, interleaved, n, nkv):
    b, s, width = qkv.shape
    d = width // (n + 2 * nkv)
    q, k = qkv[:, :, :n * d].reshape(b, s, n, d), qkv[:, :, n * d:(n + nkv) * d].reshape(b, s, nkv, d)
    return list(_heads(q, k, cos, sin, wq, wk, positions, interleaved))


def _heads_train_program(q, k, cos, sin, wq, wk, positions, interleaved, dq, dk):
    import lumen_amd as L

    def heads(q, k, wq, wk):
        return _heads(q, k, cos, sin, wq, wk, positions, interleaved)

    out, pullback = L.vjp(heads, q, k, wq, wk)
    return [*out, *pullback((dq, dk))]


def _gated_program(x, gate, up, activation):
    import lumen_amd.functional as F

    return [F.gated_linear(x, gate, up, activation=activation)]


def _gated_train_program(x, gate, up, activation, dh):
    import lumen_amd as L
    import lumen_amd.functional as F

    h, pullback = L.vjp(lambda x, gate, up: F.gated_linear(x, gate, up, activation=activation), x, gate, up)
    return [h, *pullback(dh)]


def _clip_program(bound, *grads):
    import lumen_amd.functional as F

    clipped, norm = F.clip_grad_norm(grads, bound, eps=CLIP_EPS)
    return [norm, *clipped]


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
    if case["kind"] == "heads":
        tail = [x["cos"], x["sin"], x["wq"], x["wk"], x.get("positions"), case["interleaved"]]
        if case["packed"]:
            fn, args = _heads_packed_program, [x["qkv"], *tail, case["n"], case["nkv"]]
        elif case["train"]:
            fn, args = _heads_train_program, [x["q"], x["k"], *tail, x["dq"], x["dk"]]
        else:
            fn, args = _heads_program, [x["q"], x["k"], *tail]
    elif case["kind"] == "gated":
        args = [x["x"], x["gate"], x["up"], case["activation"]]
        fn = _gated_program
        if case["train"]:
            fn, args = _gated_train_program, [*args, x["dh"]]
    else:
        fn, args = _clip_program, [state["bound"], *x.values()]
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
    if kind == "heads":
        tokens, d = case["b"] * case["s"], case["d"]
        heads = tokens * (case["n"] + case["nkv"]) * d * size
        table = min(tokens if case["positions"] else case["s"], case["table"]) * case["rot"] * 4
        rest = table + 2 * d * size + (4 * tokens if case["positions"] else 0)
        return {"bytes": (4 * heads if case["train"] else 2 * heads) + rest + (2 * d * size if case["train"] else 0), "flops": 0}
    if kind == "gated":
        t, d, f = case["tokens"], case["dim"], case["ffn"]
        if case["train"]:  # x, dh, h, dx and the weights with their gradients; six products
            return {"bytes": size * (2 * t * d + 2 * t * f + 4 * d * f), "flops": 12 * t * d * f}
        return {"bytes": size * (t * d + t * f + 2 * d * f), "flops": 4 * t * d * f}
    count = sum(math.prod(s) for s in _gradient_shapes(case))
    return {"bytes": 2 * size * count + 4, "flops": 0}


# ---- the same in 64 bits


def _heads64(case, x):
    """Each pair of a head as a complex number times exp(i angle), the angle's cosine and sine as given."""
    q, k = (t.double() for t in _split(case, x))
    wq, wk = x["wq"].double(), x["wk"].double()
    table = torch.complex(x["cos"].double(), x["sin"].double())
    turn = (table[x["positions"].long()] if "positions" in x else table[:case["s"]].unsqueeze(0)).unsqueeze(2)
    half = case["rot"] // 2

    def f(h, w):
        y = h / torch.sqrt(h.pow(2).mean(-1, keepdim=True) + EPS) * w
        part, rest = y[..., :2 * half], y[..., 2 * half:]
        if case["interleaved"]:
            z = torch.view_as_complex(part.reshape(*part.shape[:-1], half, 2).contiguous()) * turn
            part = torch.view_as_real(z).reshape(part.shape)
        else:
            z = torch.complex(part[..., :half].contiguous(), part[..., half:].contiguous()) * turn
            part = torch.cat((z.real, z.imag), -1)
        return torch.cat((part, rest), -1)

    if not case["train"]:
        return [f(q, wq), f(k, wk)]
    leaves = [t.requires_grad_() for t in (q, k, wq, wk)]
    out = [f(q, wq), f(k, wk)]
    grads = torch.autograd.grad(out, leaves, [x["dq"].double(), x["dk"].double()])
    return [*(y.detach() for y in out), *grads]


def _gated64(case, x):
    rows, gate, up = (x[n].double() for n in ("x", "gate", "up"))

    def act(g):
        if case["activation"] == "silu":
            return g / (1 + torch.exp(-g))
        if case["activation"] == "sigmoid":
            return 1 / (1 + torch.exp(-g))
        if case["activation"] == "relu":
            return g * (g > 0)
        return g / (1 + torch.exp(-2 * 0.7978845608 * (g + 0.044715 * g.pow(3))))  # 1 + tanh(v) is 2 / (1 + exp(-2 v))

    if not case["train"]:
        return [act(rows @ gate.t()) * (rows @ up.t())]
    leaves = [t.requires_grad_() for t in (rows, gate, up)]
    h = act(rows @ gate.t()) * (rows @ up.t())
    return [h.detach(), *torch.autograd.grad(h, leaves, x["dh"].double())]


def exact(case, seed):
    x = _inputs(case, seed)
    if case["kind"] == "heads":
        return _heads64(case, x)
    if case["kind"] == "gated":
        return _gated64(case, x)
    grads = [g.double() for g in x.values()]
    norm = math.sqrt(sum(float(g.pow(2).sum()) for g in grads))
    scale = min(1.0, _bound(case) / (norm + CLIP_EPS))
    return [torch.tensor(norm, dtype=torch.float64)] + [g * scale for g in grads]
