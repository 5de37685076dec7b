"""Lowering of the operators of ``functional/operators.py``, ``optimizer.py``, ``packed.py`` and
``linear_cross_entropy.py``: a ``fusion`` of each name becomes a built-in step whose
descriptor and pointers this module makes from the operands' places (``include/nhip.h``).

Unlike the generated kernels these read rows: an operand whose view would not keep its last axis contiguous (or, where
the kernel takes no strides, any axis) is copied by a loop kernel instead of being read through the view.
"""

from __future__ import annotations

import ctypes as C

from lumen_amd import dtypes as D
from lumen_amd.graph.ir import ELEMENTWISE, Graph

KINDS = {
    "qk_norm_rope": "heads_fwd",
    "qk_norm_rope_backward": "heads_bwd",
    "gated_linear": "gated_fwd",
    "gated_linear_grad": "gated_grad",
    "gated_input_grad": "gated_input",
    "gated_weight_grad": "gated_weight",
    "clip_grad_norm": "clip",
    "adamw": "adamw",
    "packed_attention": "packed_fwd",
    "packed_attention_backward": "packed_bwd",
    "head_loss": "head_loss",
    "head_loss_backward": "head_loss",
}
BOTH = "gated_both"  # a gated_weight and a gated_input step in one
STEPS = {*KINDS.values(), BOTH}
NHIP_DT = {"float32": 0, "bfloat16": 1, "float16": 2}
# The last axis contiguous; rows that start on 16 bytes; these, or all of a length that the library copies itself; every
# axis contiguous; and from 16 bytes on.
ROWS, CHUNK_ROWS, WIDE_ROWS, DENSE, WIDE = "rows", "chunk rows", "wide rows", "dense", "wide"


def _wants(node):
    """How the kernel reads each operand of ``node``."""
    name = node.params["name"]
    if name.startswith("qk_norm_rope"):
        return [ROWS if r in ("q", "k", "gq", "gk") else DENSE for r in node.params["roles"]]
    if name == "gated_linear":
        return [WIDE_ROWS, WIDE, WIDE]
    if name in ("gated_input_grad", "gated_weight_grad"):
        return [WIDE] * len(node.inputs)
    if name == "gated_linear_grad":
        return [ROWS, DENSE, DENSE]
    if name in ("head_loss", "head_loss_backward"):
        return [WIDE_ROWS, WIDE] + [DENSE] * (len(node.inputs) - 2)
    if name == "packed_attention":
        return [CHUNK_ROWS] * 3 + [DENSE]
    if name == "packed_attention_backward":
        return [CHUNK_ROWS] * 3 + [DENSE] + [CHUNK_ROWS, DENSE, CHUNK_ROWS, DENSE]
    return [DENSE] * len(node.inputs)


def _fusions(step):
    return [n for n in step.nodes if n.prim == "fusion"]


def layouts(steps) -> dict:
    """The layouts that each value read by such steps must have, each of its readers' (none stands for another: rows on 16 bytes
    need not be contiguous, nor contiguous ones start on 16). An eval loss's step over a product reads contiguous operands too."""
    out = {}
    for st in steps:
        if st.kind in STEPS:
            for node in _fusions(st):
                for v, want in zip(node.inputs, _wants(node)):
                    out.setdefault(v, set()).add(want)
        elif st.kind == "linear_cross_entropy":
            for v in st.nodes[0].inputs:
                out.setdefault(v, set()).add(DENSE)
    return out


def reads(loc, wants) -> bool:
    """Whether a place has every layout of ``wants``."""
    return all(_reads(loc, want) for want in wants)


def _reads(loc, want) -> bool:
    if want in (WIDE, WIDE_ROWS, CHUNK_ROWS) and loc.offset * D.size_of(loc.dtype) % 16:
        return False
    if want in (DENSE, WIDE):
        return loc.contiguous()
    if loc.shape and loc.shape[-1] != 1 and loc.strides[-1] != 1:
        return False
    if want == CHUNK_ROWS:
        return all(n == 1 or st % 8 == 0 for n, st in zip(loc.shape[:-1], loc.strides))
    if want == WIDE_ROWS and loc.shape[-1] % 8 == 0:  # [rows, k]; tiles of 256 rows within 2^31 bytes, as head_check has it
        return loc.strides[0] % 8 == 0 and 256 * loc.strides[0] + loc.shape[-1] < (1 << 30) - 1024
    return True


def _heads_desc(node, types):
    """``nhip_heads_desc`` of a heads node without its strides; ``types`` of its operands by role."""
    from lumen_amd import native as nv

    p = node.params
    q, k, cos = types["q"], types["k"], types["cos"]
    d = nv.HeadsDesc()
    d.batch, d.seq, d.heads, d.head_dim = q.shape
    d.kv_heads = k.shape[2]
    d.rot, d.table_rows = 2 * cos.shape[1], cos.shape[0]
    d.dtype = NHIP_DT[q.dtype]
    d.positions = nv.NHIP_POS_NONE
    if "positions" in types:
        d.positions = nv.NHIP_POS_I64 if types["positions"].dtype == "int64" else nv.NHIP_POS_I32
    d.interleaved, d.eps = int(p["interleaved"]), p["eps"]
    return d


def _roles(graph, node):
    return {r: graph.types[v] for r, v in zip(node.params["roles"], node.inputs)}


def scratch_bytes(graph, node) -> int:
    """Workspace bytes of the step, as the library reports them."""
    from lumen_amd import native as nv

    n, name = C.c_size_t(), node.params["name"]
    if name == "qk_norm_rope_backward":
        nv.call("nhip_qk_norm_rope_workspace", C.byref(_heads_desc(node, _roles(graph, node))), C.byref(n))
    elif name == "gated_linear":
        nv.call("nhip_gated_linear_workspace", C.byref(_gated_node_desc(graph, node)), C.byref(n))
    elif name in ("gated_input_grad", "gated_weight_grad"):
        nv.call("nhip_gated_backward_workspace", C.byref(_gated_backward_desc(graph, node)), C.byref(n))
    elif name in ("head_loss", "head_loss_backward"):
        nv.call("nhip_head_loss_workspace", C.byref(_head_desc(graph, node)), int(name != "head_loss"), C.byref(n))
    elif name in ("packed_attention", "packed_attention_backward"):
        n.value = _packed_workspace(graph, node)
        if name != "packed_attention":
            read = {m.params["index"] for m in graph.nodes if m.prim == "fusion_output" and m.inputs[0] == node.output}
            n.value += sum(_up256(graph.types[node.inputs[i]].nbytes()) for i in (1, 2) if i not in read)
    elif name == "clip_grad_norm":
        nv.call("nhip_clip_grad_norm_workspace", C.byref(nv.ClipDesc(count=len(_clip_grads(node)))), C.byref(n))
    return _up256(n.value)


def pair_gradients(graph, steps) -> list:
    """``steps`` with the weights' and the input's gradients of one gated projection as one step where the library runs
    both in one launch and nothing between them reads the first's results."""
    from lumen_amd import native as nv
    from lumen_amd.compiler.fusion import Step

    steps, paired = list(steps), C.c_int()
    for weight in [st for st in steps if st.kind == "gated_weight"]:
        node = weight.nodes[0]
        other = next((st for st in steps if st.kind == "gated_input" and st.nodes[0].inputs[0] == node.inputs[0]), None)
        if other is None:
            continue
        nv.call("nhip_gated_backward_paired", C.byref(_gated_backward_desc(graph, node)), C.byref(paired))
        first, last = (i for i, st in enumerate(steps) if st is weight or st is other)
        if not paired.value or any(v in st.inputs for st in steps[first + 1:last + 1] for v in steps[first].outputs):
            continue
        both = Step(BOTH, weight.nodes + other.nodes, weight.outputs + other.outputs,
                    weight.inputs + [v for v in other.inputs if v not in weight.inputs])
        both.scratch = max(weight.scratch, other.scratch)
        steps[last] = both
        del steps[first]
    return steps


def _outputs(plan, step, node=None) -> dict:
    """The places of the step's outputs by their index in the body of ``node`` (by default its first), those that nothing
    reads left out."""
    node = step.nodes[0] if node is None else node
    index = {n.output: n.params["index"] for n in plan.graph.nodes
             if n.prim == "fusion_output" and n.inputs[0] == node.output}
    index[node.output] = 0
    return {index[v]: plan.loc[v] for v in step.outputs if v in index}


def lower(plan, step):
    """``(step kind, descriptor bytes, [(pointer slot, place)])`` of an operator's step."""
    name = step.nodes[0].params["name"]
    if step.kind == BOTH:
        return _lower_gated_both(plan, step)
    if name.startswith("qk_norm_rope"):
        return _lower_heads(plan, step)
    return {"gated_linear": _lower_gated, "gated_linear_grad": _lower_gated_grad,
            "gated_input_grad": _lower_gated_backward, "gated_weight_grad": _lower_gated_backward,
            "clip_grad_norm": _lower_clip, "adamw": _lower_adamw,
            "packed_attention": _lower_packed, "packed_attention_backward": _lower_packed,
            "head_loss": _lower_head, "head_loss_backward": _lower_head}[name](plan, step)


def _slots(places):
    return [(i, loc) for i, loc in enumerate(places) if loc is not None]


def _lower_heads(plan, step):
    from lumen_amd import native as nv

    node = step.nodes[0]
    at = {r: plan.loc[v] for r, v in zip(node.params["roles"], node.inputs)}
    d = _heads_desc(node, _roles(plan.graph, node))
    out = _outputs(plan, step)
    backward = step.kind == "heads_bwd"
    weights = iter([out.get(2), out.get(3)])
    dw = [next(weights) if r in at else None for r in ("q_weight", "k_weight")]
    places = [("q", at["q"]), ("k", at["k"]), ("oq", out.get(0)), ("ok", out.get(1))]
    if backward:
        places += [("dq", at["gq"]), ("dk", at["gk"])]
    for prefix, loc in places:
        if loc is not None:
            for axis, i in (("b", 0), ("s", 1), ("n", 2)):
                setattr(d, f"{prefix}_{axis}", loc.strides[i])
    # keys of which nothing is read are left out (the first result, the queries', always has a place)
    if out.get(1) is None and not (backward and dw[1] is not None):
        d.kv_heads = 0
    head = [at["q"], at["k"], at.get("q_weight"), at.get("k_weight"), at["cos"], at["sin"], at.get("positions")]
    if not backward:
        return nv.NHIP_STEP_HEADS, bytes(d), _slots(head + [out.get(0), out.get(1)])
    return nv.NHIP_STEP_HEADS_BWD, bytes(d), _slots(head + [at["gq"], at["gk"], out.get(0), out.get(1), *dw,
                                                           plan.scratch.get(id(step))])


def _gated_desc(dtype, activation, m, n, k):
    from lumen_amd import native as nv

    d = nv.GatedDesc(m=m, n=n, k=k, x_m=k, w_n=k, h_m=n, config=-1)
    d.dtype, d.activation = NHIP_DT[dtype], nv.NHIP_ACT[activation]
    return d


def _gated_node_desc(graph, node):
    x, gate = (graph.types[v] for v in node.inputs[:2])
    return _gated_desc(x.dtype, node.params["activation"], x.shape[0], gate.shape[0], x.shape[1])


def _lower_gated(plan, step):
    from lumen_amd import native as nv

    node = step.nodes[0]
    d = _gated_node_desc(plan.graph, node)
    places = [plan.loc[v] for v in node.inputs]
    d.x_m = places[0].strides[0]
    out = _outputs(plan, step)
    return nv.NHIP_STEP_GATED, bytes(d), _slots(places + [out[0], out.get(1), out.get(2), plan.scratch.get(id(step))])


def _gated_backward_desc(graph, node):
    dgu, other = (graph.types[v] for v in node.inputs[:2])  # the gate weight [features, k], or x [tokens, k]
    return _gated_desc(dgu.dtype, "silu", dgu.shape[0], node.params["features"], other.shape[1])


def _lower_gated_backward(plan, step):
    from lumen_amd import native as nv

    node = step.nodes[0]
    kind = nv.NHIP_STEP_GATED_INPUT if step.kind == "gated_input" else nv.NHIP_STEP_GATED_WEIGHT
    out = _outputs(plan, step)
    places = [plan.loc[v] for v in node.inputs]
    places += [out[0], out.get(1)] if step.kind == "gated_weight" else [out[0]]
    return kind, bytes(_gated_backward_desc(plan.graph, node)), _slots(places + [plan.scratch.get(id(step))])


def _lower_gated_both(plan, step):
    from lumen_amd import native as nv

    weight, given = _fusions(step)
    dw, dx = (_outputs(plan, step, n) for n in (weight, given))
    places = [plan.loc[v] for v in (*given.inputs, weight.inputs[1])]
    return (nv.NHIP_STEP_GATED_BACKWARD, bytes(_gated_backward_desc(plan.graph, given)),
            _slots(places + [dx[0], dw[0], dw.get(1), plan.scratch.get(id(step))]))


def _lower_gated_grad(plan, step):
    from lumen_amd import native as nv

    node, g = step.nodes[0], plan.graph
    dh = g.types[node.inputs[0]]
    d = _gated_desc(dh.dtype, node.params["activation"], dh.shape[0], dh.shape[1], 0)
    places = [plan.loc[v] for v in node.inputs]
    d.h_m = places[0].strides[0]
    return nv.NHIP_STEP_GATED_GRAD, bytes(d), _slots(places + [_outputs(plan, step)[0]])


def _clip_grads(node):
    return node.inputs if node.params["max_norm"] is not None else node.inputs[1:]


def _lower_clip(plan, step):
    from lumen_amd import native as nv

    node, g = step.nodes[0], plan.graph
    grads, p = _clip_grads(node), node.params
    bound = p["max_norm"]
    d = nv.ClipDesc(count=len(grads), max_norm=0.0 if bound is None else bound, eps=p["eps"])
    tensors = (nv.ClipTensor * len(grads))()
    out = _outputs(plan, step)
    ops = _slots([None if bound is not None else plan.loc[node.inputs[0]], out[0], out.get(1), plan.scratch[id(step)]])
    for i, v in enumerate(grads):
        t = g.types[v]
        tensors[i].numel, tensors[i].dtype = t.numel(), NHIP_DT[t.dtype]
        ops.append((4 + 2 * i, plan.loc[v]))
        if 2 + i in out:
            ops.append((5 + 2 * i, out[2 + i]))
    return nv.NHIP_STEP_CLIP, bytes(d) + bytes(tensors), ops


def _packed_desc(graph, node):
    """``nhip_packed_desc`` of a packed attention node without its strides."""
    from lumen_amd import native as nv
    from lumen_amd.compiler.attention import stored_ds_bytes

    q, k, v, offsets = (graph.types[u] for u in node.inputs[:4])
    d = nv.PackedDesc(causal=int(node.params["causal"]), scale=node.params["scale"], dtype=NHIP_DT[q.dtype])
    d.tokens, d.heads, d.head_dim = q.shape
    d.kv_heads, d.value_head_dim, d.sequences = k.shape[1], v.shape[2], offsets.shape[0] - 1
    d.offsets_dtype = nv.NHIP_POS_I64 if offsets.dtype == "int64" else nv.NHIP_POS_I32
    d.ds_bytes = stored_ds_bytes()
    return d


def _packed_workspace(graph, node) -> int:
    from lumen_amd import native as nv

    n = C.c_size_t()
    nv.call("nhip_packed_workspace", C.byref(_packed_desc(graph, node)), int(node.params["name"] != "packed_attention"), C.byref(n))
    return _up256(n.value)


def _up256(n) -> int:
    return -(-n // 256) * 256


def _dense(t, at):
    """A contiguous place of type ``t`` at byte ``at`` of the workspace."""
    from lumen_amd.compiler.plan import Loc, _contig

    return Loc(("ws", 0), at // D.size_of(t.dtype), _contig(t.shape), t.dtype, t.shape)


def _lower_packed(plan, step):
    from lumen_amd import native as nv

    node = step.nodes[0]
    d, out = _packed_desc(plan.graph, node), _outputs(plan, step)
    at = [plan.loc[v] for v in node.inputs]
    backward = step.kind == "packed_bwd"
    names = [("q", at[0]), ("k", at[1]), ("v", at[2])]
    if backward:
        # the kernels compute all three gradients: one that nothing reads goes into the scratch
        spare = plan.scratch[id(step)].offset * 4 + _packed_workspace(plan.graph, node)
        for index, operand in ((1, 1), (2, 2)):
            if index not in out:
                t = plan.graph.types[node.inputs[operand]]
                out[index] = _dense(t, spare)
                spare += _up256(t.nbytes())
        names += [("o", at[4]), ("do", at[6]), ("dq", out[0]), ("dk", out[1]), ("dv", out[2])]
    else:
        names.append(("o", out[0]))
    for name, loc in names:
        # the library takes strides of whole 16 bytes; that of an axis of one element, any number in a view, is not used
        d_s, d_n = (0 if n == 1 else st for n, st in zip(loc.shape, loc.strides[:2]))
        setattr(d, f"{name}_s", d_s)
        setattr(d, f"{name}_n", d_n)
    scratch = plan.scratch[id(step)]
    if not backward:
        return nv.NHIP_STEP_PACKED_FWD, bytes(d), _slots([*at, out[0], out.get(1), out.get(2), scratch])
    return nv.NHIP_STEP_PACKED_BWD, bytes(d), _slots([*at, *(loc for _, loc in names[5:]), scratch])


def _head_desc(graph, node):
    from lumen_amd import native as nv
    from lumen_amd.config import config

    h, w, target = (graph.types[v] for v in node.inputs[:3])
    d = nv.HeadDesc(rows=h.shape[0], classes=w.shape[0], k=h.shape[1], h_m=h.shape[1], w_n=h.shape[1],
                    ignore_index=node.params["ignore"], piece_bytes=config.compiler.head_piece_bytes, dtype=NHIP_DT[h.dtype])
    d.target_dtype = nv.NHIP_LCE_I64 if target.dtype == "int64" else nv.NHIP_LCE_I32
    return d


def _lower_head(plan, step):
    from lumen_amd import native as nv

    node = step.nodes[0]
    d, out = _head_desc(plan.graph, node), _outputs(plan, step)
    at = [plan.loc[v] for v in node.inputs]
    if d.rows > 1:
        d.h_m = at[0].strides[0]
    scratch = plan.scratch.get(id(step))
    if node.params["name"] == "head_loss":
        return nv.NHIP_STEP_HEAD_LOSS, bytes(d), _slots([*at, None, out[0], None, None, scratch])
    return nv.NHIP_STEP_HEAD_LOSS, bytes(d), _slots([*at, out.get(2), out[0], out.get(1), scratch])


def losses_with_gradients(graph: Graph) -> Graph:
    """The losses of a vocabulary head whose gradients are computed too come from the gradients' step, which computes them
    anyway, where the losses' cotangents do not depend on them: one product over the classes less."""
    forward = {}
    for n in graph.nodes:
        if n.prim == "fusion" and n.params["name"] == "head_loss":
            forward.setdefault((n.inputs, n.params["ignore"]), n)
    if not forward:
        return graph
    depends = {}  # value -> the losses that it depends on
    pairs, needs = {}, {}  # loss -> the gradients that it is to come from, and the losses that these depend on

    def from_gradients(loss, target):
        """Whether `loss` is `target` or comes to depend on it by the pairs that there are."""
        seen, todo = set(), [loss]
        while todo:
            v = todo.pop()
            if v == target:
                return True
            if v not in seen:
                seen.add(v)
                todo += needs.get(v, ())
        return False

    for n in graph.nodes:
        found = frozenset().union(*(depends.get(v, ()) for v in n.inputs))
        if n.prim == "fusion" and n.params["name"] == "head_loss":
            found |= {n.output}
        elif n.prim == "fusion" and n.params["name"] == "head_loss_backward":
            f = forward.get((n.inputs[:3], n.params["ignore"]))
            if f is not None and f.output not in pairs and not any(from_gradients(v, f.output) for v in found):
                pairs[f.output], needs[f.output] = n, found
        if found:
            depends[n.output] = found
    if not pairs:
        return graph
    g = Graph()
    remap = {v: g.input(graph.types[v].dtype, graph.types[v].shape) for v in graph.inputs}
    by_gradients = {b.output: v for v, b in pairs.items()}
    # what depends on a loss that is taken over comes after everything else
    waiting = [n for n in graph.nodes if n.output not in pairs]
    while waiting:
        later = []
        for n in waiting:
            if not all(v in remap for v in n.inputs):
                later.append(n)
                continue
            remap[n.output] = g.add_node(n.prim, tuple(remap[v] for v in n.inputs), n.params, graph.types[n.output], n.backward)
            if n.output in by_gradients:
                loss = by_gradients[n.output]
                ty = graph.types[loss]
                remap[loss] = g.add_node("fusion_output", (remap[n.output],), {"index": 2, "ty": ty}, ty, n.backward)
        waiting = later
    g.set_outputs([remap[v] for v in graph.outputs])
    return g


def _adamw_tensors(node):
    """The operands of each of an ``adamw`` node's weights: its values (or its master's), gradient and moments."""
    from lumen_amd.functional.optimizer import OPERANDS, adamw_scalars

    rest = node.inputs[len(adamw_scalars(node.params)):]
    return [rest[i:i + OPERANDS] for i in range(0, len(rest), OPERANDS)]


def _adamw_results(node):
    """The index in the body's results of each weight's new value, moments and (None: none) master."""
    masters = node.params["masters"]
    n, at = len(masters), iter(range(3 * len(masters), 4 * len(masters)))
    return [(i, n + i, 2 * n + i, next(at) if m else None) for i, m in enumerate(masters)]


def _lower_adamw(plan, step):
    from lumen_amd import native as nv
    from lumen_amd.functional.optimizer import adamw_scalars

    node, g, p = step.nodes[0], plan.graph, step.nodes[0].params
    names, out = adamw_scalars(p), _outputs(plan, step)
    weights = _adamw_tensors(node)
    d = nv.AdamwDesc(count=len(weights), lr=p["lr"] or 0.0, step=p["step"] or 1.0, beta1=p["beta1"], beta2=p["beta2"],
                     eps=p["eps"], weight_decay=p["weight_decay"])
    if "step" in names:
        d.step_type = {"int32": nv.NHIP_POS_I32, "int64": nv.NHIP_POS_I64}.get(g.types[node.inputs[names.index("step")]].dtype,
                                                                              nv.NHIP_POS_NONE)
    tensors = (nv.AdamwTensor * len(weights))()
    ops = [(("lr", "step", "scale").index(n), plan.loc[v]) for n, v in zip(names, node.inputs)]
    for i, ((w, grad, m, v), results) in enumerate(zip(weights, _adamw_results(node))):
        t = g.types[grad]
        tensors[i].numel, tensors[i].dtype = t.numel(), NHIP_DT[t.dtype]
        new, first, second, master = (out.get(j) for j in results)
        places = [None if p["masters"][i] else plan.loc[w], plan.loc[grad], plan.loc[m], plan.loc[v],
                  plan.loc[w] if p["masters"][i] else None, new, first, second, master]
        ops += [(3 + 9 * i + j, loc) for j, loc in enumerate(places) if loc is not None]
    return nv.NHIP_STEP_ADAMW, bytes(d) + bytes(tensors), ops


def writes_over(graph, node, result, operand) -> bool:
    """Whether a step of ``node`` may write its ``result`` over its operand ``operand``, or over another value that it does
    not read: an element of a weight's results is written by the thread that has read that element of its operands."""
    if node.params["name"] != "adamw":
        return False
    index = next((n.params["index"] for n in graph.nodes if n.prim == "fusion_output" and n.output == result), 0)
    own = next(k for k, r in enumerate(_adamw_results(node)) if index in r)
    return operand not in node.inputs[:len(node.inputs) - sum(map(len, _adamw_tensors(node)))] \
        and all(k == own for k, xs in enumerate(_adamw_tensors(node)) if operand in xs)


def _clipped_steps(graph, clips, users):
    """The ``adamw`` nodes that may take the clipping's scale themselves, by output: every gradient of theirs is a result of
    one clipping that only such nodes (as their gradients) and elementwise ones read."""
    from lumen_amd.functional.optimizer import OPERANDS, adamw_scalars

    clipped = {n.output: n.inputs[0] for n in graph.nodes if n.prim == "fusion_output" and n.inputs[0] in clips
               and n.params["index"] >= 2 and n.output not in graph.outputs}
    steps = {n.output: n for n in graph.nodes if n.prim == "fusion" and n.params.get("name") == "adamw"
             and not n.params["scaled"]}

    def gradients(n):
        return n.inputs[len(adamw_scalars(n.params)) + 1::OPERANDS]

    def only_gradients(v, u):
        return u.output in steps and u.inputs.count(v) == gradients(u).count(v)

    while True:
        bad = [k for k, n in steps.items() if len({clipped.get(v) for v in gradients(n)} | {None}) != 2
               or any(v not in clipped or not all(u.prim in ELEMENTWISE or only_gradients(v, u) for u in users[v])
                      for v in gradients(n))]
        if not bad:
            return steps
        for k in bad:
            del steps[k]


def clip_in_consumers(graph: Graph) -> Graph:
    """A clipped gradient that only elementwise nodes and AdamW steps read (an optimizer's update) is multiplied by the
    scale there instead of being written by the clipping step and read again: the same values, one pass over the gradient
    less."""
    from lumen_amd.functional.optimizer import OPERANDS, adamw_body, adamw_scalars
    from lumen_amd.graph import tracer
    from lumen_amd.graph.ir import TensorType

    users = graph.users()
    clips = {n.output: n for n in graph.nodes if n.prim == "fusion" and n.params.get("name") == "clip_grad_norm"}
    steps = _clipped_steps(graph, clips, users) if clips else {}
    moved = {}
    for n in graph.nodes:
        if n.prim == "fusion_output" and n.inputs[0] in clips and n.params["index"] >= 2 \
                and n.output not in graph.outputs and users.get(n.output) \
                and all(u.prim in ELEMENTWISE or u.output in steps for u in users[n.output]):
            moved[n.output] = _clip_grads(clips[n.inputs[0]])[n.params["index"] - 2]
    if not moved:
        return graph
    clip_of = {n.output: n.inputs[0] for n in graph.nodes if n.output in moved}
    g = Graph()
    remap = {v: g.input(graph.types[v].dtype, graph.types[v].shape) for v in graph.inputs}
    scale = {}

    def scale_of(clip, backward):
        """The step's scale, float32: the body's second result."""
        if clip not in scale:
            f32 = TensorType("float32", ())
            scale[clip] = g.add_node("fusion_output", (remap[clip],), {"index": 1, "ty": f32}, f32, backward)
        return scale[clip]

    def scaled_step(n):
        """The AdamW step over the gradients as they were, with their scale."""
        names = adamw_scalars(n.params)
        head, rest = [remap[v] for v in n.inputs[:len(names)]], list(n.inputs[len(names):])
        clip = clip_of[rest[1]]
        ins = head + [scale_of(clip, n.backward)] + [
            remap[moved[v]] if i % OPERANDS == 1 else remap[v] for i, v in enumerate(rest)]
        params = {k: v for k, v in n.params.items() if k not in ("name", "body")}
        params["scaled"] = True
        body = Graph()
        xs = [tracer.TracedTensor(body, body.input(g.types[v].dtype, g.types[v].shape)) for v in ins]
        with tracer.tracing(body):
            body.set_outputs([r.var for r in adamw_body(xs, params)])
        return g.add_node("fusion", tuple(ins), dict(params, name="adamw", body=body), graph.types[n.output], n.backward)

    for n in graph.nodes:
        if n.output in steps:
            remap[n.output] = scaled_step(n)
            continue
        if n.output not in moved:
            remap[n.output] = g.add_node(n.prim, tuple(remap[v] for v in n.inputs), n.params, graph.types[n.output], n.backward)
            continue
        if not any(u.prim in ELEMENTWISE for u in users[n.output]):
            continue
        ty = graph.types[n.output]
        wide = TensorType("float32", ty.shape)
        grad, factor = remap[moved[n.output]], scale_of(n.inputs[0], n.backward)
        if ty.dtype != "float32":
            grad = g.add_node("cast", (grad,), {"new_dtype": "float32"}, wide, n.backward)
        if ty.shape:
            factor = g.add_node("broadcast_in_dim", (factor,), {"shape": ty.shape, "broadcast_dimensions": ()}, wide, n.backward)
        v = g.add_node("mul", (grad, factor), {}, wide, n.backward)
        if ty.dtype != "float32":
            v = g.add_node("cast", (v,), {"new_dtype": ty.dtype}, ty, n.backward)
        remap[n.output] = v
    g.set_outputs([remap[v] for v in graph.outputs])
    g.prune()
    return g
