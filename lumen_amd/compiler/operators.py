"""Lowering of the operators of ``functional/operators.py``: a ``fusion`` of each name becomes a built-in step whose
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
}
BOTH = "gated_both"  # a gated_weight and a gated_input step in one
STEPS = {*KINDS.values(), BOTH}
NHIP_DT = {"float32": 0, "bfloat16": 1, "float16": 2}
# The last axis contiguous; and rows that start on 16 bytes, or all of a length that the library copies itself; every axis
# contiguous; and from 16 bytes on.
ROWS, WIDE_ROWS, DENSE, WIDE = "rows", "wide rows", "dense", "wide"
STRICTER = [ROWS, WIDE_ROWS, DENSE, WIDE]


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
    return [DENSE] * len(node.inputs)


def _fusions(step):
    return [n for n in step.nodes if n.prim == "fusion"]


def layouts(steps) -> dict:
    """The layout that each value read by such a step must have (the stricter of its readers')."""
    out = {}
    for st in steps:
        if st.kind in STEPS:
            for node in _fusions(st):
                for v, want in zip(node.inputs, _wants(node)):
                    out[v] = max(want, out.get(v, ROWS), key=STRICTER.index)
    return out


def reads(loc, want) -> bool:
    """Whether a place has the layout ``want`` (None: any)."""
    if want is None:
        return True
    if want in (WIDE, WIDE_ROWS) and loc.offset * D.size_of(loc.dtype) % 16:
        return False
    if want in (DENSE, WIDE):
        return loc.contiguous()
    if loc.shape and loc.shape[-1] != 1 and loc.strides[-1] != 1:
        return False
    if want == WIDE_ROWS and loc.shape[-1] % 8 == 0:  # [rows, k]; tiles of 256 rows within 2^31 bytes
        return loc.strides[0] % 8 == 0 and 256 * loc.strides[0] + loc.shape[-1] < 1 << 30
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
    elif name == "clip_grad_norm":
        nv.call("nhip_clip_grad_norm_workspace", C.byref(nv.ClipDesc(count=len(_clip_grads(node)))), C.byref(n))
    return -(-n.value // 256) * 256


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
            "clip_grad_norm": _lower_clip}[name](plan, step)


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


def clip_in_consumers(graph: Graph) -> Graph:
    """A clipped gradient that only elementwise nodes read (an optimizer's update) is multiplied by the scale there
    instead of being written by the clipping step and read again: the same values, one pass over the gradient less."""
    from lumen_amd.graph.ir import TensorType

    users = graph.users()
    clips = {n.output: n for n in graph.nodes if n.prim == "fusion" and n.params.get("name") == "clip_grad_norm"}
    moved = {}
    for n in graph.nodes:
        if n.prim == "fusion_output" and n.inputs[0] in clips and n.params["index"] >= 2 \
                and n.output not in graph.outputs and users.get(n.output) \
                and all(u.prim in ELEMENTWISE for u in users[n.output]):
            moved[n.output] = _clip_grads(clips[n.inputs[0]])[n.params["index"] - 2]
    if not moved:
        return graph
    g = Graph()
    remap = {v: g.input(graph.types[v].dtype, graph.types[v].shape) for v in graph.inputs}
    scale = {}

    def scale_of(clip, backward):
        """The step's scale, float32: the body's second result."""
        if clip not in scale:
            f32 = TensorType("float32", ())
            scale[clip] = g.add_node("fusion_output", (remap[clip],), {"index": 1, "ty": f32}, f32, backward)
        return scale[clip]

    for n in graph.nodes:
        if n.output not in moved:
            remap[n.output] = g.add_node(n.prim, tuple(remap[v] for v in n.inputs), n.params, graph.types[n.output], n.backward)
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
