"""What the operators around the experts' rows are timed on: rows of tokens in the order of their experts and back, with
the weights and the gradient, and products in 8-bit integers with a scale for each token and channel, of all rows with one
matrix and of the experts' rows with theirs.

A case is a dict of plain values.  `listed()` names the fixed ones, `draw(rng)` gives one more of the same ranges,
`prepare(case, seed)` makes what a user's program holds before the call, `run(state)` is one pass and `work(case)` the
bytes and operations that a pass cannot do without.  With `own` false a pass is the operator's plain form, elementary
torch operations in 32 bits (64 where a rounding to 8 bits lies next to a border); with `own` true it is the library's
calls.  `exact(case, seed)` is the operator's definition in 64 bits.

The ops: "dispatch" orders the entries of a routing by expert and lays every token's row out in that order; "combine" sums
a token's rows, with the routing's weights or, as the gradient of "dispatch", without; "combine_grad" is the gradient of a
weighted "combine"; "scaled" rounds a batch of rows to 8 bits and multiplies them by a matrix that is kept in 8 bits;
"experts_scaled" does so for a routing, every token's row by its experts' matrices, results in the order of the experts.

Run with the repository's root as the working folder.
"""
from __future__ import annotations

import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def package():
    name = "ops_sparse_b200"
    if name not in sys.modules:
        folder = Path.cwd() / "ops-sparse_b200"
        spec = importlib.util.spec_from_file_location(name, folder / "__init__.py",
                                                      submodule_search_locations=[str(folder)])
        module = importlib.util.module_from_spec(spec)
        sys.modules[name] = module
        spec.loader.exec_module(module)
    return sys.modules[name]


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # Serving: the one token that a sequence has just been given, to its experts.  Latency.
        {"name": "dispatch_one_bf16", "op": "dispatch", "tokens": 1, "experts": 64, "k": 8, "width": 4096,
         "type": "bf16", "out": "bf16", "skew": 0.5},
        # A batch of prompts.
        {"name": "dispatch_prompt_bf16", "op": "dispatch", "tokens": 8192, "experts": 32, "k": 4, "width": 4096,
         "type": "bf16", "out": "bf16", "skew": 0.5},
        # Serving: one token's results.  Latency.
        {"name": "combine_one_f16", "op": "combine", "tokens": 1, "experts": 64, "k": 8, "width": 4096, "type": "f16",
         "out": "f16", "weighted": True, "skew": 0.5},
        # A batch of prompts.
        {"name": "combine_prompt_bf16", "op": "combine", "tokens": 8192, "experts": 64, "k": 8, "width": 2048,
         "type": "bf16", "out": "bf16", "weighted": True, "skew": 0.5},
        # Training: the gradient of the rows that were dispatched, summed into 32 bits.
        {"name": "dispatch_grad_bf16", "op": "combine", "tokens": 4096, "experts": 16, "k": 2, "width": 2048,
         "type": "bf16", "out": "f32", "weighted": False, "skew": 0.5},
        # Training of a small model on one short sequence; odd sizes, uneven experts.
        {"name": "combine_grad_odd_f32", "op": "combine_grad", "tokens": 509, "experts": 17, "k": 3, "width": 777,
         "type": "f32", "out": "f32", "skew": 1.0},
        # A training step.
        {"name": "combine_grad_bf16", "op": "combine_grad", "tokens": 8192, "experts": 32, "k": 4, "width": 2048,
         "type": "bf16", "out": "bf16", "skew": 0.5},
        # Serving: one token through a layer.  The matrix is read once.
        {"name": "scaled_one_bf16", "op": "scaled", "tokens": 1, "in": 4096, "out_width": 4096, "type": "bf16",
         "out": "bf16"},
        # Serving some sequences, a token each, through a layer of odd sizes.
        {"name": "scaled_batch_odd_f16", "op": "scaled", "tokens": 61, "in": 2040, "out_width": 1111, "type": "f16",
         "out": "f32"},
        # A batch of prompts through a wide layer.
        {"name": "scaled_prompt_bf16", "op": "scaled", "tokens": 8192, "in": 4096, "out_width": 8192, "type": "bf16",
         "out": "bf16"},
        # Serving: sixteen sequences, a token each.  The matrices of the experts that they reach are read once.
        {"name": "experts_scaled_decode_bf16", "op": "experts_scaled", "tokens": 16, "experts": 64, "k": 8, "in": 2048,
         "out_width": 1024, "type": "bf16", "out": "bf16", "skew": 0.5},
        # A batch of prompts.
        {"name": "experts_scaled_prompt_bf16", "op": "experts_scaled", "tokens": 8192, "experts": 32, "k": 4,
         "in": 2048, "out_width": 2048, "type": "bf16", "out": "bf16", "skew": 0.5},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    step = rng.choice([8, 8, 64, 1])
    return max(low, _log(rng, low, high) // step * step)


def draw(rng):
    op = rng.choice(["dispatch", "combine", "combine_grad", "scaled", "experts_scaled"])
    kind = rng.choice(["f32", "f16", "bf16"])
    if op == "scaled":
        return {"op": op, "tokens": _log(rng, 1, 8192), "in": _width(rng, 64, 4096), "out_width": _width(rng, 64, 8192),
                "type": kind, "out": rng.choice([kind, "f32"])}
    experts = _log(rng, 4, 64)
    case = {"op": op, "tokens": _log(rng, 1, 8192), "experts": experts, "k": rng.randint(1, min(8, experts)), "type": kind,
            "out": rng.choice([kind, "f32"]) if op in ("dispatch", "combine") else kind, "skew": rng.choice([0.0, 0.5, 1.0])}
    if op == "experts_scaled":
        case |= {"in": _width(rng, 64, 2048), "out_width": _width(rng, 64, 2048)}
        case["k"] = min(case["k"], max(1, 32768 // case["tokens"]))
        return case
    if op == "combine":
        case["weighted"] = rng.random() < 0.6
    # up to 320 MB of rows: those of the tokens and of the entries, of which a gradient reads some and writes others
    moved = {"dispatch": lambda s, o, k: s + k * o, "combine": lambda s, o, k: k * s + o,
             "combine_grad": lambda s, o, k: s + 2 * k * s}[op](BYTES[case["type"]], BYTES[case["out"]], case["k"])
    case["width"] = min(_width(rng, 64, 4096), (320 << 20) // (case["tokens"] * moved))
    return case


def work(case):
    op, t = case["op"], case["tokens"]
    s, o = BYTES[case["type"]], BYTES[case["out"]]
    if op == "scaled":
        n, d = case["out_width"], case["in"]
        return {"bytes": t * d * s + n * d + 4 * n + t * n * o, "flops": 2 * t * n * d}
    e, k = case["experts"], case["k"]
    if op == "experts_scaled":
        n, d = case["out_width"], case["in"]
        reached = e * (1.0 - (1.0 - k / e) ** t)
        return {"bytes": int(t * d * s + reached * n * (d + 4) + t * k * (4 + n * o)), "flops": 2 * t * k * n * d}
    h = case["width"]
    if op == "dispatch":  # columns and rows in; rows and the experts' first ones out
        return {"bytes": t * h * s + t * k * (4 + h * o) + 4 * (e + 1), "flops": t * k * h}
    if op == "combine":  # places, weights and rows in
        return {"bytes": t * k * (4 + 4 * case["weighted"] + h * s) + t * h * o, "flops": 2 * t * k * h}
    # places, weights, gradient and rows in; the rows' and the weights' gradients out
    return {"bytes": t * h * s + t * k * (12 + 2 * h * s), "flops": 3 * t * k * h}


# ---------------------------------------------------------------- inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, kind, size=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * size).to(DTYPE[kind])


def _chosen(g, t, e, k, skew):
    """k experts for every token, ascending; some experts are liked better than others."""
    x = torch.randn((t, e), generator=g, device="cuda") + skew * torch.randn(e, generator=g, device="cuda")
    return x.topk(k, dim=1).indices.sort(dim=1).values.to(torch.int32)


def _weights_8(g, rows, width):
    """A matrix in 8 bits with a scale for each of its rows, as it was rounded when the model was loaded.  Its rows start
    on 16 bytes."""
    w = torch.randn((rows, width), generator=g, device="cuda") / math.sqrt(width)
    top = w.abs().amax(1, keepdim=True)
    held = torch.zeros((rows, (width + 15) // 16 * 16), dtype=torch.int8, device="cuda")
    held[:, :width] = torch.round(127 * (w / top)).to(torch.int8)
    return held[:, :width], (top / 127)[:, 0].contiguous()


def _inputs(case, seed):
    g, op, t = _generator(seed), case["op"], case["tokens"]
    if op == "scaled":
        x = _normal(g, (t, case["in"]), case["type"])
        w, scales = _weights_8(g, case["out_width"], case["in"])
        return {"x": x, "w": w, "w_scales": scales}
    e, k = case["experts"], case["k"]
    made = {"columns": _chosen(g, t, e, k, case["skew"])}
    if op == "experts_scaled":
        made["x"] = _normal(g, (t, case["in"]), case["type"])
        made["w"], made["w_scales"] = _weights_8(g, e * case["out_width"], case["in"])
        return made
    h = case["width"]
    if op == "dispatch":
        made["x"] = _normal(g, (t, h), case["type"])
        return made
    made["values"] = torch.softmax(torch.randn((t, k), generator=g, device="cuda"), 1)
    made["rows"] = _normal(g, (t * k, h), case["type"])
    if op == "combine_grad":
        made["grad"] = _normal(g, (t, h), case["type"])
    return made


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    op, t = case["op"], case["tokens"]
    if not own:
        if op in ("combine", "combine_grad"):
            # The order that the rows lie in was made when they were dispatched.
            order = torch.sort(state["columns"].view(-1).long(), stable=True).indices
            places = torch.empty_like(order)
            places[order] = torch.arange(t * case["k"], device="cuda")
            state |= {"places": places.view(t, case["k"])}
        return state
    # What a program of the library's keeps: a handle, descriptors, outputs and buffers.
    package()
    from ops_sparse_b200 import api
    h = api.Handle()
    new = lambda shape, kind: torch.empty(shape, dtype=DTYPE[kind], device="cuda")  # noqa: E731
    raw = lambda size: torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")  # noqa: E731
    mat, vec = api.DnMat.row_major, api.DnVec
    state |= {"api": api, "handle": h}
    if op in ("scaled", "experts_scaled"):
        d, n = case["in"], case["out_width"]
        rows = t if op == "scaled" else t * case["k"]
        q = torch.empty((rows, (d + 15) // 16 * 16), dtype=torch.int8, device="cuda")[:, :d]
        scales, y = new(rows, "f32"), new((rows, n), case["out"])
        X, Q, W, Y = mat(state["x"]), mat(q), mat(state["w"]), mat(y)
        S, WS = vec(scales), vec(state["w_scales"])
        state["result"] = y
        if op == "scaled":
            state |= {"args": (X, Q, S, W, WS, Y), "buffer": raw(api.scaled_mm_buffer_size(h, Q, W, Y))}
            return state
    e, k = case["experts"], case["k"]
    offsets = torch.arange(0, t * k + 1, k, dtype=torch.int32, device="cuda")
    values = state["values"].view(-1) if "values" in state else new(t * k, "f32")
    R = api.CsrMatrix(offsets, state["columns"].view(-1), values, t, e)
    if op == "experts_scaled":
        state |= {"args": (R, X, Q, S, W, WS, Y), "buffer": raw(api.experts_scaled_mm_buffer_size(h, R, Q, W, Y))}
        return state
    state["buffer"] = raw(api.experts_order_buffer_size(h, R))
    width = case["width"]
    if op == "dispatch":
        out, starts = new((t * k, width), case["out"]), torch.empty(e + 1, dtype=torch.int32, device="cuda")
        state |= {"result": (out, starts), "args": (R, mat(state["x"]), mat(out), vec(starts))}
        return state
    api.experts_preprocess(h, R, state["buffer"])
    rows = mat(state["rows"])
    if op == "combine":
        out = new((t, width), case["out"])
        state |= {"result": out, "args": (R, rows, mat(out))}
    else:
        d_rows, d_values = new((t * k, width), case["type"]), new((t, k), "f32")
        state |= {"result": (d_rows, d_values),
                  "args": (R, mat(state["grad"]), rows, mat(d_rows), vec(d_values.view(-1)))}
    return state


# ---------------------------------------------------------------- a pass

def run(state):
    case = state["case"]
    return (_call if own else _plain)(case["op"], case, state)


def _call(op, case, s):
    api, h, args, buffer = s["api"], s["handle"], s["args"], s["buffer"]
    if op == "dispatch":
        R, X, S, starts = args
        api.experts_preprocess(h, R, buffer)
        api.experts_dispatch(h, R, X, S, offsets=starts, buffer=buffer)
    elif op == "combine":
        api.experts_combine(h, *args, weighted=case["weighted"], buffer=buffer)
    elif op == "combine_grad":
        api.experts_combine_grad(h, *args, buffer=buffer)
    elif op == "scaled":
        X, Q, S, W, WS, Y = args
        api.quantise_rows(h, X, Q, S)
        api.scaled_mm(h, Q, S, W, WS, Y, buffer=buffer)
    else:
        R, X, Q, S, W, WS, Y = args
        api.experts_preprocess(h, R, buffer)
        api.experts_quantise(h, R, X, Q, S, buffer=buffer)
        api.experts_scaled_mm(h, R, Q, S, W, WS, Y, buffer=buffer)
    return s["result"]


def _by_expert(case, columns):
    """The entries in the order of their experts, and how many every expert has."""
    experts = columns.view(-1).long()
    return torch.sort(experts, stable=True).indices, torch.bincount(experts, minlength=case["experts"])


def _plain_rounded(x):
    """Rows as whole numbers of up to 127, and their scales."""
    top = x.double().abs().amax(1, keepdim=True)
    q = torch.where(top > 0, torch.round(127 * x.double() / top), 0.0)
    return q.float(), top.float() / 127


def _plain(op, case, s):
    kind = DTYPE[case["out"]]
    if op == "dispatch":
        order, counts = _by_expert(case, s["columns"])
        starts = torch.zeros(case["experts"] + 1, dtype=torch.int32, device="cuda")
        starts[1:] = counts.cumsum(0)
        return s["x"][order // case["k"]].to(kind), starts
    if op == "combine":
        rows = s["rows"][s["places"]].float()
        if case["weighted"]:
            rows = rows * s["values"][:, :, None]
        return rows.sum(1).to(kind)
    if op == "combine_grad":
        grad = s["grad"].float()
        d_rows = torch.empty_like(s["rows"])
        d_rows[s["places"]] = (s["values"][:, :, None] * grad[:, None]).to(kind)
        return d_rows, (s["rows"][s["places"]].float() * grad[:, None]).sum(2)
    q, scales = _plain_rounded(s["x"])
    if op == "scaled":
        return ((q @ s["w"].float().T) * scales * s["w_scales"]).to(kind)
    # every expert's rows in one product
    order, counts = _by_expert(case, s["columns"])
    rows, n = order // case["k"], case["out_width"]
    y, at = torch.empty((len(order), n), dtype=kind, device="cuda"), 0
    for i, c in enumerate(counts.tolist()):
        if c:
            token, w = rows[at:at + c], slice(i * n, (i + 1) * n)
            y[at:at + c] = ((q[token] @ s["w"][w].float().T) * scales[token] * s["w_scales"][w]).to(kind)
        at += c
    return y


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_rounded(x):
    """Whole numbers by comparison with the borders between them, which 64 bits hold: a border itself goes to the even one."""
    x = x.double()
    size = x.abs()
    top = size.amax(1, keepdim=True)
    q = torch.floor(127 * size / torch.where(top > 0, top, 1.0))
    over = 254 * size - (2 * q + 1) * top
    q = q + ((over > 0) | ((over == 0) & (top > 0) & (q % 2 == 1)))
    return torch.sign(x) * q, top / 127


def exact(case, seed):
    """Written expert by expert, or entry by entry of a row, from the definitions, by other operations than the plain forms."""
    s, op = _inputs(case, seed), case["op"]
    if op == "scaled":
        q, scales = _exact_rounded(s["x"])
        return torch.einsum("td,nd->tn", q, s["w"].double()) * (scales * s["w_scales"].double()[None])
    columns, k = s["columns"].long(), case["k"]
    found = [(columns == i).nonzero(as_tuple=True) for i in range(case["experts"])]  # tokens and their entries, by expert
    tokens, entries = torch.cat([f[0] for f in found]), torch.cat([f[1] for f in found])
    if op == "dispatch":
        starts = [0]
        for token, _ in found:
            starts.append(starts[-1] + len(token))
        return torch.index_select(s["x"], 0, tokens).double(), torch.tensor(starts, dtype=torch.int32, device="cuda")
    if op == "experts_scaled":
        q, scales = _exact_rounded(s["x"])
        n, parts = case["out_width"], []
        for i, (token, _) in enumerate(found):
            w = s["w"][i * n:(i + 1) * n].double() * s["w_scales"][i * n:(i + 1) * n].double()[:, None]
            parts.append(torch.einsum("td,nd->tn", q[token] * scales[token], w))
        return torch.cat(parts)
    w = s["values"].double()
    if op == "combine":
        out = torch.zeros((case["tokens"], case["width"]), dtype=torch.float64, device="cuda")
        rows = s["rows"].double()
        for j in range(k):  # a token has one j-th entry
            which = (entries == j).nonzero()[:, 0]
            out[tokens[which]] += rows[which] * (w[tokens[which], j][:, None] if case["weighted"] else 1.0)
        return out
    grad = s["grad"].double()
    d_rows = torch.index_select(grad, 0, tokens) * w[tokens, entries][:, None]
    d_values = torch.zeros((case["tokens"], k), dtype=torch.float64, device="cuda")
    d_values[tokens, entries] = torch.einsum("ih,ih->i", s["rows"].double(), grad[tokens])
    return d_rows, d_values
