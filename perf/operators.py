"""What the token operators are timed on: embedding rows and their gradient, routing to experts and its gradient, the
experts' products and theirs.

A case is a dict of plain values.  `listed()` names the fixed ones, `draw(rng)` gives one more of the same ranges,
`prepare(case, seed)` makes what a user's program holds before the call, `run(state)` is one pass and `work(case)` the
bytes and operations that a pass cannot do without.  With `own` false a pass is the operator's plain form, elementary
torch operations in 32 bits (64 where choices next to a border depend on it); with `own` true it is the library's
call.  `exact(case, seed)` is the operator's definition in 64 bits.

Run with the repository's root as the working folder.
"""
from __future__ import annotations

import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i32": torch.int32, "i64": torch.int64}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "i32": 4, "i64": 8}


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
        # Serving: the one token that a sequence has just been given.  Latency.
        {"name": "embed_one_bf16", "op": "embed", "count": 1, "vocab": 32000, "width": 4096, "type": "bf16",
         "out": "bf16", "index": "i64", "alpha": 1.0},
        # A batch of prompts, rows scaled by the square root of their width.
        {"name": "embed_prompt_bf16", "op": "embed", "count": 16384, "vocab": 128000, "width": 4096, "type": "bf16",
         "out": "bf16", "index": "i64", "alpha": 64.0},
        # Training of a small model on one short sequence: a handful of rows of the table get a gradient; odd sizes.
        {"name": "embed_grad_odd_f32", "op": "embed_grad", "count": 509, "vocab": 10007, "width": 777, "type": "f32",
         "out": "f32", "index": "i64", "alpha": 1.0},
        # A training step: word frequencies after Zipf, gradients of 16 bits summed into the table's of 32.
        {"name": "embed_grad_bf16", "op": "embed_grad", "count": 16384, "vocab": 65536, "width": 2048, "type": "bf16",
         "out": "f32", "index": "i32", "alpha": 1.0},
        # Serving: one token's experts.  Latency.
        {"name": "route_one_bf16", "op": "route", "tokens": 1, "experts": 64, "k": 8, "score": "softmax",
         "bias": False, "groups": 1, "kept": 1, "group_score": "max", "renormalise": True, "scale": 1.0,
         "type": "bf16", "value": "f32"},
        # A batch of prompts over many experts in groups, with the bias that balances their load.
        {"name": "route_prompt_groups", "op": "route", "tokens": 16384, "experts": 256, "k": 8, "score": "sigmoid",
         "bias": True, "groups": 8, "kept": 4, "group_score": "top2", "renormalise": True, "scale": 2.5,
         "type": "f32", "value": "f32"},
        # Training, odd sizes: the gradient of sigmoid weights.
        {"name": "route_grad_odd_f32", "op": "route_grad", "tokens": 3001, "experts": 60, "k": 6, "score": "sigmoid",
         "renormalise": True, "scale": 1.0, "type": "f32", "value": "f32"},
        # A training step: the gradient of softmax weights.
        {"name": "route_grad_bf16", "op": "route_grad", "tokens": 16384, "experts": 128, "k": 8, "score": "softmax",
         "renormalise": True, "scale": 1.0, "type": "bf16", "value": "f32"},
        # Serving: sixteen sequences, a token each.  The weights of the experts that they reach are read once.
        {"name": "experts_decode_bf16", "op": "experts", "tokens": 16, "experts": 64, "k": 8, "in": 2048, "out": 1024,
         "type": "bf16", "skew": 0.5},
        # A batch of prompts.
        {"name": "experts_prompt_bf16", "op": "experts", "tokens": 8192, "experts": 32, "k": 4, "in": 2048, "out": 2048,
         "type": "bf16", "skew": 0.5},
        # Training, odd sizes and uneven experts: gradients of the rows and of the weights.
        {"name": "experts_grad_ragged_f16", "op": "experts_grad", "tokens": 1003, "experts": 17, "k": 3, "in": 1000,
         "out": 520, "type": "f16", "skew": 1.0},
        # A training step.
        {"name": "experts_grad_bf16", "op": "experts_grad", "tokens": 4096, "experts": 16, "k": 2, "in": 1024,
         "out": 2048, "type": "bf16", "skew": 0.5},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["embed", "embed_grad", "route", "route_grad", "experts", "experts_grad"])
    if op in ("embed", "embed_grad"):
        width = _log(rng, 64, 4096)
        if rng.random() < 0.7:
            width = (width + 7) // 8 * 8
        most = 128000 if op == "embed" else min(65536, (1 << 27) // width)
        kind = rng.choice(["f32", "f16", "bf16"])
        return {"op": op, "count": _log(rng, 1, 16384), "vocab": _log(rng, 1000, most), "width": width, "type": kind,
                "out": rng.choice([kind, "f32"]), "index": rng.choice(["i32", "i64"]),
                "alpha": rng.choice([1.0, 0.125, math.sqrt(width)])}
    if op in ("route", "route_grad"):
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * max(4, _log(rng, 8, 256) // groups)
        kept = rng.randint((groups + 1) // 2, groups)
        k = rng.randint(1, min(8, kept * (experts // groups)))
        score = rng.choice(["softmax", "sigmoid"])
        case = {"op": op, "tokens": _log(rng, 1, 16384), "experts": experts, "k": k, "score": score,
                "renormalise": rng.random() < 0.7, "scale": rng.choice([1.0, 2.5]), "type": rng.choice(["f32", "bf16", "f16"]),
                "value": "f32"}
        if op == "route":
            case |= {"bias": rng.random() < 0.5, "groups": groups, "kept": kept,
                     "group_score": rng.choice(["max", "top2"])}
        return case
    experts = _log(rng, 4, 64)
    step = rng.choice([8, 8, 64, 1])
    sizes = [max(64, _log(rng, 64, 2048) // step * step) for _ in range(2)]
    return {"op": op, "tokens": _log(rng, 1, 8192 if op == "experts" else 4096), "experts": experts,
            "k": rng.randint(1, min(experts, 8 if op == "experts" and sizes[0] * sizes[1] <= 1 << 20 else 4)),
            "in": sizes[0], "out": sizes[1], "type": rng.choice(["bf16", "f16"]), "skew": rng.choice([0.0, 0.5, 1.0])}


def work(case):
    op = case["op"]
    if op in ("embed", "embed_grad"):
        n, h = case["count"], case["width"]
        rows = n if op == "embed" else case["vocab"]
        return {"bytes": n * (BYTES[case["index"]] + h * BYTES[case["type"]]) + rows * h * BYTES[case["out"]],
                "flops": n * h}
    if op == "route":
        t, e, k = case["tokens"], case["experts"], case["k"]
        return {"bytes": t * e * BYTES[case["type"]] + 4 * e * case["bias"] + t * k * (4 + BYTES[case["value"]]) + 4 * (t + 1),
                "flops": 5 * t * e}
    if op == "route_grad":
        t, e, k = case["tokens"], case["experts"], case["k"]
        chosen = case["renormalise"] or case["score"] == "sigmoid"  # otherwise every logit of the row is read
        return {"bytes": t * (k if chosen else e) * BYTES[case["type"]] + t * e * BYTES[case["type"]]
                + t * k * (4 + 2 * BYTES[case["value"]]), "flops": 5 * t * (k if chosen else e)}
    t, e, k, n, d, s = case["tokens"], case["experts"], case["k"], case["out"], case["in"], BYTES[case["type"]]
    reached = e * (1.0 - (1.0 - k / e) ** t)
    if op == "experts":
        return {"bytes": int(s * (t * d + reached * d * n + t * k * n) + 4 * t * k), "flops": 2 * t * k * d * n}
    # rows' gradients: dY and W in, dX out; weights' gradients: dY and X in, dW out (whole, zeros of the others too)
    return {"bytes": int(s * (t * k * n + t * d + reached * d * n + t * k * d + e * d * n) + 4 * t * k),
            "flops": 4 * t * k * d * n}


# ---------------------------------------------------------------- inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, kind, size=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * size).to(DTYPE[kind])


def _tokens(g, case):
    """Word frequencies after Zipf (1 / (rank + 2.7)), the words in no order."""
    v = case["vocab"]
    u = torch.rand(case["count"], generator=g, device="cuda", dtype=torch.float64)
    rank = (2.7 * ((v + 2.7) / 2.7) ** u - 2.7).long().clamp(0, v - 1)
    return torch.randperm(v, generator=g, device="cuda")[rank].to(DTYPE[case["index"]])


def _chosen(g, t, e, k, skew):
    """k experts for every token, ascending; some experts are liked better than others."""
    x = torch.randn((t, e), generator=g, device="cuda") + skew * torch.randn(e, generator=g, device="cuda")
    return x.topk(k, dim=1).indices.sort(dim=1).values.to(torch.int32)


def _logits(g, case):
    """As a trained router gives them: some experts are liked better than others."""
    t, e = case["tokens"], case["experts"]
    x = torch.randn((t, e), generator=g, device="cuda") * 1.5 + 0.5 * torch.randn(e, generator=g, device="cuda")
    return x.to(DTYPE[case["type"]])


def _inputs(case, seed):
    g, op = _generator(seed), case["op"]
    if op == "embed":
        table = _normal(g, (case["vocab"], case["width"]), case["type"], 0.02 if case["alpha"] != 0.125 else 1.0)
        return {"table": table, "tokens": _tokens(g, case)}
    if op == "embed_grad":
        return {"tokens": _tokens(g, case), "grad": _normal(g, (case["count"], case["width"]), case["type"])}
    if op == "route":
        bias = 0.1 * torch.randn(case["experts"], generator=g, device="cuda") if case["bias"] else None
        return {"logits": _logits(g, case), "bias": bias}
    if op == "route_grad":
        x = _logits(g, case)
        t, k = case["tokens"], case["k"]
        columns = x.float().topk(k, dim=1).indices.sort(dim=1).values
        p = torch.softmax(x.double(), 1) if case["score"] == "softmax" else torch.sigmoid(x.double())
        w = p.gather(1, columns)
        w = case["scale"] * (w / w.sum(1, keepdim=True) if case["renormalise"] else w)
        return {"logits": x, "columns": columns.to(torch.int32), "values": w.to(DTYPE[case["value"]]),
                "grad": _normal(g, (t, k), case["value"])}
    t, e, k, n, d = case["tokens"], case["experts"], case["k"], case["out"], case["in"]
    made = {"columns": _chosen(g, t, e, k, case["skew"]), "x": _normal(g, (t, d), case["type"])}
    made["w"] = _normal(g, (e, n, d), case["type"], 1.0 / math.sqrt(d))
    if op == "experts_grad":
        made["grad"] = _normal(g, (t * k, n), case["type"])
    return made


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if not own:
        return state
    # What a program of the library's keeps: a handle, descriptors, outputs and buffers.
    package()
    from ops_sparse_b200 import api
    op, h = case["op"], api.Handle()
    new = lambda shape, kind: torch.empty(shape, dtype=DTYPE[kind], device="cuda")  # noqa: E731
    mat = lambda t: api.DnMat.row_major(t)  # noqa: E731
    state |= {"api": api, "handle": h}
    if op == "embed":
        out = new((case["count"], case["width"]), case["out"])
        state |= {"result": out, "args": (mat(state["table"]), api.DnVec(state["tokens"]), mat(out))}
    elif op == "embed_grad":
        out = new((case["vocab"], case["width"]), case["out"])
        args = (mat(state["grad"]), api.DnVec(state["tokens"]), mat(out))
        size = api.embedding_grad_buffer_size(h, *args)
        state |= {"result": out, "args": args, "buffer": torch.empty(size, dtype=torch.uint8, device="cuda")}
    else:
        t, e, k = case["tokens"], case["experts"], case["k"]
        offsets = torch.arange(0, t * k + 1, k, dtype=torch.int32, device="cuda")
        if op in ("route", "route_grad"):
            state["rule"] = api.RouteRule(score=case["score"], groups=case.get("groups", 1), kept=case.get("kept", 1),
                                          group_score=case.get("group_score", "max"),
                                          renormalise=case["renormalise"], scale=case["scale"])
        if op == "route":
            columns, values = new(t * k, "i32"), new(t * k, case["value"])
            state |= {"result": (columns.view(t, k), values.view(t, k)),
                      "args": (mat(state["logits"]), api.CsrMatrix(torch.empty_like(offsets), columns, values, t, e)),
                      "bias_d": None if state["bias"] is None else api.DnVec(state["bias"])}
        elif op == "route_grad":
            out = torch.empty_like(state["logits"])
            R = api.CsrMatrix(offsets, state["columns"].view(-1), state["values"].view(-1), t, e)
            state |= {"result": out, "args": (mat(state["logits"]), R, api.DnVec(state["grad"].view(-1)), mat(out))}
        else:
            n, d = case["out"], case["in"]
            R = api.CsrMatrix(offsets, state["columns"].view(-1), new(t * k, "f32"), t, e)
            X, W = mat(state["x"]), mat(state["w"].view(e * n, d))
            if op == "experts":
                y = new((t * k, n), case["type"])
                Y = mat(y)
                size = api.experts_buffer_size(h, R, X, W, Y)
                state |= {"result": y, "args": (R, X, W, Y)}
            else:
                dx, dw = new((t * k, d), case["type"]), new((e, n, d), case["type"])
                G, DX, DW = mat(state["grad"]), mat(dx), mat(dw.view(e * n, d))
                size = max(api.experts_buffer_size(h, R, G, W, DX, transpose=False, rows="entries"),
                           api.experts_grad_buffer_size(h, R, G, X, DW))
                state |= {"result": (dx, dw), "args": (R, G, X, W, DX, DW)}
            state["buffer"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    return state


# ---------------------------------------------------------------- a pass

def run(state):
    case = state["case"]
    return (_call if own else _plain)(case["op"], case, state)


def _call(op, case, s):
    api, h, args = s["api"], s["handle"], s["args"]
    if op == "embed":
        api.embedding(h, *args, alpha=case["alpha"])
    elif op == "embed_grad":
        api.embedding_grad(h, *args, alpha=case["alpha"], buffer=s["buffer"])
    elif op == "route":
        api.route(h, s["rule"], args[0], s["bias_d"], args[1])
    elif op == "route_grad":
        api.route_grad(h, s["rule"], *args)
    elif op == "experts":
        R, X, W, Y = args
        api.experts_preprocess(h, R, s["buffer"])
        api.experts_mm(h, R, X, W, Y, buffer=s["buffer"])
    else:
        R, G, X, W, DX, DW = args
        api.experts_preprocess(h, R, s["buffer"])
        api.experts_mm(h, R, G, W, DX, transpose=False, rows="entries", buffer=s["buffer"])
        api.experts_grad(h, R, G, X, DW, buffer=s["buffer"])
    return s["result"]


def _plain(op, case, s):
    if op == "embed":
        return (case["alpha"] * s["table"][s["tokens"].long()].float()).to(DTYPE[case["out"]])
    if op == "embed_grad":
        out = torch.zeros((case["vocab"], case["width"]), device="cuda")
        out.index_add_(0, s["tokens"].long(), s["grad"].float())
        return (case["alpha"] * out).to(DTYPE[case["out"]])
    if op == "route":
        return _plain_route(case, s["logits"], s["bias"])
    if op == "route_grad":
        return _plain_route_grad(case, s["logits"].float(), s["columns"].long(), s["grad"].float())
    # the entries by expert; every expert's rows in one product
    t, e, k = case["tokens"], case["experts"], case["k"]
    experts = s["columns"].view(-1).long()
    order = torch.sort(experts, stable=True).indices
    counts = torch.bincount(experts, minlength=e).tolist()
    rows, kind = order // k, DTYPE[case["type"]]
    if op == "experts":
        y, at = torch.empty((t * k, case["out"]), dtype=kind, device="cuda"), 0
        for i, c in enumerate(counts):
            if c:
                y[order[at:at + c]] = (s["x"][rows[at:at + c]].float() @ s["w"][i].float().T).to(kind)
            at += c
        return y
    dx, dw, at = torch.empty((t * k, case["in"]), dtype=kind, device="cuda"), torch.zeros_like(s["w"]), 0
    for i, c in enumerate(counts):
        if c:
            g = s["grad"][order[at:at + c]].float()
            dx[order[at:at + c]] = (g @ s["w"][i].float()).to(kind)
            dw[i] = (g.T @ s["x"][rows[at:at + c]].float()).to(kind)
        at += c
    return dx, dw


def _plain_route(case, logits, bias):
    t, e, groups = case["tokens"], case["experts"], case["groups"]
    x = logits.double()  # neighbours in the order of the scores may lie closer than 32 bits tell apart
    p = torch.exp(x - x.amax(1, keepdim=True)) if case["score"] == "softmax" else 1 / (1 + torch.exp(-x))
    p = p / p.sum(1, keepdim=True) if case["score"] == "softmax" else p
    # without a bias the scores ascend with the logits
    by = p + bias.double() if bias is not None else x
    if groups > 1:
        inside = (by if bias is not None or case["group_score"] == "max" else p).view(t, groups, e // groups)
        best = inside.sort(dim=2, descending=True).values[:, :, :1 if case["group_score"] == "max" else 2].sum(2)
        kept = best.sort(dim=1, descending=True, stable=True).indices[:, :case["kept"]]
        open_ = torch.zeros((t, groups), dtype=torch.bool, device="cuda").scatter_(1, kept, True)
        by = torch.where(open_.repeat_interleave(e // groups, dim=1), by, -math.inf)
    columns = by.sort(dim=1, descending=True, stable=True).indices[:, :case["k"]].sort(dim=1).values
    w = p.float().gather(1, columns)
    if case["renormalise"]:
        w = w / w.sum(1, keepdim=True)
    return columns.to(torch.int32), (case["scale"] * w).to(DTYPE[case["value"]])


def _plain_route_grad(case, x, columns, g):
    out = torch.zeros_like(x)
    if case["score"] == "softmax":
        p = torch.exp(x - x.amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
        w = p.gather(1, columns)
        if case["renormalise"]:
            w = w / w.sum(1, keepdim=True)
            out.scatter_(1, columns, case["scale"] * w * (g - (g * w).sum(1, keepdim=True)))
        else:
            out = -case["scale"] * p * (g * w).sum(1, keepdim=True)
            out.scatter_add_(1, columns, case["scale"] * w * g)
    else:
        s = 1 / (1 + torch.exp(-x.gather(1, columns)))
        if case["renormalise"]:
            total = s.sum(1, keepdim=True)
            g = (g - (g * s).sum(1, keepdim=True) / total) / total
        out.scatter_(1, columns, case["scale"] * g * s * (1 - s))
    return out.to(DTYPE[case["type"]])


# ---------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    """Written row by row or expert by expert from the definitions, by other operations than the plain forms."""
    s, op = _inputs(case, seed), case["op"]
    if op == "embed":
        return torch.index_select(s["table"], 0, s["tokens"].long()).double().mul_(case["alpha"])
    if op == "embed_grad":
        # rows in the order of their tokens; differences of running sums would cancel: token by token
        tokens, order = torch.sort(s["tokens"].long(), stable=True)
        found, counts = torch.unique_consecutive(tokens, return_counts=True)
        out = torch.zeros((case["vocab"], case["width"]), dtype=torch.float64, device="cuda")
        rows, at = s["grad"].double()[order], 0
        ends = torch.cumsum(counts, 0)
        for c in torch.unique(counts).tolist():  # tokens that occur equally often at once
            which = (counts == c).nonzero()[:, 0]
            start = ends[which] - c
            for j in range(c):
                out[found[which]] += rows[start + j]
        del at
        return out.mul_(case["alpha"])
    if op == "route":
        x = s["logits"].double().cpu().numpy()
        return _exact_route(case, x, None if s["bias"] is None else s["bias"].double().cpu().numpy())
    if op == "route_grad":
        # by differentiation of the weights
        x = s["logits"].double().requires_grad_()
        p = torch.softmax(x, 1) if case["score"] == "softmax" else torch.sigmoid(x)
        w = torch.take_along_dim(p, s["columns"].long(), 1)
        if case["renormalise"]:
            w = w / w.sum(1, keepdim=True)
        return torch.autograd.grad((w * s["grad"].double()).sum() * case["scale"], x)[0]
    if work(case)["flops"] > 4e11:
        return None
    columns, k = s["columns"].long(), case["k"]
    x = s["x"].double()
    if op == "experts":
        y = torch.empty((case["tokens"], k, case["out"]), dtype=torch.float64, device="cuda")
        for i in range(case["experts"]):
            token, place = (columns == i).nonzero(as_tuple=True)
            y[token, place] = torch.einsum("td,nd->tn", x[token], s["w"][i].double())
        return y.view(-1, case["out"])
    g = s["grad"].double().view(case["tokens"], k, -1)
    dx = torch.empty((case["tokens"], k, case["in"]), dtype=torch.float64, device="cuda")
    dw = torch.empty(s["w"].shape, dtype=torch.float64, device="cuda")
    for i in range(case["experts"]):
        token, place = (columns == i).nonzero(as_tuple=True)
        dx[token, place] = torch.einsum("tn,nd->td", g[token, place], s["w"][i].double())
        dw[i] = torch.einsum("tn,td->nd", g[token, place], x[token])
    return dx.view(-1, case["in"]), dw


def _exact_route(case, x, bias):
    import numpy as np
    t, e, groups, k = case["tokens"], case["experts"], case["groups"], case["k"]
    if case["score"] == "softmax":
        p = np.exp(x - x.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
    else:
        p = 0.5 * (1 + np.tanh(0.5 * x))
        low = x < -1  # where the sum above would cancel
        p[low] = np.exp(x[low]) / (1 + np.exp(x[low]))
    by = x.copy() if bias is None else p + bias
    if groups > 1:
        inside = (p if bias is None and case["group_score"] == "top2" else by).reshape(t, groups, -1)
        best = inside.max(2) if case["group_score"] == "max" else np.partition(inside, -2, axis=2)[:, :, -2:].sum(2)
        place = np.argsort(np.argsort(-best, axis=1, kind="stable"), axis=1)
        by[np.repeat(place >= case["kept"], e // groups, axis=1)] = -np.inf
    columns = np.sort(np.argsort(-by, axis=1, kind="stable")[:, :k], axis=1)
    w = np.take_along_axis(p, columns, 1)
    if case["renormalise"]:
        w = w / w.sum(1, keepdims=True)
    return torch.from_numpy(columns.astype(np.int32)), torch.from_numpy(case["scale"] * w)
