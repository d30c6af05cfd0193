"""Plain implementations in 64 bits of the token operators, and the bounds their tests hold the kernels to.

A value that is rounded once to a type is off by half a step of it; f32 sums of n terms, in any order, by at most n * 2^-24 of
the sum of their absolute values.
"""
from __future__ import annotations

import math

import numpy as np
import torch

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
F32 = 2.0 ** -24


def rounding(dtype, value):
    """Half a step of the type at every value."""
    info = torch.finfo(dtype)
    smallest = info.tiny * info.eps  # the step of the subnormals
    return (value.abs() * (info.eps / 2)).clamp_min(smallest / 2)


def close(got, want, bound, what=""):
    """Every finite element of want within its bound; the others equal."""
    got, want, bound = got.double().cpu(), want.double().cpu(), bound.double().cpu()
    assert got.shape == want.shape
    same = (got == want) | (got.isnan() & want.isnan())
    off = ~(same | ((got - want).abs() <= bound))
    if off.any():
        i = int(off.flatten().nonzero()[0])
        raise AssertionError(f"{what}: {int(off.sum())} of {off.numel()} off, first at {np.unravel_index(i, off.shape)}: "
                             f"{got.flatten()[i].item()!r} for {want.flatten()[i].item()!r} within {bound.flatten()[i].item()!r}")


def embedding(table, tokens, alpha, beta, out):
    t = tokens.cpu().long()
    inside = (t >= 0) & (t < table.shape[0])
    rows = table.cpu().double()[torch.where(inside, t, 0)] if table.shape[0] else torch.zeros(len(t), table.shape[1], dtype=torch.float64)
    rows = torch.where(inside[:, None], rows, 0.0)
    return alpha * rows + (beta * out.cpu().double() if beta else 0.0)


def embedding_grad(grad, tokens, vocab, alpha, beta, old):
    """The gradient, and the sum of the absolute terms with their number."""
    t = tokens.cpu().long()
    inside = (t >= 0) & (t < vocab)
    g = grad.cpu().double()[inside]
    total = torch.zeros(vocab, grad.shape[1], dtype=torch.float64).index_add_(0, t[inside], g)
    size = torch.zeros(vocab, grad.shape[1], dtype=torch.float64).index_add_(0, t[inside], g.abs())
    many = torch.bincount(t[inside], minlength=vocab)[:, None]
    want = alpha * total + (beta * old.cpu().double() if beta else 0.0)
    return want, abs(alpha) * size + (abs(beta) * old.cpu().double().abs() if beta else 0.0), many


def route(x, bias, k, score="softmax", groups=1, kept=1, group_score="max", renormalise=True, scale=1.0):
    """Columns and weights, row by row, in numpy's 64 bits.  x: as the kernel reads it."""
    x = x.double().cpu().numpy()
    b = None if bias is None else bias.double().cpu().numpy()
    columns, weights = np.zeros((len(x), k), np.int32), np.zeros((len(x), k))
    for r, row in enumerate(x):
        row = np.where(np.isnan(row), -np.inf, row)
        live = row > -np.inf
        if score == "softmax":
            m = row.max(initial=-np.inf)
            p = np.zeros(len(row))
            with np.errstate(invalid="ignore"):
                p[live] = np.where(row[live] == m, 1.0, np.exp(row[live] - m))
            p = p / p.sum() if live.any() else p
        else:
            with np.errstate(over="ignore"):
                p = np.where(live, 1 / (1 + np.exp(-row)), 0.0)
        s = row.copy()
        if b is not None:
            s = np.where(live & (b > -np.inf), p + np.where(np.isnan(b), 0, b), -np.inf)
        if groups > 1:
            size = len(row) // groups
            inside = s if not (b is None and group_score == "top2") else np.where(live, p, -np.inf)
            best = []
            for g in range(groups):
                v = np.sort(inside[g * size:(g + 1) * size])[::-1]
                v = v[v > -np.inf][: 1 if group_score == "max" else 2]
                best.append(v.sum() if len(v) else -np.inf)
            order = sorted(range(groups), key=lambda g: (-best[g], g))
            for g in order[kept:]:
                s[g * size:(g + 1) * size] = -np.inf
        picked = sorted(sorted(range(len(row)), key=lambda e: (-s[e], e))[:k])
        w = np.array([p[e] if s[e] > -np.inf else 0.0 for e in picked])
        if renormalise:
            w = w / w.sum() if w.sum() > 0 else w * 0
        columns[r], weights[r] = picked, scale * w
    return torch.from_numpy(columns), torch.from_numpy(weights)


def route_weights(x, columns, score, renormalise, scale):
    """The weights of given columns, differentiable, 64 bits."""
    p = torch.softmax(x, 1) if score == "softmax" else torch.sigmoid(x)
    w = p.gather(1, columns.long())
    return scale * (w / w.sum(1, keepdim=True) if renormalise else w)


def rows_of(offsets, nnz):
    """The row of every entry."""
    return torch.searchsorted(offsets.cpu().long()[1:].contiguous(), torch.arange(nnz), right=True)


def experts_mm(offsets, columns, x, w, experts, transpose, by_entry, alpha, beta, y):
    """Y and the sum of the absolute terms; w: experts x n x d."""
    columns = columns.cpu().long()
    nnz = len(columns)
    row = torch.arange(nnz) if by_entry else rows_of(offsets, nnz)
    x, w = x.cpu().double(), w.cpu().double()
    out = torch.zeros(y.shape, dtype=torch.float64)
    size = torch.zeros_like(out)
    for e in range(experts):
        i = (columns == e).nonzero()[:, 0]
        m = w[e].T if transpose else w[e]
        out[i] = x[row[i]] @ m
        size[i] = x[row[i]].abs() @ m.abs()
    old = beta * y.cpu().double() if beta else torch.zeros_like(out)
    return alpha * out + old, abs(alpha) * size + old.abs()


def experts_grad(offsets, columns, dy, x, experts, by_entry, alpha, beta, dw):
    columns = columns.cpu().long()
    nnz = len(columns)
    row = torch.arange(nnz) if by_entry else rows_of(offsets, nnz)
    dy, x = dy.cpu().double(), x.cpu().double()
    out = torch.zeros(dw.shape, dtype=torch.float64)
    size, many = torch.zeros_like(out), torch.zeros(experts, 1, 1, dtype=torch.float64)
    for e in range(experts):
        i = (columns == e).nonzero()[:, 0]
        out[e] = dy[i].T @ x[row[i]]
        size[e] = dy[i].abs().T @ x[row[i]].abs()
        many[e] = len(i)
    old = beta * dw.cpu().double() if beta else torch.zeros_like(out)
    return alpha * out + old, abs(alpha) * size + old.abs(), many
