"""Plain implementations in 64 bits of the operators of include/b200sp_rows.h, for their tests."""
from __future__ import annotations

import torch

from token_reference import rows_of


def order_of(columns, experts):
    """The entries by expert (those of no expert last), every entry's place, and the first place of every expert with the end."""
    c = columns.cpu().long()
    c = torch.where((c >= 0) & (c < experts), c, experts)
    order = torch.sort(c, stable=True).indices
    places = torch.empty_like(order)
    places[order] = torch.arange(len(c))
    starts = torch.tensor([int((c < e).sum()) for e in range(experts + 1)], dtype=torch.int32)
    return order, places, starts


def dispatch(offsets, columns, x, experts, alpha, beta, s):
    order, _, starts = order_of(columns, experts)
    rows = x.cpu().double()[rows_of(offsets, len(order))[order]]
    rows[int(starts[-1]):] = 0
    return alpha * rows + (beta * s.cpu().double() if beta else 0.0), starts


def combine(offsets, columns, values, s, experts, alpha, beta, out):
    """The sums, those of the terms' absolute values, and the most terms of one.  values: None for no weights."""
    _, places, starts = order_of(columns, experts)
    token = rows_of(offsets, len(places))
    inside = places < int(starts[-1])
    w = torch.ones(len(places), dtype=torch.float64) if values is None else values.cpu().double()
    terms = (w[:, None] * s.cpu().double()[places])[inside]
    want = torch.zeros(out.shape, dtype=torch.float64).index_add_(0, token[inside], terms)
    size = torch.zeros(out.shape, dtype=torch.float64).index_add_(0, token[inside], terms.abs())
    old = beta * out.cpu().double() if beta else torch.zeros(out.shape, dtype=torch.float64)
    many = int(torch.bincount(token[inside]).max()) if inside.any() else 0
    return alpha * want + old, abs(alpha) * size + old.abs(), many


def combine_grad(offsets, columns, values, d_out, s, experts, alpha, beta, d_s, d_values):
    """dS, the values' gradient, and the sums of its terms' absolute values."""
    order, places, starts = order_of(columns, experts)
    token = rows_of(offsets, len(places))
    inside = places < int(starts[-1])
    g, w, s = d_out.cpu().double(), values.cpu().double(), s.cpu().double()
    rows = torch.where(inside[order][:, None], w[order][:, None] * g[token[order]], 0.0)
    terms = torch.where(inside[:, None], g[token] * s[places], 0.0)
    old = d_values.cpu().double() * beta if beta else torch.zeros(len(places), dtype=torch.float64)
    return (alpha * rows + (beta * d_s.cpu().double() if beta else 0.0), alpha * terms.sum(1) + old,
            abs(alpha) * terms.abs().sum(1) + old.abs())


def quantise(x):
    """Whole numbers and scales, by exact comparison: a value of 24 bits times 254 and an odd number times the largest are exact in 64."""
    x = x.cpu().double()
    size, top = x.abs(), x.abs().amax(1, keepdim=True)
    finite = torch.isfinite(top)
    safe = torch.where(finite & (top > 0), top, 1.0)
    q = torch.floor(127 * size / safe)
    over = 254 * size - (2 * q + 1) * safe
    q = q + ((over > 0) | ((over == 0) & (q % 2 == 1)))
    q = torch.where(finite & (top > 0), torch.sign(x) * q, 0.0).to(torch.int8)
    scale = torch.where(finite, (top.float() / 127).double(), torch.nan)[:, 0]
    return q, scale


def scaled(x, sx, w, sw, alpha, beta, y):
    """The product, and the sum of its two terms' absolute values."""
    sums = x.cpu().double() @ w.cpu().double().T
    want = alpha * (sums * sx.cpu().double()[:, None] * sw.cpu().double()[None])
    old = beta * y.cpu().double() if beta else torch.zeros(want.shape, dtype=torch.float64)
    return want + old, want.abs() + old.abs()
