"""GPU: rows in the order of the experts and back, rows in 8 bits and products of them (include/b200sp_rows.h) against plain
implementations in 64 bits (rows_reference.py), at the sizes, masks and layouts where they can go wrong."""
from __future__ import annotations

import math

import pytest
import torch

import rows_reference as rows
import token_reference as ref
from test_tokens_gpu import gen, mat, matrix, outside
from token_reference import DTYPE, F32

pytestmark = pytest.mark.gpu


def routed(api, g, tokens, experts, k, skew=0.5, wild=0.0, ragged=False, kind="f32"):
    """A routing: k different experts a token, or any number of any columns; `wild`: the share of columns that are no expert."""
    if ragged:
        lengths = torch.randint(0, 2 * k + 1, (tokens,), generator=g, device="cuda")
        lengths[tokens // 2] = min(40, experts * 3)  # more than a warp's, if there are experts enough
        offsets = torch.zeros(tokens + 1, dtype=torch.int32, device="cuda")
        offsets[1:] = lengths.cumsum(0)
        columns = torch.randint(0, experts, (int(offsets[-1]),), generator=g, device="cuda").to(torch.int32)
    else:
        offsets = torch.arange(0, tokens * k + 1, k, dtype=torch.int32, device="cuda")
        x = torch.randn((tokens, experts), generator=g, device="cuda") + skew * torch.randn(experts, generator=g, device="cuda")
        columns = x.topk(k, dim=1).indices.sort(dim=1).values.to(torch.int32).flatten()
    if wild:
        far = torch.tensor([-1, experts, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")
        columns = torch.where(torch.rand(len(columns), generator=g, device="cuda") < wild,
                              far[torch.randint(4, (len(columns),), generator=g, device="cuda")], columns)
    values = torch.randn(len(columns), generator=g, device="cuda").to(DTYPE[kind])
    return api.CsrMatrix(offsets, columns, values, tokens, experts)


def ordered(api, handle, R, size=None):
    buffer = torch.full((api.experts_order_buffer_size(handle, R) if size is None else size,), 255, dtype=torch.uint8, device="cuda")
    api.experts_preprocess(handle, R, buffer)
    return buffer


def no_error(pkg):
    assert pkg.lib().b200sp_experts_error() == 0 and pkg.lib().b200sp_scaled_error() == 0


ROWS = [  # tokens, experts, k, width, rows, other, alpha, beta, pad, shift, wild, ragged, weights
    (1, 1, 1, 1, "f32", "f32", 1.0, 0.0, 0, 0, 0.0, False, "f32"),
    (1, 64, 8, 4096, "bf16", "bf16", 1.0, 0.0, 0, 0, 0.0, False, "f32"),
    (3, 5, 5, 24, "f16", "f16", 0.5, 0.0, 0, 0, 0.4, False, "f16"),
    (37, 6, 2, 8, "bf16", "f32", 1.0, 1.0, 8, 0, 0.0, False, "bf16"),
    (61, 17, 3, 777, "f32", "f32", -1.5, 0.5, 0, 0, 0.1, True, "f32"),
    (200, 40, 4, 1030, "bf16", "bf16", 1.0, 0.0, 2, 0, 0.1, True, "f32"),  # rows that start on 16 bytes and end within a piece
    (200, 40, 4, 1030, "f16", "f32", 1.0, -0.5, 3, 1, 0.0, True, "f32"),
    (509, 1024, 1, 264, "f16", "f16", 2.0, 0.0, 0, 0, 1.0, False, "f32"),  # no entry has an expert
    (2500, 60, 6, 96, "f32", "f32", 1.0, 0.0, 4, 0, 0.05, False, "bf16"),  # more rows than CTAs have warps
    (2500, 33, 3, 520, "bf16", "bf16", 1.0, 1.0, 0, 0, 0.0, True, "f32"),
]
IDS = [f"{c[0]}x{c[3]}-{c[1]}-{c[2]}-{c[4]}-{c[5]}" for c in ROWS]


@pytest.mark.parametrize("tokens,experts,k,width,kind,other,alpha,beta,pad,shift,wild,ragged,weights", ROWS, ids=IDS)
def test_dispatch(pkg, handle, tokens, experts, k, width, kind, other, alpha, beta, pad, shift, wild, ragged, weights):
    from ops_sparse_b200 import api
    g = gen(tokens + width)
    R = routed(api, g, tokens, experts, k, 0.5, wild, ragged, weights)
    x, _ = matrix(g, tokens, width, kind, pad, shift)
    s, whole = matrix(g, R.nnz, width, other, pad, shift)
    want, starts = rows.dispatch(R.row_ptr, R.col_ind, x, experts, alpha, beta, s)
    size = want.abs() + (2 * abs(beta) * s.double().abs().cpu() if beta else 0)
    if beta == 0:
        s.fill_(math.nan)  # must not be read
    kept = outside(s, whole).clone()
    got = torch.full((experts + 1,), -7, dtype=torch.int32, device="cuda")
    api.experts_dispatch(handle, R, mat(api, x), mat(api, s), alpha, beta, offsets=api.DnVec(got), buffer=ordered(api, handle, R))
    no_error(pkg)
    assert torch.equal(got.cpu(), starts)
    ref.close(s, want, ref.rounding(s.dtype, want) + 2 * F32 * size)  # a product and a sum in f32, one rounding
    assert torch.equal(outside(s, whole), kept)


@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("tokens,experts,k,width,kind,other,alpha,beta,pad,shift,wild,ragged,weights", ROWS, ids=IDS)
def test_combine(pkg, handle, weighted, tokens, experts, k, width, kind, other, alpha, beta, pad, shift, wild, ragged, weights):
    from ops_sparse_b200 import api
    g = gen(tokens + width + 1)
    R = routed(api, g, tokens, experts, k, 0.5, wild, ragged, weights)
    s, _ = matrix(g, R.nnz, width, kind, pad, shift)
    out, whole = matrix(g, tokens, width, other, pad, shift)
    _, places, starts = rows.order_of(R.col_ind, experts)
    s[int(starts[-1]):] = math.nan  # rows of no expert take no part
    clean = s.clone()
    clean[int(starts[-1]):] = 0
    want, size, many = rows.combine(R.row_ptr, R.col_ind, R.values if weighted else None, clean, experts, alpha, beta, out)
    if beta == 0:
        out.fill_(math.nan)
    kept = outside(out, whole).clone()
    api.experts_combine(handle, R, mat(api, s), mat(api, out), alpha, beta, weighted=weighted, buffer=ordered(api, handle, R))
    no_error(pkg)
    # a sum of `many` products in f32, each added with one rounding; alpha, beta; one rounding
    ref.close(out, want, ref.rounding(out.dtype, want) + (many + 2) * F32 * size)
    assert torch.equal(outside(out, whole), kept)


@pytest.mark.parametrize("values", ["f32", "bf16", None])
@pytest.mark.parametrize("tokens,experts,k,width,kind,other,alpha,beta,pad,shift,wild,ragged,weights", ROWS, ids=IDS)
def test_combine_gradient(pkg, handle, values, tokens, experts, k, width, kind, other, alpha, beta, pad, shift, wild, ragged, weights):
    from ops_sparse_b200 import api
    g = gen(tokens + width + 2)
    R = routed(api, g, tokens, experts, k, 0.5, wild, ragged, weights)
    s, _ = matrix(g, R.nnz, width, kind, pad, shift)
    d_out, _ = matrix(g, tokens, width, other, pad, shift)
    d_s, whole = matrix(g, R.nnz, width, kind, pad, shift)
    d_values = torch.randn(R.nnz, generator=g, device="cuda").to(DTYPE[values or "f32"])
    _, _, starts = rows.order_of(R.col_ind, experts)
    want, want_v, size_v = rows.combine_grad(R.row_ptr, R.col_ind, R.values, d_out, s, experts, alpha, beta, d_s, d_values)
    s[int(starts[-1]):] = math.nan
    size = want.abs() + (2 * abs(beta) * d_s.double().abs().cpu() if beta else 0)
    if beta == 0:
        d_s.fill_(math.nan)
        d_values.fill_(math.nan)
    kept, old = outside(d_s, whole).clone(), d_values.clone()
    if values is None:
        api.experts_combine_grad(handle, R, mat(api, d_out), None, mat(api, d_s), None, alpha, beta, buffer=ordered(api, handle, R))
    else:
        api.experts_combine_grad(handle, R, mat(api, d_out), mat(api, s), mat(api, d_s), api.DnVec(d_values), alpha, beta,
                                 buffer=ordered(api, handle, R))
    no_error(pkg)
    ref.close(d_s, want, ref.rounding(d_s.dtype, want) + 3 * F32 * size)  # alpha w, times g, plus beta dS
    assert torch.equal(outside(d_s, whole), kept)
    if values is None:
        assert torch.equal(d_values.nan_to_num(), old.nan_to_num())
    else:
        ref.close(d_values, want_v, ref.rounding(d_values.dtype, want_v) + (width + 2) * F32 * size_v)


def test_combine_gradient_in_place_and_by_differences(pkg, handle):
    """dS in the place of S; and along a direction the weighted sum changes by what its gradient says."""
    from ops_sparse_b200 import api
    g = gen(5)
    R = routed(api, g, 50, 12, 3)
    s, d_out = matrix(g, R.nnz, 72, "f32")[0], matrix(g, 50, 72, "f32")[0]
    buffer = ordered(api, handle, R)

    def total(rows_, weights):
        out = torch.empty(50, 72, device="cuda")
        M = api.CsrMatrix(R.row_ptr, R.col_ind, weights, 50, 12)
        api.experts_combine(handle, M, mat(api, rows_), mat(api, out), buffer=ordered(api, handle, M))
        torch.cuda.synchronize()
        return float((out.double() * d_out.double()).sum())

    d_s, d_values = torch.empty_like(s), torch.empty(R.nnz, device="cuda")
    api.experts_combine_grad(handle, R, mat(api, d_out), mat(api, s), mat(api, d_s), api.DnVec(d_values), buffer=buffer)
    way_s, way_v = torch.randn(s.shape, generator=g, device="cuda"), torch.randn(R.nnz, generator=g, device="cuda")
    # the sum is linear in either, so that a difference of any length has no error of its own: what is left are f32 sums of 50 * 72 * 3 terms
    size = float((R.values.double().abs().sum() + 1) * s.double().abs().max() * d_out.double().abs().max() * 72)
    for step in (1.0, 0.25):
        by_s = (total(s + step * way_s, R.values) - total(s - step * way_s, R.values)) / (2 * step)
        by_v = (total(s, R.values + step * way_v) - total(s, R.values - step * way_v)) / (2 * step)
        assert abs(by_s - float((d_s.double() * way_s.double()).sum())) <= 16 * F32 * size / step * 4
        assert abs(by_v - float((d_values.double() * way_v.double()).sum())) <= 16 * F32 * size / step * 4
    in_place, again = s.clone(), torch.empty(R.nnz, device="cuda")
    api.experts_combine_grad(handle, R, mat(api, d_out), mat(api, in_place), mat(api, in_place), api.DnVec(again), buffer=buffer)
    torch.cuda.synchronize()
    assert torch.equal(in_place, d_s) and torch.equal(again, d_values)


QUANTISE = [  # rows, width, kind, pad, shift, pad of Q
    (1, 1, "f32", 0, 0, 0), (1, 4096, "bf16", 0, 0, 0), (5, 24, "f16", 0, 0, 8), (37, 777, "f32", 0, 0, 7), (2049, 130, "bf16", 6, 0, 6),
    (1300, 1030, "f16", 2, 0, 2), (1300, 2048, "bf16", 0, 0, 0), (1200, 2056, "bf16", 0, 0, 0), (3, 9000, "f32", 0, 0, 0),
    (3, 20001, "bf16", 3, 1, 3), (1250, 1032, "f32", 0, 0, 0),
]


@pytest.mark.parametrize("many,width,kind,pad,shift,padded", QUANTISE)
def test_quantise_rows(pkg, handle, many, width, kind, pad, shift, padded):
    from ops_sparse_b200 import api
    g = gen(many + width)
    x, _ = matrix(g, many, width, kind, pad, shift)
    x[many // 2] *= 1e-4
    want, want_s = rows.quantise(x)
    whole = torch.full((many, width + padded), 99, dtype=torch.int8, device="cuda")
    scales = torch.empty(many, device="cuda")
    api.quantise_rows(handle, mat(api, x), api.DnMat(whole, many, width, width + padded), api.DnVec(scales))
    torch.cuda.synchronize()
    assert torch.equal(whole[:, :width].cpu(), want) and bool((whole[:, width:] == 99).all())
    assert torch.equal(scales.double().cpu(), want_s)


def test_quantise_borders_and_special_values(pkg, handle):
    """Halves, exactly and one step of f32 beside; rows of zeros, of subnormals, of the largest values, and some that are not finite."""
    from ops_sparse_b200 import api
    tops = torch.tensor([127.0, 1.0, 3.0, 254.0, 0.1, 1e-30, 2.0 ** -126, 2.0 ** -140, 1e30, 3.4028234e38, 88.5, 7e-45], device="cuda")
    halves = torch.arange(-126.5, 127, 1.0, device="cuda", dtype=torch.float64)
    x = torch.zeros(len(tops), 1 + 3 * len(halves), device="cuda")
    x[:, 0] = tops
    border = (halves[None] * tops.double()[:, None] / 127).float()
    x[:, 1::3], x[:, 2::3], x[:, 3::3] = border, border.nextafter(torch.full_like(border, math.inf)), border.nextafter(-torch.full_like(border, math.inf))
    x = torch.minimum(torch.maximum(x, -tops[:, None]), tops[:, None]).contiguous()
    want, want_s = rows.quantise(x)
    q, scales = torch.empty(x.shape, dtype=torch.int8, device="cuda"), torch.empty(len(tops), device="cuda")
    api.quantise_rows(handle, mat(api, x), api.DnMat(q, *x.shape, x.shape[1]), api.DnVec(scales))
    torch.cuda.synchronize()
    assert torch.equal(q.cpu(), want) and torch.equal(scales.double().cpu(), want_s)
    for kind in (torch.float16, torch.bfloat16, torch.float32):
        bad = torch.ones(6, 40, device="cuda", dtype=kind)
        bad[0], bad[1, 3], bad[2, 39], bad[3, 0], bad[4] = 0, math.inf, math.nan, -math.inf, -0.0
        q, scales = torch.full((6, 40), 5, dtype=torch.int8, device="cuda"), torch.empty(6, device="cuda")
        api.quantise_rows(handle, mat(api, bad), api.DnMat(q, 6, 40, 40), api.DnVec(scales))
        torch.cuda.synchronize()
        assert bool((q[:5] == 0).all()) and bool((q[5] == 127).all())
        assert scales[[0, 4]].tolist() == [0.0, 0.0] and bool(scales[1:4].isnan().all()) and scales[5].item() == float(torch.tensor(1.0) / 127)


@pytest.mark.parametrize("tokens,experts,k,width,kind,pad,shift,wild,ragged", [
    (1, 64, 8, 2048, "bf16", 0, 0, 0.0, False), (40, 6, 2, 72, "f16", 0, 0, 0.3, True), (509, 17, 3, 777, "f32", 0, 0, 0.1, False),
    (1300, 60, 6, 520, "bf16", 8, 0, 0.05, True), (1300, 9, 2, 2600, "f32", 1, 1, 0.0, False),
])
def test_experts_quantise(pkg, handle, tokens, experts, k, width, kind, pad, shift, wild, ragged):
    from ops_sparse_b200 import api
    g = gen(tokens + width + 3)
    R = routed(api, g, tokens, experts, k, 0.5, wild, ragged)
    x, _ = matrix(g, tokens, width, kind, pad, shift)
    order, _, starts = rows.order_of(R.col_ind, experts)
    want, want_s = rows.quantise(x)
    token = ref.rows_of(R.row_ptr, R.nnz)[order]
    want, want_s = want[token], want_s[token]
    want[int(starts[-1]):], want_s[int(starts[-1]):] = 0, 0
    q, scales = torch.full((R.nnz, width), 99, dtype=torch.int8, device="cuda"), torch.empty(R.nnz, device="cuda")
    got = torch.empty(experts + 1, dtype=torch.int32, device="cuda")
    api.experts_quantise(handle, R, mat(api, x), mat(api, q), api.DnVec(scales), offsets=api.DnVec(got), buffer=ordered(api, handle, R))
    no_error(pkg)
    assert torch.equal(q.cpu(), want) and torch.equal(scales.double().cpu(), want_s) and torch.equal(got.cpu(), starts)


def eights(g, many, width, pad=0, shift=0):
    """Rows of 8 bits, among them the lowest value, a view in larger memory."""
    whole = torch.randint(-128, 128, (many * (width + pad) + shift,), generator=g, device="cuda", dtype=torch.int8)
    return whole[shift:].view(many, width + pad)[:, :width]


SCALED = [  # rows, depth, channels, out, alpha, beta, pad and shift of the operands, pad and shift of Y
    (1, 1, 1, "f32", 1.0, 0.0, 15, 0, 0, 0),
    (1, 4096, 4096, "bf16", 1.0, 0.0, 0, 0, 0, 0),
    (1, 4096, 100, "f16", 1e-3, 0.0, 0, 0, 0, 0),
    (2, 64, 129, "bf16", 0.5, 1.0, 0, 0, 7, 0),
    (7, 100, 40, "f32", 1.0, 0.0, 0, 0, 0, 0),  # rows of four bytes off sixteen
    (16, 2048, 640, "bf16", 1.0, 0.0, 0, 0, 0, 0),
    (17, 777, 333, "f32", 2.0, -0.5, 1, 3, 1, 1),
    (33, 160, 130, "f16", 1e-3, 0.0, 0, 0, 6, 0),  # rows of Y on 16 bytes, the last channels are no whole piece
    (61, 2040, 1111, "f32", 1.0, 0.0, 8, 0, 0, 0),
    (100, 128, 128, "bf16", 1.0, 0.0, 0, 0, 0, 0),
    (130, 1000, 257, "bf16", 1.0, 1.0, 8, 0, 7, 0),
    (256, 1024, 256, "f16", 1e-4, 0.0, 0, 0, 0, 0),
    (257, 96, 1000, "bf16", 1.0, 0.0, 0, 0, 0, 0),
    (600, 272, 300, "f32", 1.0, 0.0, 0, 0, 0, 0),
    (1025, 640, 513, "bf16", 1.0, 0.5, 0, 0, 3, 3),
    (2000, 513, 2100, "bf16", 1.0, 0.0, 15, 0, 4, 0),
    (5, 131071, 20, "f32", 1.0, 0.0, 1, 0, 0, 0),
]


@pytest.mark.parametrize("many,depth,channels,out,alpha,beta,pad,shift,pad_y,shift_y", SCALED)
def test_scaled_product(pkg, handle, many, depth, channels, out, alpha, beta, pad, shift, pad_y, shift_y):
    from ops_sparse_b200 import api
    g = gen(many + depth + channels)
    x, w = eights(g, many, depth, pad, shift), eights(g, channels, depth, pad, shift)
    sx, sw = torch.rand(many, generator=g, device="cuda") * 1e-2, torch.rand(channels, generator=g, device="cuda") * 1e-3
    if many > 3:
        sx[2] = 0.0
    y, whole = matrix(g, many, channels, out, pad_y, shift_y)
    want, size = rows.scaled(x, sx, w, sw, alpha, beta, y)
    if beta == 0:
        y.fill_(math.nan)
    kept = outside(y, whole).clone()
    X, W, Y = mat(api, x), mat(api, w), mat(api, y)
    room = api.scaled_mm_buffer_size(handle, X, W, Y)
    buffer = torch.full((room,), 255, dtype=torch.uint8, device="cuda") if room else None
    assert (room == 0) == all(t.data_ptr() % 16 == 0 and t.stride(0) % 16 == 0 for t in (x, w))
    api.scaled_mm(handle, X, api.DnVec(sx), W, api.DnVec(sw), Y, alpha, beta, buffer=buffer)
    no_error(pkg)
    # the sum is exact; its f32, the scales' product, theirs, alpha's and beta's are rounded, then the result
    ref.close(y, want, ref.rounding(y.dtype, want) + 5 * F32 * size)
    assert torch.equal(outside(y, whole), kept)


@pytest.mark.parametrize("many,depth,channels", [(2, 512, 200), (40, 512, 200), (40, 128, 30000), (320, 512, 200)],
                         ids=["rows", "clusters", "whole", "pairs"])
def test_scaled_extreme_scales(pkg, handle, many, depth, channels):
    """Scales whose product f32 cannot hold, of sums that bring the result back, and some that are not finite, in every way of the product."""
    from ops_sparse_b200 import api
    g = gen(77)
    x, w = eights(g, many, depth), eights(g, channels, depth)
    x[:, 0] = 127
    sx = torch.tensor([1e-30, 1e25, 1e-25, 1e38, 1.0, 0.0, 1e-38, 1e-45], device="cuda").repeat(many // 8 + 1)[:many].contiguous()
    sw = torch.tensor([1e-20, 1e-10, 1.0, 1e10, 1e-25, 1e-38, 3e38, 0.0], device="cuda").repeat(channels // 8)
    for alpha in (1.0, 1e15, 1e-15):
        y = torch.empty(many, channels, device="cuda")
        api.scaled_mm(handle, mat(api, x), api.DnVec(sx), mat(api, w), api.DnVec(sw), mat(api, y), alpha=alpha)
        torch.cuda.synchronize()
        want, _ = rows.scaled(x, sx, w, sw, float(torch.tensor(alpha)), 0.0, y)
        held = want.float().double()  # infinite where f32 is
        ref.close(y, torch.where(want.abs() > 3.4028235e38, held, want), ref.rounding(y.dtype, want) + 5 * F32 * want.abs())
    sx = torch.ones(many, device="cuda")
    sx[0], sx[1] = math.nan, math.inf
    y = torch.empty(many, channels, dtype=torch.float16, device="cuda")
    api.scaled_mm(handle, mat(api, x), api.DnVec(sx), mat(api, w), api.DnVec(torch.full((channels,), 1e-3, device="cuda")), mat(api, y))
    no_error(pkg)
    assert bool(y[0].isnan().all()) and bool((~y[1].isfinite()).all()) and not bool(y[2:].isnan().any())


EXPERTS = [  # tokens, experts, k, depth, channels, out, alpha, beta, pad, wild, ragged
    (1, 4, 2, 64, 40, "bf16", 1.0, 0.0, 0, 0.0, False),
    (16, 64, 8, 256, 160, "bf16", 1.0, 0.0, 0, 0.0, False),
    (40, 6, 2, 100, 24, "f32", 1.0, 0.0, 0, 0.2, True),
    (61, 17, 3, 777, 130, "f16", 1e-3, 0.0, 7, 0.1, True),
    (300, 5, 2, 272, 300, "bf16", 0.5, 1.0, 0, 0.1, False),
    (900, 4, 2, 384, 513, "bf16", 1.0, 0.0, 0, 0.0, False),
    (700, 1024, 2, 48, 9, "f32", 1.0, -1.0, 0, 0.05, True),
    (50, 3, 1, 64, 70, "f32", 1.0, 0.0, 0, 1.0, False),  # no entry has an expert
    (1500, 2, 1, 640, 264, "f32", 1.0, 0.0, 0, 0.0, False),
    (1, 64, 8, 2048, 130, "bf16", 1.0, 0.0, 0, 0.0, False),  # hardly an expert with more than one entry: no tiles
    (1, 100, 9, 777, 33, "f32", 2.0, 0.5, 7, 0.3, False),
    (8, 1024, 24, 520, 31, "f16", 1e-3, 0.0, 0, 0.1, True),
]


@pytest.mark.parametrize("tokens,experts,k,depth,channels,out,alpha,beta,pad,wild,ragged", EXPERTS)
def test_experts_scaled_product(pkg, handle, tokens, experts, k, depth, channels, out, alpha, beta, pad, wild, ragged):
    from ops_sparse_b200 import api
    g = gen(tokens + depth + channels)
    R = routed(api, g, tokens, experts, k, 1.0, wild, ragged)
    x, w = eights(g, R.nnz, depth, pad), eights(g, experts * channels, depth, pad)
    sx, sw = torch.rand(R.nnz, generator=g, device="cuda") * 1e-2, torch.rand(experts * channels, generator=g, device="cuda") * 1e-3
    y, whole = matrix(g, R.nnz, channels, out, 0, 0)
    _, _, starts = rows.order_of(R.col_ind, experts)
    end = int(starts[-1])
    sx[end:] = math.nan  # rows of no expert are not looked at
    want = beta * y.double().cpu() if beta else torch.zeros(y.shape, dtype=torch.float64)
    size = want.abs()
    for e in range(experts):
        a, b, c = int(starts[e]), int(starts[e + 1]), slice(e * channels, (e + 1) * channels)
        want[a:b], size[a:b] = rows.scaled(x[a:b], sx[a:b], w[c], sw[c], alpha, beta, y[a:b])
    if beta == 0:
        y.fill_(math.nan)
    X, W, Y = mat(api, x), mat(api, w), mat(api, y)
    buffer = ordered(api, handle, R, api.experts_scaled_mm_buffer_size(handle, R, X, W, Y))
    api.experts_scaled_mm(handle, R, X, api.DnVec(sx), W, api.DnVec(sw), Y, alpha, beta, buffer=buffer)
    no_error(pkg)
    ref.close(y, want, ref.rounding(y.dtype, want) + 5 * F32 * size)


# ---------------------------------------------------------------- used together, on streams and in graphs

def test_layer_in_eight_bits(pkg, handle):
    """Routing, rows to 8 bits in the order of the experts, two products with the experts' matrices, the weighted sum: one run."""
    from ops_sparse_b200 import api
    g = gen(11)
    tokens, experts, k, d, n = 70, 12, 3, 144, 200
    logits, x = torch.randn(tokens, experts, generator=g, device="cuda"), matrix(g, tokens, d, "bf16")[0]
    R = api.CsrMatrix(torch.empty(tokens + 1, dtype=torch.int32, device="cuda"), torch.empty(tokens * k, dtype=torch.int32, device="cuda"),
                      torch.empty(tokens * k, device="cuda"), tokens, experts)
    weights = [torch.randn(experts * rows_, cols, generator=g, device="cuda") for rows_, cols in ((n, d), (d, n))]
    held, scales = [], []
    for w in weights:
        held.append(torch.empty(w.shape, dtype=torch.int8, device="cuda"))
        scales.append(torch.empty(len(w), device="cuda"))
        api.quantise_rows(handle, mat(api, w), mat(api, held[-1]), api.DnVec(scales[-1]))
    q, p = (torch.empty(tokens * k, c, dtype=torch.int8, device="cuda") for c in (d, n))
    sq, sp = torch.empty(tokens * k, device="cuda"), torch.empty(tokens * k, device="cuda")
    y, z, out = torch.empty(tokens * k, n, device="cuda"), torch.empty(tokens * k, d, device="cuda"), torch.empty_like(x)
    Q, P, Y, Z = mat(api, q), mat(api, p), mat(api, y), mat(api, z)
    W = [mat(api, w) for w in held]
    size = max(api.experts_scaled_mm_buffer_size(handle, R, Q, W[0], Y), api.experts_scaled_mm_buffer_size(handle, R, P, W[1], Z))
    buffer = torch.empty(size, dtype=torch.uint8, device="cuda")
    api.route(handle, api.RouteRule(), mat(api, logits), None, R)
    api.experts_preprocess(handle, R, buffer)
    api.experts_quantise(handle, R, mat(api, x), Q, api.DnVec(sq), buffer=buffer)
    api.experts_scaled_mm(handle, R, Q, api.DnVec(sq), W[0], api.DnVec(scales[0]), Y, buffer=buffer)
    torch.nn.functional.silu(y, inplace=True)
    api.quantise_rows(handle, Y, P, api.DnVec(sp))
    api.experts_scaled_mm(handle, R, P, api.DnVec(sp), W[1], api.DnVec(scales[1]), Z, buffer=buffer)
    api.experts_combine(handle, R, Z, mat(api, out), buffer=buffer)
    no_error(pkg)
    # step by step in 64 bits, every step from what the one before left
    order, places, starts = rows.order_of(R.col_ind, experts)
    token = ref.rows_of(R.row_ptr, tokens * k)[order]
    want_q, want_s = rows.quantise(x)
    assert torch.equal(q.cpu(), want_q[token]) and torch.equal(sq.double().cpu(), want_s[token])
    want_p, want_sp = rows.quantise(y)
    assert torch.equal(p.cpu(), want_p) and torch.equal(sp.double().cpu(), want_sp)
    for e in range(experts):
        a, b = int(starts[e]), int(starts[e + 1])
        want, many = rows.scaled(p[a:b], sp[a:b], held[1][e * d:(e + 1) * d], scales[1][e * d:(e + 1) * d], 1.0, 0.0, z[a:b])
        ref.close(z[a:b], want, 5 * F32 * many)
    want, many, _ = rows.combine(R.row_ptr, R.col_ind, R.values, z, experts, 1.0, 0.0, out)
    ref.close(out, want, ref.rounding(out.dtype, want) + 5 * F32 * many)


def test_dispatch_combine_gradients_of_a_layer(pkg, handle):
    """Dispatch, a product of every expert, combine, and back: against 64 bits' automatic differentiation."""
    from ops_sparse_b200 import api
    g = gen(12)
    tokens, experts, k, d = 45, 7, 2, 40
    R = routed(api, g, tokens, experts, k)
    x, w, d_out = torch.randn(tokens, d, generator=g, device="cuda"), torch.randn(experts, d, d, generator=g, device="cuda"), torch.randn(tokens, d, generator=g, device="cuda")
    buffer, starts = ordered(api, handle, R), torch.empty(experts + 1, dtype=torch.int32, device="cuda")
    new = lambda rows_: torch.empty(rows_, d, device="cuda")  # noqa: E731
    s, z, out, d_z, d_x, d_values = new(R.nnz), new(R.nnz), new(tokens), new(R.nnz), new(tokens), torch.empty(R.nnz, device="cuda")
    api.experts_dispatch(handle, R, mat(api, x), mat(api, s), offsets=api.DnVec(starts), buffer=buffer)
    at = starts.tolist()
    for e in range(experts):
        z[at[e]:at[e + 1]] = (s[at[e]:at[e + 1]].double() @ w[e].double()).float()
    api.experts_combine(handle, R, mat(api, z), mat(api, out), buffer=buffer)
    api.experts_combine_grad(handle, R, mat(api, d_out), mat(api, z), mat(api, d_z), api.DnVec(d_values), buffer=buffer)
    d_s = torch.cat([(d_z[at[e]:at[e + 1]].double() @ w[e].double().T).float() for e in range(experts)])
    api.experts_combine(handle, R, mat(api, d_s), mat(api, d_x), weighted=False, buffer=buffer)
    no_error(pkg)
    leaf, values = x.double().requires_grad_(), R.values.double().requires_grad_()
    token = torch.arange(tokens, device="cuda").repeat_interleave(k)
    terms = values[:, None] * torch.einsum("ih,ihf->if", leaf[token], w.double()[R.col_ind.long()])
    total = torch.zeros(tokens, d, dtype=torch.float64, device="cuda").index_add(0, token, terms)
    gx, gv = torch.autograd.grad((total * d_out.double()).sum(), (leaf, values))
    # sums of d products, whose terms are f32 roundings of sums of k (or d) terms: all of them within 6 d of 2^-24 of the largest sizes
    total, gx, gv = total.detach(), gx.detach(), gv.detach()
    size = float(d_out.abs().max()) * float(w.abs().max()) * d * max(1.0, float(R.values.abs().max()))
    assert float((out.double() - total).abs().max()) <= 6 * F32 * k * size * float(x.abs().max())
    assert float((d_x.double() - gx).abs().max()) <= 6 * F32 * d * size
    assert float((d_values.double() - gv).abs().max()) <= 6 * F32 * d * d * size * float(x.abs().max())


def small(api, handle, g, tokens=40, experts=6, k=2, n=48, d=64, h=None):
    """A routing with everything that the calls take, and all of them as functions of a handle."""
    R = routed(api, g, tokens, experts, k)
    x, s = matrix(g, tokens, d, "f32")[0], matrix(g, R.nnz, d, "f32")[0]
    w, sw = eights(g, experts * n, d), torch.rand(experts * n, generator=g, device="cuda")
    made = {"S": torch.zeros(R.nnz, d, device="cuda"), "out": torch.zeros(tokens, d, device="cuda"), "dS": torch.zeros(R.nnz, d, device="cuda"),
            "dv": torch.zeros(R.nnz, device="cuda"), "q": torch.zeros(R.nnz, d, dtype=torch.int8, device="cuda"),
            "sq": torch.zeros(R.nnz, device="cuda"), "y": torch.zeros(R.nnz, n, device="cuda"),
            "starts": torch.zeros(experts + 1, dtype=torch.int32, device="cuda")}
    q, W = mat(api, made["q"]), mat(api, w)
    vec = {name: api.DnVec(made[name]) for name in ("dv", "sq", "starts")}
    m = {name: mat(api, made[name]) for name in ("S", "out", "dS", "y")}
    X, S, SW = mat(api, x), mat(api, s), api.DnVec(sw)
    buffer = torch.zeros(api.experts_scaled_mm_buffer_size(handle, R, q, W, m["y"]), dtype=torch.uint8, device="cuda")

    def run(h):
        api.experts_dispatch(h, R, X, m["S"], offsets=vec["starts"], buffer=buffer)
        api.experts_combine(h, R, S, m["out"], buffer=buffer)
        api.experts_combine_grad(h, R, X, S, m["dS"], vec["dv"], buffer=buffer)
        api.experts_quantise(h, R, X, q, vec["sq"], buffer=buffer)
        api.experts_scaled_mm(h, R, q, vec["sq"], W, SW, m["y"], buffer=buffer)

    def check():
        order, places, starts = rows.order_of(R.col_ind, experts)
        token = ref.rows_of(R.row_ptr, R.nnz)
        assert torch.equal(made["starts"].cpu(), starts) and torch.equal(made["S"].cpu(), x.cpu()[token[order]])
        want, size, many = rows.combine(R.row_ptr, R.col_ind, R.values, s, experts, 1.0, 0.0, made["out"])
        ref.close(made["out"], want, (many + 2) * F32 * size)
        want, want_v, size_v = rows.combine_grad(R.row_ptr, R.col_ind, R.values, x, s, experts, 1.0, 0.0, made["dS"], made["dv"])
        ref.close(made["dS"], want, 3 * F32 * want.abs())
        ref.close(made["dv"], want_v, (d + 2) * F32 * size_v)
        want_q, want_s = rows.quantise(x)
        assert torch.equal(made["q"].cpu(), want_q[token[order]])
        for e in range(experts):
            a, b, c = int(starts[e]), int(starts[e + 1]), slice(e * n, (e + 1) * n)
            want, size = rows.scaled(made["q"][a:b], want_s[token[order]][a:b], w[c], sw[c], 1.0, 0.0, made["y"][a:b])
            ref.close(made["y"][a:b], want, 5 * F32 * size)

    return R, buffer, made, run, check, (X, S, W, SW, q)


def test_captured_and_replayed_on_other_routings(pkg, handle):
    """A graph of the order and all that follows it, replayed on new columns, on a stream of its own."""
    from ops_sparse_b200 import api
    g = gen(21)
    stream = torch.cuda.Stream()
    h = api.Handle(stream)
    R, buffer, made, run, check, keep = small(api, h, g)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        api.experts_preprocess(h, R, buffer)
        run(h)
    for seed in (1, 2):
        fresh = gen(seed)
        other = torch.randn((40, 6), generator=fresh, device="cuda").topk(2, dim=1).indices.sort(dim=1).values
        R.col_ind.copy_(other.to(torch.int32).flatten())
        R.values.copy_(torch.randn(80, generator=fresh, device="cuda"))
        torch.cuda.synchronize()
        graph.replay()
        no_error(pkg)
        check()
    h.close()
    assert keep


def test_order_that_has_not_been_made(pkg, handle):
    """A captured Preprocess that has not been replayed has left no order: calls after it touch nothing and say so; replayed, they run."""
    from ops_sparse_b200 import api
    L = pkg.lib()
    stream = torch.cuda.Stream()
    h = api.Handle(stream)
    R, buffer, made, run, check, keep = small(api, h, gen(22))
    X, S, W, SW, q = keep
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        api.experts_preprocess(h, R, buffer)
    L.b200sp_experts_error_clear()
    L.b200sp_scaled_error_clear()
    m = {name: mat(api, made[name]) for name in ("S", "out", "dS", "y")}
    dv, sq = api.DnVec(made["dv"]), api.DnVec(made["sq"])
    calls = [lambda: api.experts_dispatch(h, R, X, m["S"], buffer=buffer), lambda: api.experts_combine(h, R, S, m["out"], buffer=buffer),
             lambda: api.experts_combine_grad(h, R, X, S, m["dS"], dv, buffer=buffer),
             lambda: api.experts_quantise(h, R, X, q, sq, buffer=buffer)]
    for call in calls:
        call()
        assert L.b200sp_experts_error() == 2
        L.b200sp_experts_error_clear()
    api.experts_scaled_mm(h, R, q, sq, W, SW, m["y"], buffer=buffer)
    assert L.b200sp_scaled_error() == 2 and L.b200sp_experts_error() == 0
    L.b200sp_scaled_error_clear()
    assert all(not bool(t.any()) for t in made.values())
    graph.replay()
    torch.cuda.synchronize()
    run(h)
    no_error(pkg)
    check()
    h.close()


def test_stale_order_is_refused(pkg, handle):
    from ops_sparse_b200 import api
    g = gen(23)
    R, buffer, made, run, check, keep = small(api, handle, g)
    bad = pkg.ACL_SPARSE_STATUS_INVALID_VALUE

    def refused(call):
        with pytest.raises(pkg.AclSparseError) as e:
            call()
        assert e.value.status == bad

    refused(lambda: run(handle))  # never ordered
    api.experts_preprocess(handle, R, buffer)
    run(handle)
    check()
    api.route(handle, api.RouteRule(), api.DnMat.row_major(torch.randn(40, 6, generator=g, device="cuda")), None, R)
    refused(lambda: run(handle))  # the routing has changed
    api.experts_preprocess(handle, R, buffer)
    run(handle)
    no_error(pkg)
    check()
    # a copy for a product without experts is written into the buffer: the order is gone
    x, w = eights(g, 20, 40, 1), eights(g, 30, 40)
    y = torch.empty(20, 30, device="cuda")
    one = torch.ones(30, device="cuda")
    api.scaled_mm(handle, mat(api, x), api.DnVec(one[:20]), mat(api, w), api.DnVec(one), mat(api, y), buffer=buffer)
    refused(lambda: run(handle))
    want, size = rows.scaled(x, one[:20], w, one, 1.0, 0.0, y)
    ref.close(y, want, 5 * F32 * size)


def test_scalars_on_the_device(pkg, handle):
    from ops_sparse_b200 import api
    g = gen(24)
    R, buffer, made, run, check, (X, S, W, SW, q) = small(api, handle, g)
    api.experts_preprocess(handle, R, buffer)
    run(handle)
    alpha, beta = torch.tensor([0.5], device="cuda"), torch.tensor([-2.0], device="cuda")
    before = {name: t.clone() for name, t in made.items()}
    m = {name: mat(api, made[name]) for name in ("S", "out", "dS", "y")}
    dv, sq = api.DnVec(made["dv"]), api.DnVec(made["sq"])
    h = api.Handle()
    h.set_pointer_mode_device(True)
    api.experts_dispatch(h, R, X, m["S"], alpha, beta, buffer=buffer)
    api.experts_combine(h, R, S, m["out"], alpha, beta, buffer=buffer)
    api.experts_combine_grad(h, R, X, S, m["dS"], dv, alpha, beta, buffer=buffer)
    api.experts_scaled_mm(h, R, q, sq, W, SW, m["y"], alpha, beta, buffer=buffer)
    few = torch.ones(2, 48, device="cuda")
    api.scaled_mm(h, api.DnMat(q.values[:2], 2, 64, 64), api.DnVec(made["sq"][:2]), api.DnMat(W.values[:48], 48, 64, 64), api.DnVec(SW.values[:48]),
                  mat(api, few), alpha, beta)
    no_error(pkg)
    for name in ("S", "out", "dS", "dv", "y"):  # 0.5 t - 2 t, from sums that are the same bits
        want = -1.5 * before[name].double()
        ref.close(made[name], want, 3 * F32 * 2.5 * want.abs())
    want, size = rows.scaled(q.values[:2], made["sq"][:2], W.values[:48], SW.values[:48], 0.5, -2.0, torch.ones(2, 48))
    ref.close(few, want, 5 * F32 * size)
    h.close()


def test_same_bits_in_every_run(pkg, handle):
    from ops_sparse_b200 import api
    g = gen(25)
    R, buffer, made, run, check, keep = small(api, handle, g, tokens=1500, experts=9, k=3, n=130, d=264)
    api.experts_preprocess(handle, R, buffer)
    run(handle)
    torch.cuda.synchronize()
    first = {name: t.clone() for name, t in made.items()}
    for _ in range(3):
        run(handle)
        torch.cuda.synchronize()
        assert all(torch.equal(first[name], t) for name, t in made.items())
    assert keep


@pytest.mark.parametrize("many,depth,channels", [(300, 2048, 600), (40, 2048, 300), (40, 512, 20000)], ids=["pairs", "clusters", "whole"])
def test_scaled_wait_that_runs_out(pkg, handle, many, depth, channels):
    """Every wait for a copy runs out (bytes are expected that nobody sends): the flag says so, Y is as it was, and the next product is right."""
    from ops_sparse_b200 import api
    L, g = pkg.lib(), gen(26)
    x, w = eights(g, many, depth), eights(g, channels, depth)
    sx, sw = torch.rand(many, generator=g, device="cuda"), torch.rand(channels, generator=g, device="cuda")
    y = torch.full((many, channels), 3.0, dtype=torch.bfloat16, device="cuda")
    args = (mat(api, x), api.DnVec(sx), mat(api, w), api.DnVec(sw), mat(api, y))
    L.b200sp_scaled_wait_test(200_000, 16)
    try:
        api.scaled_mm(handle, *args)
        asked = L.b200sp_scaled_error()
        left = bool((y == 3.0).all())
    finally:
        L.b200sp_scaled_wait_test(0, 0)
        L.b200sp_scaled_error_clear()
    assert asked == 1 and left
    api.scaled_mm(handle, *args)
    no_error(pkg)
    want, size = rows.scaled(x, sx, w, sw, 1.0, 0.0, y)
    ref.close(y, want, ref.rounding(y.dtype, want) + 5 * F32 * size)


def test_rows_beyond_32_bits(pkg, handle):
    """Rows that lie more than 2^32 bytes (and 2^31 elements) apart."""
    from ops_sparse_b200 import api
    g = gen(27)
    far, width = 2 ** 30 + 16, 40
    R = api.CsrMatrix(torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda"), torch.tensor([0, 2, 1, 2], dtype=torch.int32, device="cuda"),
                      torch.tensor([1.0, -2.0, 0.5, 3.0], device="cuda"), 2, 3)
    buffer = ordered(api, handle, R)
    s = torch.zeros(3 * far + width, dtype=torch.bfloat16, device="cuda")
    view = s.as_strided((4, width), (far, 1))
    x = torch.randn(2, width, generator=g, device="cuda").bfloat16()
    S = api.DnMat(s, 4, width, far)
    api.experts_dispatch(handle, R, mat(api, x), S, buffer=buffer)
    torch.cuda.synchronize()
    assert torch.equal(view.cpu(), x.cpu()[[0, 1, 0, 1]])
    out = torch.empty(2, width, device="cuda")
    api.experts_combine(handle, R, S, mat(api, out), buffer=buffer)
    torch.cuda.synchronize()
    ref.close(out, torch.stack([-1.0 * x[0].double(), 3.5 * x[1].double()]), 4 * F32 * 4 * x.double().abs())
    d_values = torch.empty(4, device="cuda")
    api.experts_combine_grad(handle, R, mat(api, x), S, S, api.DnVec(d_values), buffer=buffer)
    torch.cuda.synchronize()
    ref.close(view, torch.stack([x[0], 0.5 * x[1], -2.0 * x[0], 3.0 * x[1]]).double(), 0.01 * torch.ones(4, width))
    del view, S, s
    far = 2 ** 31 - 16
    q = torch.zeros(3 * far + width, dtype=torch.int8, device="cuda")
    view = q.as_strided((4, width), (far, 1))
    scales = torch.empty(4, device="cuda")
    Q = api.DnMat(q, 4, width, far)
    api.experts_quantise(handle, R, mat(api, x), Q, api.DnVec(scales), buffer=buffer)
    torch.cuda.synchronize()
    want, _ = rows.quantise(x)
    assert torch.equal(view.cpu(), want[[0, 1, 0, 1]])
    y = torch.empty(4, 4, device="cuda")
    api.scaled_mm(handle, Q, api.DnVec(scales), Q, api.DnVec(scales), mat(api, y))  # without tiles
    torch.cuda.synchronize()
    want, size = rows.scaled(view, scales, view, scales, 1.0, 0.0, y)
    ref.close(y, want, 5 * F32 * size)
    one = api.CsrMatrix(R.row_ptr, torch.zeros(4, dtype=torch.int32, device="cuda"), R.values, 2, 1)
    tiles = torch.empty(4, 4, device="cuda")
    more = ordered(api, handle, one, api.experts_scaled_mm_buffer_size(handle, one, Q, Q, mat(api, tiles)))
    api.experts_scaled_mm(handle, one, Q, api.DnVec(scales), Q, api.DnVec(scales), mat(api, tiles), buffer=more)
    no_error(pkg)
    ref.close(tiles, want, 5 * F32 * size)


@pytest.mark.parametrize("half", ["f16", "bf16"])
def test_rows_of_32_bits_summed_into_16(pkg, handle, half):
    """Products' results in f32, their sum and its gradient in 16 bits; numbers that f16 cannot hold become infinite."""
    from ops_sparse_b200 import api
    g = gen(31)
    R = routed(api, g, 90, 11, 3, wild=0.1, kind=half)
    s, _ = matrix(g, R.nnz, 130, "f32", 2)
    s[5] = 1e6
    out, whole = matrix(g, 90, 130, half, 6)
    buffer = ordered(api, handle, R)
    for beta in (0.0, 1.5):
        want, size, many = rows.combine(R.row_ptr, R.col_ind, R.values, s, 11, 2.0, beta, out)
        held = want.to(DTYPE[half]).double()  # infinite where the type is
        kept = outside(out, whole).clone()
        api.experts_combine(handle, R, mat(api, s), mat(api, out), 2.0, beta, buffer=buffer)
        no_error(pkg)
        ref.close(out, torch.where(held.isinf(), held, want), ref.rounding(out.dtype, want) + (many + 2) * F32 * size)
        assert torch.equal(outside(out, whole), kept)
        out.copy_(torch.randn(90, 130, generator=g, device="cuda"))
    d_s, d_values = torch.empty(R.nnz, 130, device="cuda"), torch.empty(R.nnz, device="cuda").to(DTYPE[half])
    s[5] = 1.0
    want, want_v, size_v = rows.combine_grad(R.row_ptr, R.col_ind, R.values, out, s, 11, 1.0, 0.0, d_s, d_values)
    api.experts_combine_grad(handle, R, mat(api, out), mat(api, s), mat(api, d_s), api.DnVec(d_values), buffer=buffer)
    no_error(pkg)
    ref.close(d_s, want, 3 * F32 * want.abs())
    ref.close(d_values, want_v, ref.rounding(d_values.dtype, want_v) + 132 * F32 * size_v)


def test_room_for_copies_has_to_be_asked_for(pkg, handle):
    """Operands off 16 bytes are copied behind the order: refused where no BufferSize call through this routing has counted them."""
    from ops_sparse_b200 import api
    g = gen(32)
    R = routed(api, g, 30, 5, 2)
    x, w = eights(g, R.nnz, 33, 3), eights(g, 5 * 20, 33, 0)
    sx, sw, y = torch.rand(R.nnz, generator=g, device="cuda"), torch.rand(100, generator=g, device="cuda"), torch.empty(R.nnz, 20, device="cuda")
    buffer = ordered(api, handle, R, 1 << 20)
    args = (mat(api, x), api.DnVec(sx), mat(api, w), api.DnVec(sw), mat(api, y))
    with pytest.raises(pkg.AclSparseError) as e:
        api.experts_scaled_mm(handle, R, *args, buffer=buffer)
    assert e.value.status == pkg.ACL_SPARSE_STATUS_INVALID_VALUE
    assert api.experts_scaled_mm_buffer_size(handle, R, args[0], args[2], args[4]) <= buffer.numel()
    api.experts_scaled_mm(handle, R, *args, buffer=buffer)
    no_error(pkg)
    _, _, starts = rows.order_of(R.col_ind, 5)
    for e in range(5):
        a, b, c = int(starts[e]), int(starts[e + 1]), slice(20 * e, 20 * e + 20)
        want, size = rows.scaled(x[a:b], sx[a:b], w[c], sw[c], 1.0, 0.0, y[a:b])
        ref.close(y[a:b], want, 5 * F32 * size)


def test_two_streams_at_once(pkg, handle):
    """Products of all forms on two streams side by side, again and again: the same bits as one after the other."""
    from ops_sparse_b200 import api
    g = gen(33)
    jobs = []
    for many, depth, channels, out in ((300, 2048, 600, "f32"), (40, 2048, 300, "f32"), (2, 512, 900, "bf16"), (40, 128, 20000, "bf16"), (20, 96, 200, "f16")):
        x, w = eights(g, many, depth), eights(g, channels, depth)
        sx, sw = torch.rand(many, generator=g, device="cuda") * 1e-3, torch.rand(channels, generator=g, device="cuda") * 1e-3
        y = torch.empty(many, channels, dtype=DTYPE[out], device="cuda")
        jobs.append((mat(api, x), api.DnVec(sx), mat(api, w), api.DnVec(sw), y))
        api.scaled_mm(handle, *jobs[-1][:4], mat(api, y))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    handles = [api.Handle(s) for s in streams]
    copies = [[(j, torch.empty_like(j[4])) for j in jobs] for _ in streams]
    made = [[(j, y, mat(api, y)) for j, y in c] for c in copies]
    torch.cuda.synchronize()
    for turn in range(20):
        for i in range(len(jobs)):
            for k, h in enumerate(handles):
                j, _, Y = made[k][(i + 2 * k + turn) % len(jobs)]
                api.scaled_mm(h, *j[:4], Y)
    no_error(pkg)
    for c in made:
        assert all(torch.equal(j[4], y) for j, y, _ in c)
    for h in handles:
        h.close()
