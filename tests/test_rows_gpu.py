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


def test_scaled_extreme_scales(pkg, handle):
    """Scales whose product f32 cannot hold, of sums that bring the result back, and some that are not finite."""
    from ops_sparse_b200 import api
    g = gen(77)
    x, w = eights(g, 40, 512), eights(g, 200, 512)
    x[:, 0] = 127
    sx = torch.tensor([1e-30, 1e-25, 1e25, 1e38, 1.0, 0.0, 1e-38, 1e-45], device="cuda").repeat(5)
    sw = torch.tensor([1e-20, 1e-10, 1.0, 1e10, 1e-25, 1e-38, 3e38, 0.0], device="cuda").repeat(25)
    for alpha in (1.0, 1e15, 1e-15):
        y = torch.empty(40, 200, device="cuda")
        api.scaled_mm(handle, mat(api, x), api.DnVec(sx), mat(api, w), api.DnVec(sw), mat(api, y), alpha=alpha)
        torch.cuda.synchronize()
        want, _ = rows.scaled(x, sx, w, sw, float(torch.tensor(alpha)), 0.0, y)
        held = want.float().double()  # infinite where f32 is
        ref.close(y, torch.where(want.abs() > 3.4028235e38, held, want), ref.rounding(y.dtype, want) + 5 * F32 * want.abs())
    sx = torch.ones(40, device="cuda")
    sx[3], sx[4] = math.nan, math.inf
    y = torch.empty(40, 200, dtype=torch.float16, device="cuda")
    api.scaled_mm(handle, mat(api, x), api.DnVec(sx), mat(api, w), api.DnVec(torch.ones(200, device="cuda")), mat(api, y))
    torch.cuda.synchronize()
    assert bool(y[3].isnan().all()) and bool((~y[4].isfinite()).all()) and not bool(y[[0, 1, 2, 5, 39]].isnan().any())


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
