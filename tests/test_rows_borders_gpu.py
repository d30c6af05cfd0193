"""GPU: operators of include/b200sp_rows.h at their borders -- beside other streams, in each form of a product, at far addresses."""
from __future__ import annotations

import math
from ctypes import c_int32

import pytest
import torch

import rows_reference as rows
import token_reference as ref
from test_rows_gpu import eights, no_error, ordered, routed
from test_tokens_gpu import gen, mat, matrix, outside
from token_reference import DTYPE, F32

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- beside other streams

def test_long_order_leaves_the_sms_to_other_streams(pkg, handle):
    """An order of a million entries takes eight SMs for some 300 us.  The product that follows it takes all of them, and has to leave them to another
    stream's product until the order is there: that one is done first."""
    from ops_sparse_b200 import api
    g = gen(51)
    streams = [torch.cuda.Stream() for _ in range(2)]
    first, other = api.Handle(streams[0]), api.Handle(streams[1])
    R = routed(api, g, 131072, 64, 8)
    x, w = eights(g, R.nnz, 64), eights(g, 64 * 64, 64)
    sx, sw, y = torch.rand(R.nnz, device="cuda"), torch.rand(64 * 64, device="cuda"), torch.empty(R.nnz, 64, device="cuda").bfloat16()
    X, W, Y, SX, SW = mat(api, x), mat(api, w), mat(api, y), api.DnVec(sx), api.DnVec(sw)
    buffer = torch.empty(api.experts_scaled_mm_buffer_size(first, R, X, W, Y), dtype=torch.uint8, device="cuda")
    few, wide = eights(g, 40, 128), eights(g, 20000, 128)
    ones, many, out = torch.ones(40, device="cuda"), torch.ones(20000, device="cuda"), torch.empty(40, 20000, device="cuda")
    args = (mat(api, few), api.DnVec(ones), mat(api, wide), api.DnVec(many), mat(api, out))
    torch.cuda.synchronize()
    parts = []
    for _ in range(6):  # the host may be late in one of them
        start, *ends = [torch.cuda.Event(enable_timing=True) for _ in range(3)]
        start.record(streams[0])
        api.experts_preprocess(first, R, buffer)
        api.experts_scaled_mm(first, R, X, SX, W, SW, Y, buffer=buffer)
        api.scaled_mm(other, *args)
        ends[0].record(streams[0])
        ends[1].record(streams[1])
        torch.cuda.synchronize()
        parts.append(start.elapsed_time(ends[1]) / start.elapsed_time(ends[0]))
    no_error(pkg)
    assert min(parts) < 0.5, parts  # 35 us of 460; held back it is 1
    want, size = rows.scaled(few, ones, wide, many, 1.0, 0.0, out)
    ref.close(out, want, 5 * F32 * size)
    first.close()
    other.close()


# ---------------------------------------------------------------- products in 8 bits, each in the form that it says

WHOLE, PAIRS, SHARED, FEW = range(4)


def form_of(pkg, X, W, Y, R=None):
    info = (c_int32 * 3)()
    assert pkg.lib().b200spScaledMMInfo(None if R is None else R.raw, X.raw, W.raw, Y.raw, info) == 0
    return tuple(info)


def exact_sums(x, w):
    """Sums of products of 8 bits, in 64, on the GPU."""
    return x.double() @ w.double().T


FORMS = [  # rows, depth, channels, out, alpha, beta, pad and shift of Y, form
    (1836, 38, 2524, "bf16", 1.0, 0.0, 4, 0, (PAIRS, 64, 1)),  # rows of Y on 16 bytes that end within a piece
    (900, 128, 4744, "f16", 0.5, 0.0, 0, 0, (PAIRS, 64, 1)),
    (900, 128, 4744, "bf16", 1.0, 0.5, 1, 1, (PAIRS, 64, 1)),
    (638, 32, 13146, "f32", 1.0, 0.0, 0, 0, (PAIRS, 128, 1)),
    (842, 32, 14333, "bf16", 2.0, 0.0, 3, 0, (PAIRS, 256, 1)),
    (2048, 4096, 4096, "bf16", 1.0, 0.0, 0, 0, (PAIRS, 256, 1)),
    (2048, 4096, 4096, "f32", -1.0, 2.0, 0, 0, (PAIRS, 256, 1)),
    (4096, 2048, 2048, "f16", 1.0, 0.0, 0, 0, (PAIRS, 256, 1)),
    (17, 2048, 4360, "bf16", 1.0, 0.0, 0, 0, (SHARED, 16, 2)),
    (1128, 2950, 138, "f32", 1.0, 1.0, 0, 0, (SHARED, 32, 2)),
    (39, 4008, 5224, "f16", 1.0, 0.0, 0, 0, (SHARED, 64, 2)),
    (66, 2788, 2212, "bf16", 1.0, -0.5, 5, 3, (SHARED, 128, 4)),
    (142, 3856, 4062, "f32", 1.0, 0.0, 0, 0, (SHARED, 256, 4)),
    (132, 1941, 1724, "bf16", 1.0, 0.0, 4, 0, (SHARED, 256, 8)),
    (320, 512, 200, "bf16", 1.0, 0.0, 0, 0, (WHOLE, 16, 1)),
    (700, 512, 4100, "bf16", 1.0, 0.0, 4, 0, (WHOLE, 256, 1)),
    (16, 2048, 640, "f32", 1.0, 1.0, 0, 0, (FEW, 0, 1)),
]


@pytest.mark.parametrize("many,depth,channels,out,alpha,beta,pad,shift,form", FORMS)
def test_scaled_product_of_a_form(pkg, handle, many, depth, channels, out, alpha, beta, pad, shift, form):
    from ops_sparse_b200 import api
    g = gen(many + depth + channels)
    x, w = eights(g, many, depth, -depth % 16), eights(g, channels, depth, -depth % 16)
    sx, sw = torch.rand(many, generator=g, device="cuda") * 1e-2, torch.rand(channels, generator=g, device="cuda") * 1e-3
    y, whole = matrix(g, many, channels, out, pad, shift)
    X, W, Y = mat(api, x), mat(api, w), mat(api, y)
    assert form_of(pkg, X, W, Y) == form and api.scaled_mm_buffer_size(handle, X, W, Y) == 0
    want = alpha * exact_sums(x, w) * sx.double()[:, None] * sw.double()
    old = beta * y.double() if beta else torch.zeros_like(want)
    if beta == 0:
        y.fill_(math.nan)  # must not be read
    kept = outside(y, whole).clone()
    api.scaled_mm(handle, X, api.DnVec(sx), W, api.DnVec(sw), Y, alpha, beta)
    no_error(pkg)
    # the sum is exact; its f32, the scales' product, theirs, alpha's and beta's are rounded, then the result
    ref.close(y, want + old, ref.rounding(y.dtype, want + old) + 5 * F32 * (want.abs() + old.abs()))
    assert torch.equal(outside(y, whole), kept)


@pytest.mark.parametrize("many,depth,channels,form", [(900, 128, 4744, (PAIRS, 64, 1)), (17, 2048, 4360, (SHARED, 16, 2))])
def test_scaled_extreme_scales_of_a_form(pkg, handle, many, depth, channels, form):
    """Scales whose product f32 cannot hold, of sums that bring the result back, and some that are not finite."""
    from ops_sparse_b200 import api
    g = gen(79)
    x, w = eights(g, many, depth), eights(g, channels, depth)
    x[:, 0] = 127
    sx = torch.tensor([1e-30, 1e25, 1e-25, 1e38, 1.0, 0.0, 1e-38, 1e-45], device="cuda").repeat(many // 8 + 1)[:many].contiguous()
    sw = torch.tensor([1e-20, 1e-10, 1.0, 1e10, 1e-25, 1e-38, 3e38, 0.0], device="cuda").repeat(channels // 8)
    y = torch.empty(many, channels, device="cuda")
    X, W, Y = mat(api, x), mat(api, w), mat(api, y)
    assert form_of(pkg, X, W, Y) == form
    sums = exact_sums(x, w)
    for alpha in (1.0, 2.0 ** 50, 2.0 ** -50):
        api.scaled_mm(handle, X, api.DnVec(sx), W, api.DnVec(sw), Y, alpha=alpha)
        torch.cuda.synchronize()
        want = alpha * (sums * sx.double()[:, None] * sw.double())
        held = want.float().double()  # infinite where f32 is
        ref.close(y, torch.where(want.abs() > 3.4028235e38, held, want), ref.rounding(y.dtype, want) + 5 * F32 * want.abs())
    sx = torch.ones(many, device="cuda")
    sx[0], sx[1] = math.nan, math.inf
    half = torch.empty(many, channels, dtype=torch.float16, device="cuda")
    api.scaled_mm(handle, X, api.DnVec(sx), W, api.DnVec(torch.full((channels,), 1e-3, device="cuda")), mat(api, half))
    no_error(pkg)
    assert bool(half[0].isnan().all()) and bool((~half[1].isfinite()).all()) and not bool(half[2:].isnan().any())


@pytest.mark.parametrize("tokens,experts,k,depth,channels,out,pad,form", [
    (900, 4, 2, 384, 520, "bf16", 0, (PAIRS, 256, 1)), (901, 4, 2, 272, 393, "f16", 7, (PAIRS, 256, 1)),
    (333, 9, 2, 640, 260, "bf16", 4, (PAIRS, 128, 1)), (333, 9, 2, 640, 128, "bf16", 0, (WHOLE, 128, 1)),
    (1, 8, 2, 512, 300, "bf16", 4, (FEW, 0, 1)), (2, 8, 2, 512, 300, "bf16", 4, (WHOLE, 16, 1)),
])
def test_experts_scaled_product_of_a_form(pkg, handle, tokens, experts, k, depth, channels, out, pad, form):
    """Results of 16 bits in rows that start on 16 bytes: stored by way of shared memory, with ends within a piece and a tile."""
    from ops_sparse_b200 import api
    g = gen(tokens + depth + channels)
    R = routed(api, g, tokens, experts, k, 1.0, 0.05 if tokens > 9 else 0.0)
    x, w = eights(g, R.nnz, depth), eights(g, experts * channels, depth)
    sx, sw = torch.rand(R.nnz, generator=g, device="cuda") * 1e-2, torch.rand(experts * channels, generator=g, device="cuda") * 1e-3
    y, whole = matrix(g, R.nnz, channels, out, pad)
    X, W, Y = mat(api, x), mat(api, w), mat(api, y)
    assert form_of(pkg, X, W, Y, R) == form
    _, _, starts = rows.order_of(R.col_ind, experts)
    sx[int(starts[-1]):] = math.nan  # rows of no expert are not looked at
    want = torch.zeros(y.shape, dtype=torch.float64, device="cuda")
    for e in range(experts):
        a, b, c = int(starts[e]), int(starts[e + 1]), slice(e * channels, (e + 1) * channels)
        want[a:b] = exact_sums(x[a:b], w[c]) * sx[a:b].double()[:, None] * sw[c].double()
    y.fill_(math.nan)
    kept = outside(y, whole).clone()
    buffer = ordered(api, handle, R, api.experts_scaled_mm_buffer_size(handle, R, X, W, Y))
    api.experts_scaled_mm(handle, R, X, api.DnVec(sx), W, api.DnVec(sw), Y, buffer=buffer)
    no_error(pkg)
    ref.close(y, want, ref.rounding(y.dtype, want) + 5 * F32 * want.abs())
    assert torch.equal(outside(y, whole), kept)


@pytest.mark.parametrize("many,depth,channels,form", [(2048, 4096, 4096, (PAIRS, 256, 1)), (900, 128, 4744, (PAIRS, 64, 1)),
                                                      (17, 2048, 4360, (SHARED, 16, 2))])
def test_scaled_wait_that_runs_out_in_a_form(pkg, handle, many, depth, channels, form):
    """Every wait for a copy runs out (bytes are expected that nobody sends): the flag says so, Y is as it was, and the next product is right."""
    from ops_sparse_b200 import api
    L, g = pkg.lib(), gen(26)
    x, w = eights(g, many, depth), eights(g, channels, depth)
    sx, sw = torch.rand(many, generator=g, device="cuda"), torch.rand(channels, generator=g, device="cuda")
    y = torch.full((many, channels), 3.0, dtype=torch.bfloat16, device="cuda")
    args = (mat(api, x), api.DnVec(sx), mat(api, w), api.DnVec(sw), mat(api, y))
    assert form_of(pkg, args[0], args[2], args[4]) == form
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
    want = exact_sums(x, w) * sx.double()[:, None] * sw.double()
    ref.close(y, want, ref.rounding(y.dtype, want) + 5 * F32 * want.abs())


def test_all_forms_on_two_streams_at_once(pkg, handle):
    """Products of all forms on two streams side by side, again and again: the same bits as one after the other."""
    from ops_sparse_b200 import api
    g, jobs, forms = gen(34), [], set()
    for many, depth, channels, out in ((2048, 4096, 4096, "bf16"), (900, 128, 4744, "bf16"), (638, 32, 13146, "f32"), (17, 2048, 4360, "f16"),
                                       (142, 3856, 4062, "f32"), (700, 512, 4100, "bf16"), (2, 512, 900, "bf16")):
        x, w = eights(g, many, depth), eights(g, channels, depth)
        sx, sw = torch.rand(many, generator=g, device="cuda") * 1e-3, torch.rand(channels, generator=g, device="cuda") * 1e-3
        y = torch.empty(many, channels, dtype=DTYPE[out], device="cuda")
        jobs.append((mat(api, x), api.DnVec(sx), mat(api, w), api.DnVec(sw), y))
        forms.add(form_of(pkg, jobs[-1][0], jobs[-1][2], mat(api, y))[0])
        api.scaled_mm(handle, *jobs[-1][:4], mat(api, y))
    assert forms == {WHOLE, PAIRS, SHARED, FEW}
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    handles = [api.Handle(s) for s in streams]
    made = [[(j, y, mat(api, y)) for j, y in [(j, torch.empty_like(j[4])) for j in jobs]] for _ in streams]
    torch.cuda.synchronize()
    for turn in range(20):
        for i in range(len(jobs)):
            for k, h in enumerate(handles):
                j, _, Y = made[k][(i + 3 * k + turn) % len(jobs)]
                api.scaled_mm(h, *j[:4], Y)
    no_error(pkg)
    for c in made:
        assert all(torch.equal(j[4], y) for j, y, _ in c)
    for h in handles:
        h.close()


# ---------------------------------------------------------------- gradients, and rows far apart

def test_gradients_of_a_layer_term_by_term(pkg, handle):
    """Dispatch, a product of every expert, combine, and back, against 64 bits' automatic differentiation, within what the terms of each sum allow."""
    from ops_sparse_b200 import api
    g = gen(12)
    tokens, experts, k, d = 45, 7, 2, 40
    R = routed(api, g, tokens, experts, k)
    x, w, d_out = (torch.randn(s, generator=g, device="cuda") for s in ((tokens, d), (experts, d, d), (tokens, d)))
    buffer, starts = ordered(api, handle, R), torch.empty(experts + 1, dtype=torch.int32, device="cuda")
    new = lambda many: torch.full((many, d), math.nan, device="cuda")  # noqa: E731
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
    token, G, W = torch.arange(tokens, device="cuda").repeat_interleave(k), d_out.double(), w.double()[R.col_ind.long()]
    rows_ = torch.einsum("ih,ihf->if", leaf[token], W)
    total = torch.zeros(tokens, d, dtype=torch.float64, device="cuda").index_add(0, token, values[:, None] * rows_)
    gx, gv = torch.autograd.grad((total * G).sum(), (leaf, values))
    rows_, values, total = rows_.detach(), values.detach(), total.detach()
    of_token = lambda terms: torch.zeros(tokens, d, dtype=torch.float64, device="cuda").index_add(0, token, terms)  # noqa: E731
    # rows of f32, a product and a sum for each of a token's k entries, alpha
    ref.close(out, total, (k + 2) * F32 * of_token((values[:, None] * rows_).abs()), "sums")
    # rows of f32, d products each added with one rounding, the sums of a warp's lanes among them, alpha
    ref.close(d_values, gv, (d + 2) * F32 * (G[token] * rows_).abs().sum(1), "weights' gradient")
    # alpha w and its product with dOut, rows of f32, a sum for each of the k entries, alpha
    ref.close(d_x, gx, (k + 4) * F32 * of_token(torch.einsum("if,ihf->ih", (values[:, None] * G[token]).abs(), W.abs())), "tokens' gradient")


def test_gradients_of_rows_beyond_32_bits(pkg, handle):
    """The weights' gradient of rows that lie 2^31 bytes apart, and theirs, beside them and in their place."""
    from ops_sparse_b200 import api
    g = gen(28)
    far, width = 2 ** 30 + 16, 40
    R = api.CsrMatrix(torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda"), torch.tensor([0, 2, 1, 2], dtype=torch.int32, device="cuda"),
                      torch.tensor([1.0, -2.0, 0.5, 3.0], device="cuda"), 2, 3)
    buffer = ordered(api, handle, R)
    s = torch.zeros(3 * far + width, dtype=torch.bfloat16, device="cuda")
    view = s.as_strided((4, width), (far, 1))
    view.copy_(torch.randn(4, width, generator=g, device="cuda"))
    x = torch.randn(2, width, generator=g, device="cuda").bfloat16()
    S, held = api.DnMat(s, 4, width, far), view.clone()
    d_rows, d_values = torch.empty(4, width, device="cuda").bfloat16(), torch.empty(4, device="cuda")
    want, want_v, size_v = rows.combine_grad(R.row_ptr, R.col_ind, R.values, x, held, 3, 1.0, 0.0, d_rows, d_values)
    for to, seen in ((mat(api, d_rows), d_rows), (S, view)):
        d_values.fill_(math.nan)
        api.experts_combine_grad(handle, R, mat(api, x), S, to, api.DnVec(d_values), buffer=buffer)
        no_error(pkg)
        ref.close(d_values, want_v, (width + 2) * F32 * size_v)
        ref.close(seen, want, ref.rounding(torch.bfloat16, want) + 2 * F32 * want.abs())


@pytest.mark.parametrize("tokens", [3, 2000])
@pytest.mark.parametrize("beta", [0.0, 2.0])
def test_entries_of_no_expert_whatever_alpha_is(pkg, handle, tokens, beta):
    """Their first terms are 0 in every call, with an alpha that is not finite, too."""
    from ops_sparse_b200 import api
    g = gen(71)
    R = routed(api, g, tokens, 6, 2, wild=0.5)
    buffer = ordered(api, handle, R)
    _, places, starts = rows.order_of(R.col_ind, 6)
    end, none = int(starts[-1]), places >= int(starts[-1])
    assert 0 < end < R.nnz
    x, s = matrix(g, tokens, 24, "f32")[0], matrix(g, R.nnz, 24, "f32")[0]
    d_rows, d_values, out = matrix(g, R.nnz, 24, "f32")[0], torch.randn(R.nnz, generator=g, device="cuda"), matrix(g, R.nnz, 24, "f32")[0]
    want = [beta * t.cpu() for t in (d_rows[end:], d_values.cpu()[none], out[end:])]
    api.experts_combine_grad(handle, R, mat(api, x), mat(api, s), mat(api, d_rows), api.DnVec(d_values), math.inf, beta, buffer=buffer)
    api.experts_dispatch(handle, R, mat(api, x), mat(api, out), math.inf, beta, buffer=buffer)
    no_error(pkg)
    for t, w in zip((d_rows[end:], d_values.cpu()[none], out[end:]), want):
        assert torch.equal(t.cpu(), w)
    assert not bool(d_rows[:end].isfinite().any()) and not bool(out[:end].isfinite().any())


@pytest.mark.parametrize("out,beta", [("bf16", 0.0), ("f16", 0.5), ("f32", 0.0)])
@pytest.mark.parametrize("many,depth,channels,kind", [(2, 96, 72, FEW), (4, 4096, 4096, SHARED), (4, 96, 72, None)], ids=["rows", "clusters", "tiles"])
def test_results_beyond_32_bits(pkg, handle, many, depth, channels, kind, out, beta):
    """Rows of Y that lie more than 2^31 elements from the first; `None`: those of an expert, by tiles."""
    from ops_sparse_b200 import api
    g = gen(many + depth)
    far = (2 ** 31 if many == 2 else 2 ** 30) - 16 if out == "f32" else 2 ** 31 - 16
    x, w = eights(g, many, depth), eights(g, channels, depth)
    sx, sw = torch.rand(many, generator=g, device="cuda") * 1e-2, torch.rand(channels, generator=g, device="cuda") * 1e-3
    y = torch.zeros((many - 1) * far + channels, dtype=DTYPE[out], device="cuda")
    view = y.as_strided((many, channels), (far, 1))
    view.copy_(torch.randn(many, channels, generator=g, device="cuda"))
    X, W, Y = mat(api, x), mat(api, w), api.DnMat(y, many, channels, far)
    want = exact_sums(x, w) * sx.double()[:, None] * sw.double()
    old = beta * view.double()
    if kind is None:
        R = api.CsrMatrix(torch.tensor([0, many], dtype=torch.int32, device="cuda"), torch.zeros(many, dtype=torch.int32, device="cuda"),
                          torch.ones(many, device="cuda"), 1, 1)
        assert form_of(pkg, X, W, Y, R)[0] == WHOLE
        buffer = ordered(api, handle, R, api.experts_scaled_mm_buffer_size(handle, R, X, W, Y))
        api.experts_scaled_mm(handle, R, X, api.DnVec(sx), W, api.DnVec(sw), Y, 1.0, beta, buffer=buffer)
    else:
        assert form_of(pkg, X, W, Y)[0] == kind
        api.scaled_mm(handle, X, api.DnVec(sx), W, api.DnVec(sw), Y, 1.0, beta)
    no_error(pkg)
    ref.close(view, want + old, ref.rounding(y.dtype, want + old) + 5 * F32 * (want.abs() + old.abs()))


# ---------------------------------------------------------------- rounding to 8 bits

@pytest.mark.parametrize("kind,bits,far", [("bf16", 8, 0), ("bf16", 8, -110), ("bf16", 8, 110), ("f16", 11, 0)])
def test_every_quotient_of_16_bits(pkg, handle, kind, bits, far):
    """Each mantissa as a row's largest value, beside every value of ten powers of two below it: all quotients there are, halves among them."""
    from ops_sparse_b200 import api
    mantissas = torch.arange(2 ** (bits - 1), 2 ** bits, dtype=torch.float64, device="cuda")
    values = torch.cat([mantissas * 2.0 ** -e for e in range(10)])
    x = torch.where(values[None] <= mantissas[:, None], values[None], 0.0)
    x[:, 1::2] *= -1
    x[:, -1] = mantissas
    x = (x * 2.0 ** (far - 4)).to(DTYPE[kind])
    size, top = x.double().abs(), x.double().abs().amax(1, keepdim=True)
    want = torch.floor(127 * size / top)
    over = 254 * size - (2 * want + 1) * top  # exact: few bits each
    want = torch.sign(x.double()) * (want + ((over > 0) | ((over == 0) & (want % 2 == 1))))
    assert int((over == 0).sum()) > 0 and torch.equal(top[:, 0], mantissas * 2.0 ** (far - 4))
    q, scales = torch.empty(x.shape, dtype=torch.int8, device="cuda"), torch.empty(len(x), device="cuda")
    api.quantise_rows(handle, mat(api, x), mat(api, q), api.DnVec(scales))
    torch.cuda.synchronize()
    assert torch.equal(q.double(), want) and torch.equal(scales.cpu(), top[:, 0].float().cpu() / 127)


@pytest.mark.parametrize("many,width,kind", [(9000, 2300, "bf16"), (14000, 1100, "f32"), (4100, 4200, "f16"), (40000, 40, "f32"), (5000, 8300, "bf16")])
def test_more_rows_to_8_bits_than_ctas(pkg, handle, many, width, kind):
    """CTAs that go on to further rows, with one to eight warps at each."""
    from ops_sparse_b200 import api
    x, _ = matrix(gen(many), many, width, kind, -width % 8)
    x[::3] *= 2.0 ** -10
    size, top = x.double().abs(), x.double().abs().amax(1, keepdim=True)
    want = torch.floor(127 * size / top)
    over = 254 * size - (2 * want + 1) * top
    want = torch.sign(x.double()) * (want + ((over > 0) | ((over == 0) & (want % 2 == 1))))
    q, scales = torch.empty(x.shape, dtype=torch.int8, device="cuda"), torch.empty(many, device="cuda")
    api.quantise_rows(handle, mat(api, x), mat(api, q), api.DnVec(scales))
    torch.cuda.synchronize()
    assert torch.equal(q.double(), want) and torch.equal(scales.cpu(), top[:, 0].float().cpu() / 127)


def test_copies_of_operands_in_a_graph(pkg, handle):
    """Operands off 16 bytes, captured with the order of a routing and without, replayed on other values; the order is made anew in between."""
    from ops_sparse_b200 import api
    g, stream = gen(61), torch.cuda.Stream()
    h = api.Handle(stream)
    R = routed(api, g, 30, 5, 2)
    x, w, w1 = eights(g, R.nnz, 33, 3), eights(g, 5 * 20, 33), eights(g, 50, 33)
    sx, sw, one = torch.rand(R.nnz, generator=g, device="cuda"), torch.rand(100, generator=g, device="cuda"), torch.rand(50, generator=g, device="cuda")
    y, y1 = torch.empty(R.nnz, 20, device="cuda"), torch.empty(R.nnz, 50, device="cuda")
    X, W, W1, Y, Y1 = mat(api, x), mat(api, w), mat(api, w1), mat(api, y), mat(api, y1)
    SX, SW, ONE = api.DnVec(sx), api.DnVec(sw), api.DnVec(one)
    size = api.experts_scaled_mm_buffer_size(h, R, X, W, Y)
    buffer = torch.full((size + 3,), 255, dtype=torch.uint8, device="cuda")[3:]
    own = torch.full((api.scaled_mm_buffer_size(h, X, W1, Y1) + 5,), 255, dtype=torch.uint8, device="cuda")[5:]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        api.experts_preprocess(h, R, buffer)
        api.experts_scaled_mm(h, R, X, SX, W, SW, Y, buffer=buffer)
        api.scaled_mm(h, X, SX, W1, ONE, Y1, buffer=own)
    for turn in range(3):
        x.copy_(eights(g, R.nnz, 33))
        w.copy_(eights(g, 100, 33))
        R.col_ind.copy_(torch.randint(0, 5, (R.nnz,), generator=g, device="cuda").int())
        torch.cuda.synchronize()
        graph.replay()
        no_error(pkg)
        _, _, starts = rows.order_of(R.col_ind, 5)
        for e in range(5):
            a, b, c = int(starts[e]), int(starts[e + 1]), slice(20 * e, 20 * e + 20)
            want, much = rows.scaled(x[a:b], sx[a:b], w[c], sw[c], 1.0, 0.0, y[a:b])
            ref.close(y[a:b], want, 5 * F32 * much)
        want, much = rows.scaled(x, sx, w1, one, 1.0, 0.0, y1)
        ref.close(y1, want, 5 * F32 * much)
    h.close()
