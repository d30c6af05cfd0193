"""GPU: token operators at their borders -- values that f32 cannot tell apart, weights that underflow, loops and offsets at the
last sizes that are taken, orders that are out of date."""
from __future__ import annotations

import math

import pytest
import torch

import token_reference as ref
from test_tokens_gpu import check_route, gen, mat, matrix, ragged, routed
from token_reference import DTYPE, F32

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- the choice

def test_route_three_saturated_scores(pkg, handle):
    """Scores that are all 1 in f32: the one left out equals the last one taken, the first one taken lies below both."""
    from ops_sparse_b200 import api
    R = check_route(api, handle, torch.tensor([[20.0, 21.0, 21.0]], device="cuda"), torch.zeros(3, device="cuda"), 2, score="sigmoid")
    assert R.col_ind.tolist() == [1, 2]


@pytest.mark.parametrize("score,high", [("sigmoid", 20.0), ("softmax", 0.0)])
@pytest.mark.parametrize("level", [0.0, 0.25])
@pytest.mark.parametrize("experts,k,groups", [(12, 4, 1), (64, 8, 4), (300, 10, 1)])
def test_route_equals_of_the_last_beside_near_ones(pkg, handle, score, high, level, experts, k, groups):
    """Few different logits, one bias for all, scores closer than a step of the selection values: a sigmoid near 1, or a softmax beside an
    expert that is larger by e^30.  In the second half of the rows all that are left out equal the last one taken, while lower ones have been taken."""
    from ops_sparse_b200 import api
    g = gen(experts + k)
    x = high + 0.5 * torch.randint(0, 4, (200, experts), generator=g, device="cuda").float()
    x[100:] = high + 1.0
    x[100:, :k - 1] -= 0.5 * torch.randint(0, 2, (100, k - 1), generator=g, device="cuda")
    if score == "softmax":
        x[torch.arange(200, device="cuda"), torch.randint(0, experts, (200,), generator=g, device="cuda")] = 30.0
    bias = torch.full((experts,), level, device="cuda")
    bias[experts // 2 if groups > 1 else experts:] -= 5.0  # which groups are kept is clear
    check_route(api, handle, x.bfloat16(), bias, k, score=score, groups=groups, kept=max(groups // 2, 1))


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("size,tokens", [(300.0, 1000), (64.0, 3000)])
def test_route_group_sums_of_large_opposite_biases(pkg, handle, score, size, tokens):
    """The sum of a group's two best is near 1, its terms are not: what is rounded are the terms.  All experts of the kept groups are taken."""
    from ops_sparse_b200 import api
    x = (1e-4 if score == "sigmoid" else 0.5) * torch.randn(tokens, 64, generator=gen(31), device="cuda")
    bias = torch.tensor([size, -size], device="cuda").repeat(32)
    check_route(api, handle, x, bias, 32, score=score, groups=32, kept=16, group_score="top2")


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_route_groups_of_the_lowest_biases(pkg, handle, score):
    """A bias of f32's lowest value masks nothing: a group whose two best have it is behind others, and before groups of masked experts."""
    from ops_sparse_b200 import api
    g = gen(37)
    lowest = torch.finfo(torch.float32).min
    x = torch.randn(400, 32, generator=g, device="cuda")
    x[:200, :8] = -math.inf  # the first groups are masked
    x[200:300, torch.randint(0, 32, (16,), generator=g, device="cuda")] = -math.inf
    bias = torch.where(torch.rand(32, generator=g, device="cuda") < 0.25, 0.5, lowest)
    check_route(api, handle, x, torch.full((32,), lowest, device="cuda"), 6, score=score, groups=8, kept=4, group_score="top2")
    check_route(api, handle, x, bias, 6, score=score, groups=8, kept=5, group_score="top2")
    check_route(api, handle, x, bias, 6, score=score, groups=8, kept=5, group_score="max")
    x[:200, 2:8] = 0.25 * torch.randint(0, 3, (200, 6), generator=g, device="cuda")
    # groups of two, the first masked; all experts of the kept ones are taken, so that no other comparison asks for f64
    check_route(api, handle, x[:200, :8], torch.full((8,), lowest, device="cuda"), 4, score=score, groups=4, kept=2, group_score="top2")


# ---------------------------------------------------------------- weights that underflow

FAR = [[-100.0, -101.0, -math.inf, -103.5], [-88.0, -89.0, -95.0, -400.0], [-90.0, -90.0, -90.0, -90.0], [3.0, -60.0, -95.0, -100.0],
       [-700.0, -699.0, -698.5, -702.0], [-0.5, -88.5, -89.0, 0.25]]


@pytest.mark.parametrize("x", ["f32", "bf16"])
@pytest.mark.parametrize("k", [2, 4])
def test_renormalised_weights_of_vanishing_sigmoids(pkg, handle, x, k):
    """Scores below the least f32: their quotients are not."""
    from ops_sparse_b200 import api
    check_route(api, handle, torch.tensor(FAR, device="cuda").to(DTYPE[x]), None, k, score="sigmoid", scale=2.0)
    R = routed(api, 1, 2, 2)
    api.route(handle, api.RouteRule(score="sigmoid"), mat(api, torch.tensor([[-10001.0, -10000.0]], device="cuda")), None, R)
    want = torch.softmax(torch.tensor([[0.0, 1.0]], dtype=torch.float64), 1)  # e^x / (1 + e^x) is e^x there
    ref.close(R.values.view(1, 2), want, want * 16 * F32)


def test_renormalised_weights_far_below_the_largest_logit(pkg, handle):
    """A softmax whose largest logit is not among the chosen, which a bias or a group brings about."""
    from ops_sparse_b200 import api
    x = torch.tensor([[0.0, -120.0, -121.0, -300.0], [50.0, -60.0, -60.0, -61.5], [5.0, 2.0, 3.0, -200.0]], device="cuda")
    R = check_route(api, handle, x, torch.tensor([0.0, 2.0, 2.0, 0.5], device="cuda"), 2)
    assert R.col_ind.tolist() == [1, 2] * 3
    check_route(api, handle, x, torch.tensor([0.0, 0.0, 2.0, 1.5], device="cuda"), 2, groups=2, kept=1, group_score="top2")


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("grad", ["f32", "bf16"])
def test_gradient_of_renormalised_weights_that_vanish(pkg, handle, score, grad):
    from ops_sparse_b200 import api
    x = torch.tensor(FAR, device="cuda")
    rule = {"score": score, "scale": 1.5}
    columns, weights = ref.route(x, None, 3, **rule)
    values = weights.float().cuda()  # as if they had been kept: none is 0 but that of the masked
    offsets = torch.arange(0, 3 * len(FAR) + 1, 3, dtype=torch.int32, device="cuda")
    R = api.CsrMatrix(offsets, columns.flatten().cuda(), values.flatten(), len(FAR), 4)
    d = torch.randn(3 * len(FAR), generator=gen(7), device="cuda").to(DTYPE[grad])
    out = torch.full_like(x, math.nan)
    api.route_grad(handle, api.RouteRule(**rule), mat(api, x), R, api.DnVec(d), mat(api, out))
    # dx = scale * q (g - sum g q) (1 - s for a sigmoid), q the weights over scale; each term with the errors of q: an exponential of a
    # difference of up to 302 and of x, to two units each, three additions, a division
    q, g = (weights / 1.5), d.double().cpu().view(-1, 3)
    chosen = x.double().cpu().gather(1, columns.long())
    rest = 1 / (1 + chosen.exp()) if score == "sigmoid" else 1.0
    want = torch.zeros(x.shape, dtype=torch.float64).scatter_(1, columns.long(), 1.5 * q * rest * (g - (g * q).sum(1, keepdim=True)))
    size = torch.zeros_like(want).scatter_(1, columns.long(), 1.5 * q * 2 * g.abs().amax(1, keepdim=True))
    ref.close(out, want, (size * (2 * 302 + 24) * F32).clamp_min(1e-37))
    assert (want[0].abs() > 1e-3).sum() >= 2


# ---------------------------------------------------------------- loops at the last sizes that are taken

def test_table_gradient_of_the_most_rows(pkg, handle):
    """2^31 - 2 rows, the largest table that is taken: a step past the last row is no int.  Scaled rows, and zeros of rows with a gap behind."""
    from ops_sparse_b200 import api
    vocab = 2 ** 31 - 2
    tokens, d = torch.tensor([vocab - 1, 3, vocab - 1], device="cuda"), torch.tensor([[1.0], [2.0], [4.0]], device="cuda").half()
    memory = torch.full((2 * vocab,), 3.0, dtype=torch.float16, device="cuda")
    table = memory[:vocab]
    api.embedding_grad(handle, mat(api, d), api.DnVec(tokens), api.DnMat(table, vocab, 1, 1), beta=0.5)
    assert table[-1] == 6.5 and table[3] == 3.5
    table[-1] = table[3] = 1.5
    assert (table == 1.5).all() and (memory[vocab:] == 3.0).all()
    memory.fill_(3.0)
    api.embedding_grad(handle, mat(api, d), api.DnVec(tokens), api.DnMat(memory, vocab, 1, 2))
    table = memory.view(vocab, 2)
    assert table[-1].tolist() == [5.0, 3.0] and table[3].tolist() == [2.0, 3.0]
    table[-1, 0] = table[3, 0] = 0.0
    assert (table[:, 0] == 0).all() and (table[:, 1] == 3.0).all()


def test_table_gradient_of_more_than_a_billion_tokens(pkg, handle):
    """Past 2^30 positions the sum of two of them is no int: rows whose tokens would come behind all that occur are looked for there."""
    from ops_sparse_b200 import api
    count = 2 ** 30 + 4097
    tokens = torch.full((count,), 5, dtype=torch.int32, device="cuda")
    d = torch.zeros(count, 1, dtype=torch.float16, device="cuda")
    d[::1 << 20] = 1.0  # 1025 of them
    table = torch.full((8, 1), 3.0, device="cuda")
    api.embedding_grad(handle, mat(api, d), api.DnVec(tokens), mat(api, table), alpha=2.0, beta=0.5)
    assert table.flatten().tolist() == [1.5] * 5 + [2051.5] + [1.5] * 2


def test_experts_of_more_than_a_billion_entries(pkg, handle):
    """1024 experts (two passes of the sort, experts' first places by search) and more than 2^30 entries."""
    from ops_sparse_b200 import api
    tokens, each, experts = 1024, 2 ** 20 + 2, 1024
    nnz = tokens * each
    columns = torch.tensor([3, experts - 1], dtype=torch.int32, device="cuda").repeat(nnz // 2)
    offsets = each * torch.arange(tokens + 1, dtype=torch.int32, device="cuda")
    R = api.CsrMatrix(offsets, columns, torch.empty(1, device="cuda"), tokens, experts, nnz)
    x, w = torch.zeros(tokens, 8, dtype=torch.bfloat16, device="cuda"), torch.zeros(experts, 8, dtype=torch.bfloat16, device="cuda")
    x[:, 0] = (torch.arange(tokens, device="cuda") % 8).bfloat16()
    w[3, 0], w[-1, 0] = 1.0, 2.0
    y = torch.full((nnz, 1), 9.0, dtype=torch.bfloat16, device="cuda")
    X, W, Y = mat(api, x), mat(api, w), mat(api, y)
    buffer = torch.empty(api.experts_buffer_size(handle, R, X, W, Y), dtype=torch.uint8, device="cuda")
    api.experts_preprocess(handle, R, buffer)
    api.experts_mm(handle, R, X, W, Y, buffer=buffer)
    torch.cuda.synchronize()
    assert pkg.lib().b200sp_experts_error() == 0
    y = y.view(tokens, each // 2, 2)
    assert (y[:, :, 0] == x[:, :1]).all() and (y[:, :, 1] == 2 * x[:, :1]).all()


def test_experts_of_more_than_a_billion_columns(pkg, handle):
    """Past 2^30 columns twice a column is no int: gradients of an expert that is one row of so many, or one column."""
    from ops_sparse_b200 import api
    wide = 2 ** 30 + 72
    one = torch.tensor([[3.0]], dtype=torch.bfloat16, device="cuda").expand(1, 8).contiguous()
    long = torch.zeros(1, wide, dtype=torch.bfloat16, device="cuda")
    spots = [0, 5, 2 ** 29 + 1, 2 ** 30 - 1, 2 ** 30, 2 ** 30 + 71]
    long[0, spots] = torch.arange(1, 7, device="cuda").bfloat16()
    R = api.CsrMatrix(torch.tensor([0, 1], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), torch.empty(1, device="cuda"), 1, 1)
    for dy, x in ((one, long), (long, one)):  # dW of 8 x wide, of wide x 8
        dw = torch.full((dy.shape[1], x.shape[1]), 9.0, dtype=torch.bfloat16, device="cuda")
        DY, X, DW = mat(api, dy), mat(api, x), mat(api, dw)
        buffer = torch.empty(api.experts_grad_buffer_size(handle, R, DY, X, DW), dtype=torch.uint8, device="cuda")
        api.experts_preprocess(handle, R, buffer)
        api.experts_grad(handle, R, DY, X, DW, buffer=buffer)
        torch.cuda.synchronize()
        assert pkg.lib().b200sp_experts_error() == 0
        if x is long:
            assert all(torch.equal(row, 3 * long[0]) for row in dw)
        else:
            assert all(torch.equal(dw[:, c], 3 * long[0]) for c in range(8))
        del dw, DW


def _waits(pkg):
    import ctypes
    f = pkg.lib().b200sp_experts_wait_test
    f.argtypes, f.restype = [ctypes.c_longlong, ctypes.c_uint], None
    return f


def test_a_long_sum_is_no_wait_that_runs_out(pkg, handle):
    """The results of a tile may take as long as its steps: with a limit of 400,000 clocks, an expert of 300,000 entries (4688 steps)."""
    from ops_sparse_b200 import api
    nnz = 300000
    g = gen(3)
    R = api.CsrMatrix(torch.arange(nnz + 1, dtype=torch.int32, device="cuda"), torch.zeros(nnz, dtype=torch.int32, device="cuda"), torch.empty(1, device="cuda"),
                      nnz, 1, nnz)
    x, dy = (torch.randint(-1, 2, (nnz, 64), generator=g, device="cuda").bfloat16() for _ in range(2))
    dw = torch.empty(64, 64, device="cuda")
    X, DY, DW = mat(api, x), mat(api, dy), mat(api, dw)
    buffer = torch.empty(api.experts_grad_buffer_size(handle, R, DY, X, DW), dtype=torch.uint8, device="cuda")
    api.experts_preprocess(handle, R, buffer)
    torch.cuda.synchronize()
    waits = _waits(pkg)
    try:
        waits(400_000, 0)
        api.experts_grad(handle, R, DY, X, DW, buffer=buffer)
        torch.cuda.synchronize()
    finally:
        waits(0, 0)
    error = pkg.lib().b200sp_experts_error()
    pkg.lib().b200sp_experts_error_clear()
    assert error == 0
    assert torch.equal(dw.double(), dy.double().T @ x.double())  # whole numbers below 2^24


def test_a_sum_over_more_than_a_billion_columns(pkg, handle):
    """2^24 steps in one tile: seconds, but no wait that runs out; columns past 2^30."""
    from ops_sparse_b200 import api
    wide = 2 ** 30 + 72
    x, w = torch.zeros(1, wide, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, wide, dtype=torch.bfloat16, device="cuda")
    spots = [0, 5, 2 ** 29 + 1, 2 ** 30 - 1, 2 ** 30, 2 ** 30 + 71]
    x[0, spots], w[0, spots] = torch.arange(1, 7, device="cuda").bfloat16(), torch.tensor([1.0, 8, 64, 512, 4096, 32768], device="cuda").bfloat16()
    R = api.CsrMatrix(torch.tensor([0, 1], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), torch.empty(1, device="cuda"), 1, 1)
    y = torch.full((1, 1), 9.0, device="cuda")
    X, W, Y = mat(api, x), mat(api, w), mat(api, y)
    buffer = torch.empty(api.experts_buffer_size(handle, R, X, W, Y), dtype=torch.uint8, device="cuda")
    api.experts_preprocess(handle, R, buffer)
    api.experts_mm(handle, R, X, W, Y, buffer=buffer)
    torch.cuda.synchronize()
    assert pkg.lib().b200sp_experts_error() == 0
    assert y.item() == 1 + 16 + 192 + 2048 + 20480 + 196608


def test_the_error_flag_waits_for_other_streams(pkg, device):
    """Asked, or cleared, right after a product on a stream that the default one does not wait for."""
    from ops_sparse_b200 import api
    stream = torch.cuda.Stream()
    L, waits = pkg.lib(), _waits(pkg)
    with torch.cuda.stream(stream):
        h = api.Handle(stream)
        g = gen(4)
        offsets, columns = ragged(g, 50, 4, 2, wild=0)
        x, w = matrix(g, 50, 64, "bf16")[0], matrix(g, 4 * 128, 64, "bf16")[0]
        y = torch.empty(len(columns), 128, dtype=torch.bfloat16, device="cuda")
        R = api.CsrMatrix(offsets, columns, torch.empty(len(columns), device="cuda"), 50, 4)
        X, W, Y = mat(api, x), mat(api, w), mat(api, y)
        buffer = torch.empty(api.experts_buffer_size(h, R, X, W, Y), dtype=torch.uint8, device="cuda")
        api.experts_preprocess(h, R, buffer)
        torch.cuda.synchronize()
        try:
            waits(200_000_000, 16)  # a tenth of a second
            api.experts_mm(h, R, X, W, Y, buffer=buffer)
            asked = L.b200sp_experts_error()
            L.b200sp_experts_error_clear()
            api.experts_mm(h, R, X, W, Y, buffer=buffer)
            L.b200sp_experts_error_clear()
        finally:
            waits(0, 0)
        torch.cuda.synchronize()
        left = L.b200sp_experts_error()
        L.b200sp_experts_error_clear()
        assert asked == 1 and left == 0
    h.close()


# ---------------------------------------------------------------- orders that are out of date

def small(pkg, api, handle, g, tokens=40, experts=6, k=2, n=24, d=32):
    """R as b200spRoute leaves it, the operands of a product, a buffer of its size."""
    R = routed(api, tokens, experts, k)
    logits = torch.randn(tokens, experts, generator=g, device="cuda")
    x, w = matrix(g, tokens, d, "bf16")[0], matrix(g, experts * n, d, "bf16")[0]
    y = torch.full((tokens * k, n), 5.0, dtype=torch.bfloat16, device="cuda")
    operands = mat(api, x), mat(api, w), mat(api, y)
    buffer = torch.empty(api.experts_buffer_size(handle, R, *operands), dtype=torch.uint8, device="cuda")

    def check():
        torch.cuda.synchronize()
        assert pkg.lib().b200sp_experts_error() == 0
        want, size = ref.experts_mm(R.row_ptr, R.col_ind, x, w.view(experts, n, d), experts, True, False, 1.0, 0.0, y)
        ref.close(y, want, ref.rounding(y.dtype, want) + size * (d + 4) * 2 * F32)

    return R, logits, operands, buffer, y, check


def test_routing_anew_ends_the_order(pkg, handle):
    from ops_sparse_b200 import api
    g = gen(21)
    R, logits, operands, buffer, _, check = small(pkg, api, handle, g)
    rule = api.RouteRule()
    api.route(handle, rule, mat(api, logits), None, R)
    api.experts_preprocess(handle, R, buffer)
    api.experts_mm(handle, R, *operands, buffer=buffer)
    check()
    logits.neg_()
    api.route(handle, rule, mat(api, logits), None, R)
    with pytest.raises(pkg.AclSparseError, match="INVALID_VALUE"):
        api.experts_mm(handle, R, *operands, buffer=buffer)
    api.experts_preprocess(handle, R, buffer)
    api.experts_mm(handle, R, *operands, buffer=buffer)
    check()


def test_a_matrix_made_anew_takes_a_buffer_of_the_known_size(pkg, handle):
    """Room has to have been asked for through the same descriptor for operands that are copied alone."""
    from ops_sparse_b200 import api
    g = gen(22)
    R, logits, operands, buffer, _, check = small(pkg, api, handle, g)
    api.route(handle, api.RouteRule(), mat(api, logits), None, R)
    again = api.CsrMatrix(R.row_ptr, R.col_ind, R.values, R.rows, R.cols)
    api.experts_preprocess(handle, again, buffer)
    api.experts_mm(handle, again, *operands, buffer=buffer)
    check()
    dw = torch.empty(6 * 24, 32, device="cuda")
    api.experts_grad(handle, again, operands[2], operands[0], mat(api, dw), buffer=buffer)
    want, size, many = ref.experts_grad(R.row_ptr, R.col_ind, operands[2].values, operands[0].values, 6, False, 1.0, 0.0, dw.view(6, 24, 32))
    ref.close(dw.view(6, 24, 32), want, ref.rounding(dw.dtype, want) + size * (many + 4) * 2 * F32)
    odd = mat(api, matrix(g, 40, 32, "bf16", shift=1)[0])
    with pytest.raises(pkg.AclSparseError, match="INVALID_VALUE"):
        api.experts_mm(handle, again, odd, *operands[1:], buffer=buffer)


def test_a_captured_order_is_not_the_one_before_it(pkg, device):
    """A buffer that holds an order, an order of other columns captured but not replayed: an eager product does not follow the old one."""
    from ops_sparse_b200 import api
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        h = api.Handle(stream)
        R, logits, operands, buffer, y, check = small(pkg, api, h, gen(23))
        rule, L = api.RouteRule(), mat(api, logits)
        api.route(h, rule, L, None, R)
        api.experts_preprocess(h, R, buffer)
        api.experts_mm(h, R, *operands, buffer=buffer)
        check()
        logits.neg_()
        api.route(h, rule, L, None, R)
        stream.synchronize()
        graph, both = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            api.experts_preprocess(h, R, buffer)
        y.fill_(5.0)
        api.experts_mm(h, R, *operands, buffer=buffer)
        stream.synchronize()
        error = pkg.lib().b200sp_experts_error()
        pkg.lib().b200sp_experts_error_clear()
        assert error == 2 and (y == 5).all()
        graph.replay()
        api.experts_mm(h, R, *operands, buffer=buffer)
        check()
        # products in graphs follow what the buffer holds when they are replayed: of the same graph, or of eager calls
        with torch.cuda.graph(both, stream=stream):
            api.route(h, rule, L, None, R)
            api.experts_preprocess(h, R, buffer)
            api.experts_mm(h, R, *operands, buffer=buffer)
        alone = torch.cuda.CUDAGraph()
        with torch.cuda.graph(alone, stream=stream):
            api.experts_mm(h, R, *operands, buffer=buffer)
        for _ in range(2):
            logits.mul_(-1.5)
            both.replay()
            check()
            api.experts_mm(h, R, *operands, buffer=buffer)
            check()
        logits.neg_()
        api.route(h, rule, L, None, R)
        api.experts_preprocess(h, R, buffer)
        alone.replay()
        check()
        graph.replay()
        api.experts_mm(h, R, *operands, buffer=buffer)  # an eager order before, whatever graph wrote the same since
        check()
        del graph, both, alone
    h.close()


def test_graphs_that_order_the_same_entries_in_turn(pkg, device):
    """Two graphs that route, order and multiply; eager products after either of them, the first captured replayed last."""
    from ops_sparse_b200 import api
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        h = api.Handle(stream)
        R, logits, operands, buffer, y, check = small(pkg, api, h, gen(24))
        rule, L = api.RouteRule(score="sigmoid"), mat(api, logits)
        api.route(h, rule, L, None, R)
        api.experts_preprocess(h, R, buffer)
        api.experts_mm(h, R, *operands, buffer=buffer)
        check()
        graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
        for graph in graphs:
            with torch.cuda.graph(graph, stream=stream):
                api.route(h, rule, L, None, R)
                with pytest.raises(pkg.AclSparseError, match="INVALID_VALUE"):
                    api.experts_mm(h, R, *operands, buffer=buffer)
                api.experts_preprocess(h, R, buffer)
                api.experts_mm(h, R, *operands, buffer=buffer)
        for graph in (graphs[1], graphs[0], graphs[1], graphs[0]):
            logits.mul_(-1.25)
            graph.replay()
            check()
            y.fill_(5.0)
            api.experts_mm(h, R, *operands, buffer=buffer)
            check()
        del graphs
    h.close()
