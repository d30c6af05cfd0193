"""GPU: embedding rows, routing, experts' products and their gradients against plain implementations in 64 bits
(token_reference.py), at the sizes, masks and layouts where they can go wrong."""
from __future__ import annotations

import math

import pytest
import torch

import token_reference as ref
from token_reference import DTYPE, F32

pytestmark = pytest.mark.gpu


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def matrix(g, rows, cols, kind, pad=0, shift=0, size=1.0):
    """A rows x cols view with `pad` more elements a row that starts `shift` elements into its memory, and the memory."""
    whole = torch.full((rows * (cols + pad) + shift,), 7.0, dtype=DTYPE[kind], device="cuda")
    view = whole[shift:].view(rows, cols + pad)[:, :cols]
    view.copy_((torch.randn(rows, cols, generator=g, device="cuda") * size).to(DTYPE[kind]))
    return view, whole


def mat(api, view):
    return api.DnMat(view, view.shape[0], view.shape[1], view.stride(0))


def outside(view, whole):
    """The elements of `whole` that do not belong to the view."""
    mine = torch.zeros(whole.numel(), dtype=torch.bool, device="cuda")
    first = (view.data_ptr() - whole.data_ptr()) // whole.element_size()
    index = first + torch.arange(view.shape[0], device="cuda")[:, None] * view.stride(0) + torch.arange(view.shape[1], device="cuda")
    mine[index.flatten()] = True
    return whole[~mine]


def words(g, count, vocab, index, skew):
    u = torch.rand(count, generator=g, device="cuda", dtype=torch.float64)
    t = (vocab * u ** (1 + 4 * skew)).long().clamp(max=vocab - 1)
    wild = torch.rand(count, generator=g, device="cuda") < 0.1
    far = torch.tensor([-1, vocab, -vocab - 7, 2 ** 31 - 1] + ([2 ** 40, -2 ** 40 + 1, 2 ** 32] if index == torch.int64 else []), device="cuda")
    t = torch.where(wild, far[torch.randint(len(far), (count,), generator=g, device="cuda")], t)
    return t.to(index)


EMBEDDING = [  # count, vocab, width, table, out, index, alpha, beta, pad, shift
    (1, 1, 1, "f32", "f32", torch.int32, 1.0, 0.0, 0, 0),
    (1, 50, 4096, "bf16", "bf16", torch.int64, 1.0, 0.0, 0, 0),
    (3, 1000, 8, "bf16", "bf16", torch.int32, 3.0, 0.0, 0, 0),
    (37, 500, 24, "f16", "f16", torch.int64, 1.0, 1.0, 8, 0),
    (1001, 333, 777, "f32", "f32", torch.int64, 0.5, 0.0, 0, 0),
    (513, 333, 777, "bf16", "f32", torch.int32, 64.0, 0.5, 3, 1),
    (260, 700, 1032, "f32", "bf16", torch.int64, 2.0, -1.0, 0, 0),
    (260, 700, 1030, "f16", "f32", torch.int64, 2.0, 0.0, 2, 0),  # aligned rows whose end is not a whole vector
    (4100, 129, 65, "f16", "bf16", torch.int32, 1.0, 0.0, 0, 3),
    (70000, 300, 32, "bf16", "bf16", torch.int32, 1.5, 0.0, 0, 8),
]


@pytest.mark.parametrize("count,vocab,width,table,out,index,alpha,beta,pad,shift", EMBEDDING)
def test_embedding(pkg, handle, count, vocab, width, table, out, index, alpha, beta, pad, shift):
    from ops_sparse_b200 import api
    g = gen(count + width)
    t, _ = matrix(g, vocab, width, table, pad, shift)
    o, whole = matrix(g, count, width, out, pad, shift)
    if beta == 0:
        o.fill_(math.nan)  # must not be read
    tokens = words(g, count, vocab, index, 0.5)
    want = ref.embedding(t, tokens, alpha, beta, o)
    size = want.abs() + (2 * abs(beta) * o.double().abs().cpu() if beta else 0)
    kept = outside(o, whole).clone()
    api.embedding(handle, mat(api, t), api.DnVec(tokens), mat(api, o), alpha, beta)
    torch.cuda.synchronize()
    ref.close(o, want, ref.rounding(o.dtype, want) + 2 * F32 * size)  # two operations in f32, one rounding
    assert torch.equal(outside(o, whole), kept)


def test_embedding_overflow_and_special_values(pkg, handle):
    from ops_sparse_b200 import api
    t = torch.tensor([[1e4, -1e4, math.inf, math.nan, 0.0, -0.0, 6e-8, 1.0]], device="cuda").half()
    out = torch.empty(1, 8, dtype=torch.float16, device="cuda")
    api.embedding(handle, mat(api, t), api.DnVec(torch.zeros(1, dtype=torch.int32, device="cuda")), mat(api, out), alpha=10.0)
    assert out[0, :3].tolist() == [math.inf, -math.inf, math.inf] and out[0, 3].isnan()
    assert out[0, 4:].tolist() == [0.0, -0.0, 10 * 2.0 ** -24, 10.0]


GRADIENT = [  # count, vocab, width, grad, table, index, alpha, beta, pad, shift, skew
    (1, 1, 1, "f32", "f32", torch.int32, 1.0, 0.0, 0, 0, 0),
    (1, 5000, 64, "bf16", "bf16", torch.int64, 2.0, 0.0, 0, 0, 0),
    (9, 40, 30, "f16", "f32", torch.int32, 1.0, 1.0, 2, 0, 0),
    (509, 1007, 777, "f32", "f32", torch.int64, 0.5, 0.0, 0, 0, 0.5),
    (700, 3, 40, "bf16", "f32", torch.int64, 1.0, 0.5, 0, 0, 0),  # runs of many pieces
    (2049, 1, 130, "f16", "f16", torch.int32, 0.01, 0.0, 6, 0, 0),  # one token
    (4096, 3000, 256, "bf16", "bf16", torch.int64, 1.0, -0.5, 0, 0, 1),
    (5000, 65536, 72, "bf16", "f32", torch.int32, 1.0, 0.0, 0, 0, 1),
    (9001, 131072, 17, "f32", "bf16", torch.int64, 1.0, 1.0, 1, 1, 1),
    (20000, 1500000, 4, "f32", "f32", torch.int64, 1.0, 0.0, 0, 0, 0.5),  # three passes of the sort
    (70001, 1023, 8, "f16", "f32", torch.int32, 1.0, 0.0, 0, 0, 1),
    (70001, 1024, 8, "bf16", "f32", torch.int32, 1.0, 0.0, 0, 0, 1),  # the first table that takes two
    (4096, 2 ** 19 + 1, 3, "f32", "f32", torch.int32, 1.0, 0.0, 0, 0, 0),  # a tile's worth in three passes
    (3000, 40000, 512, "bf16", "f32", torch.int64, 1.0, 0.0, 0, 0, 0.5),  # zeros in two kernels
    (3000, 40000, 513, "f16", "f32", torch.int64, 2.0, 0.0, 2, 1, 0.5),
    (300, 40000, 1030, "f32", "f16", torch.int32, 1.0, 0.5, 2, 0, 0.5),
]


@pytest.mark.parametrize("count,vocab,width,grad,table,index,alpha,beta,pad,shift,skew", GRADIENT)
def test_embedding_gradient(pkg, handle, count, vocab, width, grad, table, index, alpha, beta, pad, shift, skew):
    from ops_sparse_b200 import api
    g = gen(count + vocab)
    d, _ = matrix(g, count, width, grad, pad, shift)
    t, whole = matrix(g, vocab, width, table, pad, shift)
    tokens = words(g, count, vocab, index, skew)
    want, size, many = ref.embedding_grad(d, tokens, vocab, alpha, beta, t)
    if beta == 0:
        t.fill_(math.nan)
    kept, old = outside(t, whole).clone(), t.clone()
    D, K, T = mat(api, d), api.DnVec(tokens), mat(api, t)
    buffer = torch.full((api.embedding_grad_buffer_size(handle, D, K, T),), 255, dtype=torch.uint8, device="cuda")
    api.embedding_grad(handle, D, K, T, alpha, beta, buffer=buffer)
    torch.cuda.synchronize()
    ref.close(t, want, ref.rounding(t.dtype, want) + (many + 2) * F32 * size)
    assert torch.equal(outside(t, whole), kept)
    first = t.clone()
    t.copy_(old)
    api.embedding_grad(handle, D, K, T, alpha, beta)  # a buffer of its own
    torch.cuda.synchronize()
    assert torch.equal(t.nan_to_num(), first.nan_to_num())  # the same bits in every run


def test_embedding_gradient_without_tokens_of_the_table(pkg, handle):
    from ops_sparse_b200 import api
    d = torch.ones(100, 16, device="cuda")
    for beta, value in ((0.0, 0.0), (1.0, 3.0), (0.5, 1.5)):
        t = torch.full((50, 16), 3.0, device="cuda")
        api.embedding_grad(handle, mat(api, d), api.DnVec(torch.full((100,), -1, device="cuda")), mat(api, t), beta=beta)
        assert (t == value).all()


def test_embedding_gradient_leaves_other_rows_with_beta_one(pkg, handle):
    """beta = 1: rows of tokens that do not occur keep their bits, NaN among them."""
    from ops_sparse_b200 import api
    t = torch.full((1000, 64), math.nan, dtype=torch.bfloat16, device="cuda")
    t[7], t[9] = 1.0, 2.0
    d = torch.ones(3, 64, dtype=torch.bfloat16, device="cuda")
    api.embedding_grad(handle, mat(api, d), api.DnVec(torch.tensor([7, 9, 7], device="cuda")), mat(api, t), beta=1.0)
    assert (t[7] == 3).all() and (t[9] == 3).all() and t.isnan().sum() == 998 * 64


def test_embedding_gradient_is_the_adjoint(pkg, handle):
    """<embedding(table), d> = <table, gradient(d)>: differences of a linear function."""
    from ops_sparse_b200 import api
    g = gen(3)
    tokens = torch.randint(0, 500, (2000,), generator=g, device="cuda")
    table, d = torch.randn(500, 96, generator=g, device="cuda"), torch.randn(2000, 96, generator=g, device="cuda")
    out, grad = torch.empty_like(d), torch.empty_like(table)
    api.embedding(handle, mat(api, table), api.DnVec(tokens), mat(api, out), alpha=1.5)
    api.embedding_grad(handle, mat(api, d), api.DnVec(tokens), mat(api, grad), alpha=1.5)
    left, right = (out.double() * d.double()).sum(), (table.double() * grad.double()).sum()
    size = (out.double() * d.double()).abs().sum()
    assert abs(left - right) <= 2000 * F32 * size


# ---------------------------------------------------------------- routing

def routed(api, tokens, experts, k, kind="f32"):
    offsets = torch.full((tokens + 1,), -5, dtype=torch.int32, device="cuda")
    columns = torch.full((tokens * k,), -7, dtype=torch.int32, device="cuda")
    values = torch.full((tokens * k,), math.nan, dtype=DTYPE[kind], device="cuda")
    return api.CsrMatrix(offsets, columns, values, tokens, experts)


def check_route(api, handle, x, bias, k, kind="f32", **rule):
    R = routed(api, x.shape[0], x.shape[1], k, kind)
    api.route(handle, api.RouteRule(**rule), mat(api, x), None if bias is None else api.DnVec(bias), R)
    torch.cuda.synchronize()
    columns, weights = ref.route(x, bias, k, **rule)
    assert torch.equal(R.row_ptr.cpu(), torch.arange(0, x.shape[0] * k + 1, k, dtype=torch.int32))
    got = R.col_ind.view(-1, k).cpu()
    assert torch.equal(got, columns), (got != columns).any(1).nonzero()[:4]
    # exp and division to two units each, sums of 1024 terms by lanes and halves (37 additions), the sum of the k, two products;
    # exp of a difference of up to 100 loses 100 * 2^-24
    bound = ref.rounding(R.values.dtype, weights) + weights.abs() * (37 + 100 + k + 12) * F32
    ref.close(R.values.view(-1, k), weights, bound.clamp_min(1e-37))
    return R


ROUTES = [  # tokens, experts, k, x, value, rule, bias
    (1, 1, 1, "f32", "f32", {}, False),
    (1, 64, 8, "bf16", "f32", {}, False),
    (5, 7, 7, "f16", "f16", {"renormalise": False}, False),
    (33, 60, 6, "f32", "bf16", {"score": "sigmoid", "scale": 2.5}, True),
    (130, 32, 1, "bf16", "f32", {"score": "sigmoid"}, True),
    (500, 33, 32, "f32", "f32", {"renormalise": False, "scale": -1.5}, False),
    (300, 128, 4, "bf16", "bf16", {"groups": 8, "kept": 3, "group_score": "max"}, False),
    (300, 256, 8, "f32", "f32", {"score": "sigmoid", "groups": 8, "kept": 4, "group_score": "top2", "scale": 2.5}, True),
    (300, 160, 6, "f32", "f32", {"groups": 8, "kept": 3, "group_score": "max", "renormalise": False, "scale": 16.0}, False),
    (200, 96, 5, "f16", "f32", {"groups": 32, "kept": 5, "group_score": "top2"}, True),
    (200, 36, 4, "f32", "f32", {"groups": 12, "kept": 11, "group_score": "top2"}, False),
    (100, 300, 10, "bf16", "f32", {"score": "sigmoid"}, False),
    (64, 513, 16, "f32", "f32", {"renormalise": False}, True),
    (40, 1024, 32, "bf16", "f32", {"groups": 16, "kept": 2, "group_score": "top2", "score": "sigmoid"}, True),
    (9, 1000, 3, "f32", "f16", {}, True),
]


@pytest.mark.parametrize("tokens,experts,k,x,value,rule,bias", ROUTES)
def test_route(pkg, handle, tokens, experts, k, x, value, rule, bias):
    from ops_sparse_b200 import api
    g = gen(tokens * experts)
    logits, _ = matrix(g, tokens, experts, x, pad=tokens % 3, size=1.5)
    b = 0.2 * torch.randn(experts, generator=g, device="cuda") if bias else None
    check_route(api, handle, logits, b, k, value, **rule)


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 4])
def test_route_ties_and_masks(pkg, handle, bias, score, groups):
    """Few different logits, -0 and 0 among them; masked ones, whole rows of them, infinities, NaN; masked biases."""
    from ops_sparse_b200 import api
    g = gen(17)
    x = torch.randint(-2, 3, (400, 24), generator=g, device="cuda").float() * 0.5
    x[x == 0] *= torch.where(torch.rand(int((x == 0).sum()), generator=g, device="cuda") < 0.5, -1.0, 1.0)
    x[100:200][torch.rand(100, 24, generator=g, device="cuda") < 0.85] = -math.inf
    x[200:240] = -math.inf
    x[240:280][torch.rand(40, 24, generator=g, device="cuda") < 0.2] = math.nan
    x[280:320][torch.rand(40, 24, generator=g, device="cuda") < 0.2] = torch.finfo(torch.float32).min
    x[320:330] = math.nan
    if not bias:
        x[330:360][torch.rand(30, 24, generator=g, device="cuda") < 0.2] = math.inf
    b = None
    if bias:
        b = torch.randint(-1, 2, (24,), generator=g, device="cuda").float() * 0.25
        b[3], b[11] = -math.inf, math.nan
    for group_score in ("max", "top2"):
        for renormalise in (True, False):
            check_route(api, handle, x, b, 5, score=score, groups=groups, kept=(groups + 1) // 2, group_score=group_score, renormalise=renormalise)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,group_score", [(1, "max"), (4, "max"), (4, "top2")])
def test_route_neighbours_closer_than_f32(pkg, handle, score, groups, group_score):
    """Selection values that f32 rounds to one another: p + bias is put within 1e-8 of a few levels."""
    from ops_sparse_b200 import api
    g = gen(23)
    x = torch.randn(256, 32, generator=g, device="cuda")
    x[1:] = x[:1] + 2e-7 * torch.randn(255, 32, generator=g, device="cuda")
    p = torch.softmax(x[0].double(), 0) if score == "softmax" else torch.sigmoid(x[0].double())
    level = 0.25 * torch.randint(1, 3, (32,), generator=g, device="cuda").double()
    bias = (level - p).float()
    check_route(api, handle, x, bias, 6, score=score, groups=groups, kept=max(groups // 2, 1), group_score=group_score)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalise", [True, False])
@pytest.mark.parametrize("tokens,experts,k,x,value,grad", [(1, 64, 8, "bf16", "f32", "f32"), (70, 60, 6, "f32", "f32", "f32"),
                                                           (33, 7, 7, "f16", "f16", "bf16"), (200, 256, 1, "bf16", "bf16", "f16"),
                                                           (20, 1024, 32, "f32", "f32", "f32"), (9, 1, 1, "f32", "f32", "f32")])
def test_route_gradient(pkg, handle, score, renormalise, tokens, experts, k, x, value, grad):
    from ops_sparse_b200 import api
    g = gen(tokens + experts)
    logits, _ = matrix(g, tokens, experts, x, pad=1, size=1.5)
    rule = {"score": score, "renormalise": renormalise, "scale": 1.5}
    R = check_route(api, handle, logits, None, k, value, **rule)
    d = torch.randn(tokens * k, generator=g, device="cuda").to(DTYPE[grad])
    out, whole = matrix(g, tokens, experts, x, pad=3)
    kept = outside(out, whole).clone()
    api.route_grad(handle, api.RouteRule(**rule), mat(api, logits), R, api.DnVec(d), mat(api, out))
    torch.cuda.synchronize()
    leaf = logits.double().cpu().requires_grad_()
    w = ref.route_weights(leaf, R.col_ind.view(tokens, k).cpu(), score, renormalise, 1.5)
    want = torch.autograd.grad((w * d.double().cpu().view(tokens, k)).sum(), leaf)[0]
    # the terms of a row: scale * q * (|g| + sum |g| q), each with the errors of q (see check_route) and k more additions
    p = torch.softmax(leaf.detach(), 1) if score == "softmax" else torch.sigmoid(leaf.detach())
    q = p.gather(1, R.col_ind.view(tokens, k).cpu().long())
    most = d.double().cpu().view(tokens, k).abs().amax(1, keepdim=True)
    size = 1.5 * 2 * most * (p / (q.sum(1, keepdim=True) if renormalise else 1))
    ref.close(out, want, ref.rounding(out.dtype, want) + size * (2 * (37 + 100 + k) + 24) * F32)
    assert torch.equal(outside(out, whole), kept)
    # in place, and the same bits
    api.route_grad(handle, api.RouteRule(**rule), mat(api, logits), R, api.DnVec(d), mat(api, logits))
    torch.cuda.synchronize()
    assert torch.equal(logits, out)


def test_route_gradient_by_differences(pkg, handle):
    from ops_sparse_b200 import api
    g = gen(5)
    for score in ("softmax", "sigmoid"):
        for renormalise in (True, False):
            rule = api.RouteRule(score=score, renormalise=renormalise, scale=2.0)
            x = torch.randn(4, 12, generator=g, device="cuda")
            x[:, :4] += 4.0  # the same experts whatever the small steps
            d = torch.randn(16, generator=g, device="cuda")
            R = routed(api, 4, 12, 4)
            api.route(handle, rule, mat(api, x), None, R)
            out = torch.empty_like(x)
            api.route_grad(handle, rule, mat(api, x), R, api.DnVec(d), mat(api, out))
            for e in (0, 2, 7):
                value = []
                for step in (0.0625, -0.0625):
                    y = x.clone()
                    y[:, e] += step
                    S = routed(api, 4, 12, 4)
                    api.route(handle, rule, mat(api, y), None, S)
                    value.append((S.values.double() * d.double()).view(4, 4).sum(1))
                slope = (value[0] - value[1]) / 0.125
                # a central difference is off by step^2 / 6 of the third derivative: at most 2 * sum |d| * 1 here
                assert ((slope - out[:, e].double()).abs() <= 0.0625 ** 2 / 6 * 2 * d.abs().sum() + 1e-5).all()


def test_route_gradient_of_masked_entries(pkg, handle):
    """Rows with fewer experts than entries: what stands for nothing has weight 0 and no gradient."""
    from ops_sparse_b200 import api
    x = torch.full((3, 8), -math.inf, device="cuda")
    x[0, 5], x[1, 2], x[1, 6] = 1.0, 0.5, -0.5
    for score in ("softmax", "sigmoid"):
        for renormalise in (True, False):
            rule = {"score": score, "renormalise": renormalise}
            R = check_route(api, handle, x, None, 4, **rule)
            d, out = torch.randn(12, device="cuda"), torch.full_like(x, math.nan)
            api.route_grad(handle, api.RouteRule(**rule), mat(api, x), R, api.DnVec(d), mat(api, out))
            assert out.isfinite().all() and (out[2] == 0).all() and (out[x == -math.inf] == 0).all()


# ---------------------------------------------------------------- experts

def ragged(g, tokens, experts, mean, wild=0.1, among=None):
    """Any CSR matrix: rows of 0 to 2 * mean entries, some of them of no expert, some experts without entries."""
    lengths = torch.randint(0, 2 * mean + 1, (tokens,), generator=g, device="cuda")
    lengths[0] += 1
    offsets = torch.zeros(tokens + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = lengths.cumsum(0)
    nnz = int(offsets[-1])
    columns = torch.randint(0, among or experts, (nnz,), generator=g, device="cuda", dtype=torch.int32)
    far = torch.tensor([-1, experts, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")
    columns = torch.where(torch.rand(nnz, generator=g, device="cuda") < wild, far[torch.randint(4, (nnz,), generator=g, device="cuda")], columns)
    return offsets, columns


PRODUCTS = [  # tokens, experts, mean, n, d, type, out, transpose, rows, alpha, beta, pad, shift
    (1, 1, 1, 1, 1, "bf16", "bf16", True, "tokens", 1.0, 0.0, 0, 0),
    (1, 8, 2, 64, 128, "bf16", "bf16", True, "tokens", 1.0, 0.0, 0, 0),
    (3, 4, 2, 200, 72, "f16", "f16", True, "tokens", 1.0, 0.0, 0, 0),
    (40, 8, 2, 128, 64, "bf16", "f32", True, "tokens", 0.5, 0.0, 0, 0),
    (40, 8, 2, 128, 64, "bf16", "bf16", False, "entries", 1.0, 0.0, 0, 0),
    (300, 5, 3, 136, 200, "f16", "f32", True, "entries", 1.0, 0.5, 8, 0),
    (300, 5, 3, 136, 200, "f16", "f16", False, "tokens", 1.0, 1.0, 8, 8),
    (257, 17, 3, 77, 53, "bf16", "bf16", True, "tokens", 1.0, 0.0, 0, 0),  # odd rows
    (257, 17, 3, 77, 53, "bf16", "f32", False, "entries", 2.0, -1.0, 3, 1),
    (129, 3, 2, 260, 1000, "bf16", "bf16", True, "tokens", 1.0, 0.0, 0, 0),
    (900, 2, 2, 520, 264, "f16", "f16", False, "entries", 1.0, 0.0, 0, 0),
    (700, 40, 4, 96, 320, "bf16", "bf16", True, "tokens", 1.0, 0.0, 0, 0),
    (64, 1024, 3, 24, 40, "bf16", "bf16", True, "tokens", 1.0, 0.0, 0, 0),  # two passes of the sort
    (30, 300, 2, 40, 2056, "f16", "f16", True, "tokens", 1.0, 0.0, 0, 0),
    (5000, 4, 2, 40, 64, "bf16", "bf16", True, "tokens", 1.0, 0.0, 0, 0),
    (1, 5, 3, 1024, 2048, "bf16", "bf16", True, "tokens", 1.0, 0.0, 0, 0),
    (20, 64, 4, 256, 1024, "f16", "f16", True, "tokens", 1.0, 0.0, 0, 0),
    (3000, 6, 3, 1100, 600, "bf16", "bf16", True, "tokens", 1.0, 0.0, 4, 0),  # every CTA has several tiles
    (3000, 6, 3, 1100, 600, "bf16", "f32", False, "entries", 1.0, 0.0, 4, 0),
    (3000, 6, 3, 1100, 600, "f16", "f16", False, "tokens", 1.0, 1.0, 0, 0),
    (2500, 33, 4, 128, 1000, "bf16", "bf16", True, "entries", 1.0, 0.0, 0, 0),  # one CTA a tile of 256 entries
]


@pytest.mark.parametrize("tokens,experts,mean,n,d,kind,out,transpose,rows,alpha,beta,pad,shift", PRODUCTS)
def test_experts_product(pkg, handle, tokens, experts, mean, n, d, kind, out, transpose, rows, alpha, beta, pad, shift):
    from ops_sparse_b200 import api
    g = gen(tokens + n)
    offsets, columns = ragged(g, tokens, experts, mean, among=max(1, experts * 3 // 4))
    nnz = len(columns)
    depth, width = (d, n) if transpose else (n, d)
    x, _ = matrix(g, tokens if rows == "tokens" else nnz, depth, kind, pad, shift)
    w, _ = matrix(g, experts * n, d, kind, pad, shift, size=1 / math.sqrt(depth))
    y, whole = matrix(g, nnz, width, out, pad, shift)
    want, size = ref.experts_mm(offsets, columns, x, w.reshape(experts, n, d), experts, transpose, rows == "entries", alpha, beta, y)
    if beta == 0:
        y.fill_(math.nan)
    kept = outside(y, whole).clone()
    R = api.CsrMatrix(offsets, columns, torch.empty(nnz, device="cuda"), tokens, experts)
    X, W, Y = mat(api, x), mat(api, w), mat(api, y)
    buffer = torch.full((api.experts_buffer_size(handle, R, X, W, Y, transpose, rows),), 255, dtype=torch.uint8, device="cuda")
    api.experts_preprocess(handle, R, buffer)
    old = y.clone()
    api.experts_mm(handle, R, X, W, Y, alpha, beta, transpose, rows, buffer)
    torch.cuda.synchronize()
    # products of 16-bit values are exact in f32; additions of the tensor cores may drop what is below 2^-23 of the sum
    ref.close(y, want, ref.rounding(y.dtype, want) + size * (depth + 4) * 2 * F32)
    assert torch.equal(outside(y, whole), kept)
    first = y.clone()
    y.copy_(old)
    api.experts_mm(handle, R, X, W, Y, alpha, beta, transpose, rows, buffer)
    torch.cuda.synchronize()
    assert torch.equal(y, first)


GRADIENTS = [  # tokens, experts, mean, n, d, type, out, rows, alpha, beta, pad, shift
    (1, 1, 1, 1, 1, "f16", "f16", "tokens", 1.0, 0.0, 0, 0),
    (3, 8, 2, 64, 128, "bf16", "bf16", "tokens", 1.0, 0.0, 0, 0),
    (40, 8, 2, 200, 72, "f16", "f32", "entries", 0.5, 0.0, 0, 0),
    (300, 5, 3, 136, 264, "bf16", "bf16", "tokens", 1.0, 0.5, 8, 8),
    (257, 17, 3, 77, 53, "bf16", "f32", "tokens", 1.0, 1.0, 3, 1),
    (1003, 6, 3, 520, 100, "f16", "f16", "tokens", 1.0, 0.0, 0, 0),
    (900, 3, 4, 24, 600, "bf16", "bf16", "entries", 1.0, 0.0, 0, 0),
    (64, 1024, 3, 24, 40, "bf16", "bf16", "tokens", 1.0, 0.0, 0, 0),
    (5000, 2, 2, 40, 64, "f16", "f16", "tokens", 0.1, 0.0, 0, 0),
    (3000, 6, 3, 1100, 600, "bf16", "bf16", "tokens", 1.0, 0.0, 4, 0),
    (2000, 40, 3, 300, 1032, "bf16", "f32", "entries", 1.0, 0.0, 0, 0),
]


@pytest.mark.parametrize("tokens,experts,mean,n,d,kind,out,rows,alpha,beta,pad,shift", GRADIENTS)
def test_experts_gradient(pkg, handle, tokens, experts, mean, n, d, kind, out, rows, alpha, beta, pad, shift):
    from ops_sparse_b200 import api
    g = gen(tokens + d)
    offsets, columns = ragged(g, tokens, experts, mean, among=max(1, experts * 3 // 4))
    nnz = len(columns)
    x, _ = matrix(g, tokens if rows == "tokens" else nnz, d, kind, pad, shift)
    dy, _ = matrix(g, nnz, n, kind, pad, shift)
    dw, whole = matrix(g, experts * n, d, out, pad, shift)
    want, size, many = ref.experts_grad(offsets, columns, dy, x, experts, rows == "entries", alpha, beta, dw.reshape(experts, n, d))
    if beta == 0:
        dw.fill_(math.nan)
    kept, old = outside(dw, whole).clone(), dw.clone()
    R = api.CsrMatrix(offsets, columns, torch.empty(nnz, device="cuda"), tokens, experts)
    DY, X, DW = mat(api, dy), mat(api, x), mat(api, dw)
    buffer = torch.full((api.experts_grad_buffer_size(handle, R, DY, X, DW, rows),), 255, dtype=torch.uint8, device="cuda")
    api.experts_preprocess(handle, R, buffer)
    api.experts_grad(handle, R, DY, X, DW, alpha, beta, rows, buffer)
    torch.cuda.synchronize()
    ref.close(dw.reshape(experts, n, d), want, ref.rounding(dw.dtype, want) + size * (many + 4) * 2 * F32)
    assert torch.equal(outside(dw, whole), kept)
    first = dw.clone()
    dw.copy_(old)
    api.experts_grad(handle, R, DY, X, DW, alpha, beta, rows, buffer)
    torch.cuda.synchronize()
    assert torch.equal(dw, first)


def test_experts_keep_their_neighbours_infinities(pkg, handle):
    """NaN and infinities of a token reach its own rows only, those of an expert its own entries only, though tiles hold
    rows of both: also past the last row and column of an expert's matrix."""
    from ops_sparse_b200 import api
    g = gen(8)
    tokens, experts, n, d = 90, 4, 72, 40
    offsets = torch.arange(0, 2 * tokens + 1, 2, dtype=torch.int32, device="cuda")
    columns = torch.randint(0, experts, (2 * tokens,), generator=g, device="cuda", dtype=torch.int32)
    x, _ = matrix(g, tokens, d, "bf16")
    w, _ = matrix(g, experts * n, d, "bf16")
    dy, _ = matrix(g, 2 * tokens, n, "bf16")
    x[5], x[77, 3] = math.nan, math.inf
    w[n:2 * n] = math.nan
    dy[11] = math.inf
    R = api.CsrMatrix(offsets, columns, torch.empty(2 * tokens, device="cuda"), tokens, experts)
    y, dx, dw = (torch.zeros(s, dtype=torch.bfloat16, device="cuda") for s in ((2 * tokens, n), (2 * tokens, d), (experts * n, d)))
    X, W, Y, DY, DX, DW = (mat(api, t) for t in (x, w, y, dy, dx, dw))
    buffer = torch.empty(max(api.experts_buffer_size(handle, R, X, W, Y), api.experts_buffer_size(handle, R, DY, W, DX, False, "entries"),
                             api.experts_grad_buffer_size(handle, R, DY, X, DW)), dtype=torch.uint8, device="cuda")
    api.experts_preprocess(handle, R, buffer)
    api.experts_mm(handle, R, X, W, Y, buffer=buffer)
    api.experts_mm(handle, R, DY, W, DX, transpose=False, rows="entries", buffer=buffer)
    api.experts_grad(handle, R, DY, X, DW, buffer=buffer)
    token, one = torch.arange(2 * tokens, device="cuda") // 2, columns == 1
    assert torch.equal(~y.isfinite().all(1), one | (token == 5) | (token == 77))
    assert torch.equal(~dx.isfinite().all(1), one | (torch.arange(2 * tokens, device="cuda") == 11))
    hit = torch.zeros(experts, dtype=torch.bool, device="cuda")
    hit[columns[(token == 5) | (token == 77)].long()] = True
    hit[columns[11].long()] = True
    assert torch.equal(~dw.view(experts, -1).isfinite().all(1), hit)


def test_a_captured_order_is_none_until_it_is_replayed(pkg, device):
    """Preprocess in a graph, a product outside of it: before the first replay there is nothing to follow, whatever the buffer holds."""
    from ops_sparse_b200 import api
    L = pkg.lib()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        h = api.Handle(stream)
        g = gen(12)
        offsets, columns = ragged(g, 60, 5, 2)
        nnz = len(columns)
        x, w = matrix(g, 60, 64, "bf16")[0], matrix(g, 5 * 136, 64, "bf16")[0]
        y, dw = torch.full((nnz, 136), 5.0, dtype=torch.bfloat16, device="cuda"), torch.full((5 * 136, 64), 5.0, dtype=torch.bfloat16, device="cuda")
        R = api.CsrMatrix(offsets, columns, torch.empty(nnz, device="cuda"), 60, 5)
        X, W, Y, DW = mat(api, x), mat(api, w), mat(api, y), mat(api, dw)
        size = max(api.experts_buffer_size(h, R, X, W, Y), api.experts_grad_buffer_size(h, R, Y, X, DW))
        buffer = torch.full((size,), 127, dtype=torch.uint8, device="cuda")
        graph = torch.cuda.CUDAGraph()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            api.experts_preprocess(h, R, buffer)
        for call in (lambda: api.experts_mm(h, R, X, W, Y, buffer=buffer), lambda: api.experts_grad(h, R, Y, X, DW, buffer=buffer)):
            call()
            stream.synchronize()
            assert L.b200sp_experts_error() == 2 and L.b200sp_experts_error_clear() == 0
        assert (y == 5).all() and (dw == 5).all()
        graph.replay()
        api.experts_mm(h, R, X, W, Y, buffer=buffer)
        stream.synchronize()
        assert L.b200sp_experts_error() == 0
        want, size = ref.experts_mm(offsets, columns, x, w.view(5, 136, 64), 5, True, False, 1.0, 0.0, y)
        ref.close(y, want, ref.rounding(y.dtype, want) + size * 68 * 2 * F32)
        del graph
    h.close()


def test_products_refuse_a_buffer_sized_for_other_operands(pkg, handle):
    """Room for the copy of an operand that starts on no multiple of 16 bytes has to have been asked for."""
    from ops_sparse_b200 import api
    g = gen(6)
    offsets, columns = ragged(g, 20, 4, 2)
    nnz = len(columns)
    R = api.CsrMatrix(offsets, columns, torch.empty(nnz, device="cuda"), 20, 4)
    X, W, Y = mat(api, matrix(g, 20, 32, "bf16")[0]), mat(api, matrix(g, 64, 32, "bf16")[0]), mat(api, torch.empty(nnz, 16, dtype=torch.bfloat16, device="cuda"))
    odd = mat(api, matrix(g, 20, 32, "bf16", shift=1)[0])
    buffer = torch.empty(api.experts_buffer_size(handle, R, X, W, Y) + 20 * 32 * 2 + 256, dtype=torch.uint8, device="cuda")
    api.experts_preprocess(handle, R, buffer)
    api.experts_mm(handle, R, X, W, Y, buffer=buffer)
    with pytest.raises(pkg.AclSparseError, match="INVALID_VALUE"):
        api.experts_mm(handle, R, odd, W, Y, buffer=buffer)
    assert api.experts_buffer_size(handle, R, odd, W, Y) <= buffer.numel()
    api.experts_mm(handle, R, odd, W, Y, buffer=buffer)
    torch.cuda.synchronize()


def test_products_want_the_order_in_their_buffer(pkg, handle):
    from ops_sparse_b200 import api
    g = gen(1)
    offsets, columns = ragged(g, 20, 4, 2)
    nnz = len(columns)
    x, w = matrix(g, 20, 32, "bf16")[0], matrix(g, 4 * 16, 32, "bf16")[0]
    y = torch.empty(nnz, 16, dtype=torch.bfloat16, device="cuda")
    R = api.CsrMatrix(offsets, columns, torch.empty(nnz, device="cuda"), 20, 4)
    other = api.CsrMatrix(offsets, columns, torch.empty(nnz, device="cuda"), 20, 4)
    args = mat(api, x), mat(api, w), mat(api, y)
    buffer = torch.empty(api.experts_buffer_size(handle, R, *args), dtype=torch.uint8, device="cuda")
    with pytest.raises(pkg.AclSparseError, match="INVALID_VALUE"):
        api.experts_mm(handle, R, *args, buffer=buffer)
    api.experts_preprocess(handle, R, buffer)
    api.experts_mm(handle, R, *args, buffer=buffer)
    with pytest.raises(pkg.AclSparseError, match="INVALID_VALUE"):
        api.experts_mm(handle, other, *args, buffer=buffer)
    api.experts_preprocess(handle, other, buffer)  # the buffer holds the other's now
    with pytest.raises(pkg.AclSparseError, match="INVALID_VALUE"):
        api.experts_mm(handle, R, *args, buffer=buffer)
    with pytest.raises(pkg.AclSparseError, match="INVALID_VALUE"):
        api.experts_mm(handle, R, *args, buffer=buffer.clone())
    with pytest.raises(pkg.AclSparseError, match="INSUFFICIENT_RESOURCES"):
        api.experts_mm(handle, R, *args)
    torch.cuda.synchronize()


# ---------------------------------------------------------------- together

class Layer:
    """A table, a router and two layers of experts, in the order in which a model calls them, every operand a buffer of
    its own.  The rows of a token's experts are summed by aclsparseSpMM with the routing weights, whose gradient
    is aclsparseSDDMM's."""

    def __init__(self, pkg, handle, tokens=96, vocab=500, width=64, hidden=80, experts=12, k=3, seed=0):
        from ops_sparse_b200 import api
        self.api, self.h, self.pkg = api, handle, pkg
        self.sizes = tokens, vocab, width, hidden, experts, k
        g = gen(seed)
        new = lambda *s, t=torch.float16: torch.zeros(s, dtype=t, device="cuda")  # noqa: E731
        self.tokens = torch.randint(0, vocab, (tokens,), generator=g, device="cuda")
        self.table = matrix(g, vocab, width, "f16")[0]
        self.gate = matrix(g, experts, width, "f32", size=0.2)[0]
        self.w1, self.w2 = matrix(g, experts * hidden, width, "f16", size=0.1)[0], matrix(g, experts * width, hidden, "f16", size=0.1)[0]
        self.dout = matrix(g, tokens, width, "f16")[0]
        self.x, self.logits = new(tokens, width), new(tokens, experts, t=torch.float32)
        self.hid, self.y, self.out = new(tokens * k, hidden), new(tokens * k, width), new(tokens, width)
        self.rule = api.RouteRule(score="sigmoid", scale=2.0)
        self.R = routed(api, tokens, experts, k, "f16")
        self.combine = api.CsrMatrix(self.R.row_ptr, torch.arange(tokens * k, dtype=torch.int32, device="cuda"), self.R.values, tokens, tokens * k)
        self.spread = api.CsrMatrix(torch.arange(tokens * k + 1, dtype=torch.int32, device="cuda"),
                                    (torch.arange(tokens * k, device="cuda") // k).int(), self.R.values, tokens * k, tokens)
        self.sum = api.CsrMatrix(self.R.row_ptr, self.combine.col_ind, torch.ones(tokens * k, dtype=torch.float16, device="cuda"), tokens, tokens * k)
        self.dy, self.dhid, self.dxe, self.dx = new(tokens * k, width), new(tokens * k, hidden), new(tokens * k, width), new(tokens, width)
        self.dw1, self.dw2, self.dtable = (new(*t.shape, t=torch.float32) for t in (self.w1, self.w2, self.table))
        self.dvalues, self.dlogits = new(tokens * k), new(tokens, experts, t=torch.float32)
        self.dR = api.CsrMatrix(self.R.row_ptr, self.combine.col_ind, self.dvalues, tokens, tokens * k)
        self.m = {n: mat(api, getattr(self, n)) for n in ("table", "w1", "w2", "dout", "x", "logits", "hid", "y", "out", "dy", "dhid", "dxe", "dx",
                                                          "dw1", "dw2", "dtable", "dlogits")}
        self.words = api.DnVec(self.tokens)
        m = self.m
        self.buffer = torch.empty(max(api.experts_buffer_size(handle, self.R, m["x"], m["w1"], m["hid"]),
                                      api.experts_buffer_size(handle, self.R, m["hid"], m["w2"], m["y"], rows="entries"),
                                      api.experts_buffer_size(handle, self.R, m["dy"], m["w2"], m["dhid"], False, "entries"),
                                      api.experts_buffer_size(handle, self.R, m["dhid"], m["w1"], m["dxe"], False, "entries"),
                                      api.experts_grad_buffer_size(handle, self.R, m["dy"], m["hid"], m["dw2"], "entries"),
                                      api.experts_grad_buffer_size(handle, self.R, m["dhid"], m["x"], m["dw1"])), dtype=torch.uint8, device="cuda")
        self.grad_buffer = torch.empty(api.embedding_grad_buffer_size(handle, m["dx"], self.words, m["dtable"]), dtype=torch.uint8, device="cuda")
        self.forward()  # the routing exists: what is analysed once can be
        for A, B, C in ((self.combine, "y", "out"), (self.spread, "dout", "dy"), (self.sum, "dxe", "dx")):
            api.spmm_preprocess(handle, A, m[B], m[C])
        self.sddmm(True)

    def sddmm(self, prepare=False):
        import ctypes
        S, L = self.pkg, self.pkg.lib()
        one, zero = ctypes.c_uint16(0x3C00), ctypes.c_uint16(0)  # scalars of the compute type, f16
        args = [self.h.raw, S.ACL_SPARSE_OP_NON_TRANSPOSE, S.ACL_SPARSE_OP_TRANSPOSE, ctypes.byref(one), self.m["dout"].raw, self.m["y"].raw,
                ctypes.byref(zero), self.dR.raw, S.ACL_FLOAT16, 0]
        if prepare:
            size = ctypes.c_size_t()
            assert L.aclsparseSDDMMBufferSize(*args, ctypes.byref(size)) == 0
            self.sddmm_buffer = torch.empty(size.value, dtype=torch.uint8, device="cuda")
            assert L.aclsparseSDDMMPreprocess(*args, self.sddmm_buffer.data_ptr()) == 0
        assert L.aclsparseSDDMM(*args, self.sddmm_buffer.data_ptr()) == 0

    def forward(self):
        api, h, m = self.api, self.h, self.m
        api.embedding(h, m["table"], self.words, m["x"], alpha=0.5)
        with torch.cuda.stream(h.stream):
            torch.matmul(self.x.float(), self.gate.T, out=self.logits)
        api.route(h, self.rule, m["logits"], None, self.R)
        api.experts_preprocess(h, self.R, self.buffer)
        api.experts_mm(h, self.R, m["x"], m["w1"], m["hid"], buffer=self.buffer)
        api.experts_mm(h, self.R, m["hid"], m["w2"], m["y"], rows="entries", buffer=self.buffer)
        if self.combine.buffer is not None:
            api.spmm(h, self.combine, m["y"], m["out"])

    def backward(self):
        api, h, m = self.api, self.h, self.m
        api.spmm(h, self.spread, m["dout"], m["dy"])  # a row of dout for every entry, times its weight
        self.sddmm()
        api.route_grad(h, self.rule, m["logits"], self.R, api.DnVec(self.dvalues), m["dlogits"])
        api.experts_grad(h, self.R, m["dy"], m["hid"], m["dw2"], rows="entries", buffer=self.buffer)
        api.experts_mm(h, self.R, m["dy"], m["w2"], m["dhid"], transpose=False, rows="entries", buffer=self.buffer)
        api.experts_grad(h, self.R, m["dhid"], m["x"], m["dw1"], buffer=self.buffer)
        api.experts_mm(h, self.R, m["dhid"], m["w1"], m["dxe"], transpose=False, rows="entries", buffer=self.buffer)
        api.spmm(h, self.sum, m["dxe"], m["dx"])
        api.embedding_grad(h, m["dx"], self.words, m["dtable"], alpha=0.5, buffer=self.grad_buffer)

    RESULTS = ("out", "dlogits", "dw1", "dw2", "dtable")

    def check(self):
        """The whole in 64 bits, the choice of the experts taken as it is; the gate's part of dx is not in this chain."""
        tokens, vocab, width, hidden, experts, k = self.sizes
        leaf = {n: getattr(self, n).double().cpu().requires_grad_() for n in ("table", "w1", "w2", "logits")}
        columns = self.R.col_ind.view(tokens, k).cpu().long()
        x = 0.5 * leaf["table"][self.tokens.cpu()]
        assert torch.equal(columns, ref.route(self.logits, None, k, score="sigmoid", scale=2.0)[0].long())
        weights = ref.route_weights(leaf["logits"], columns, "sigmoid", True, 2.0)
        w1, w2 = leaf["w1"].view(experts, hidden, width), leaf["w2"].view(experts, width, hidden)
        y = torch.einsum("td,tkhd->tkh", x, w1[columns])
        y = torch.einsum("tkh,tkdh->tkd", y, w2[columns])
        out = (weights[..., None] * y).sum(1)
        grads = torch.autograd.grad((out * self.dout.double().cpu()).sum(), list(leaf.values()))
        want = dict(zip(self.RESULTS, (out.detach(), grads[3], grads[1], grads[2], grads[0])))
        for name in self.RESULTS:
            got = getattr(self, name).double().cpu()
            # each result passes at most eight tensors of f16: eight roundings of 2^-11 in the norm, twice for the terms that cancel
            off = (got - want[name]).norm() / want[name].norm()
            assert off <= 16 * 2.0 ** -11, (name, float(off))


def test_a_layer_forward_and_backward(pkg, handle):
    layer = Layer(pkg, handle)
    layer.forward()
    layer.backward()
    torch.cuda.synchronize()
    layer.check()


def test_a_layer_captured_and_replayed(pkg, device):
    """Captured once, replayed with other tokens and weights: the order of the entries is made anew in the graph."""
    from ops_sparse_b200 import api
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        h = api.Handle(stream)
        layer = Layer(pkg, h)
        layer.forward()
        layer.backward()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            layer.forward()
            layer.backward()
        for seed in (5, 6):
            g = gen(seed)
            layer.tokens.copy_(torch.randint(0, 500, (96,), generator=g, device="cuda"))
            layer.gate.copy_(0.2 * torch.randn(12, 64, generator=g, device="cuda"))
            layer.w1.mul_(-0.5)
            graph.replay()
            stream.synchronize()
            layer.check()
            kept = {n: getattr(layer, n).clone() for n in layer.RESULTS}
            layer.forward()  # eagerly, beside the graph
            layer.backward()
            stream.synchronize()
            assert all(torch.equal(kept[n], getattr(layer, n)) for n in layer.RESULTS)
        del graph
    h.close()


def test_two_layers_on_two_streams(pkg, device):
    """Handles, buffers and streams of their own; no result depends on the other's."""
    from ops_sparse_b200 import api
    streams = [torch.cuda.Stream() for _ in range(2)]
    layers = []
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            layers.append(Layer(pkg, api.Handle(s), tokens=300, experts=20, seed=i))
    torch.cuda.synchronize()
    for _ in range(5):
        for s, layer in zip(streams, layers):
            with torch.cuda.stream(s):
                layer.forward()
                layer.backward()
    torch.cuda.synchronize()
    for layer in layers:
        layer.check()


def test_scalars_on_the_device(pkg, handle):
    from ops_sparse_b200 import api
    g = gen(2)
    tokens = torch.randint(0, 30, (50,), generator=g, device="cuda")
    table, d = torch.randn(30, 24, generator=g, device="cuda"), torch.randn(50, 24, generator=g, device="cuda")
    old = torch.randn(30, 24, generator=g, device="cuda")
    handle.set_pointer_mode_device(True)
    alpha = torch.tensor([1.5], device="cuda")
    for b in (0.0, 1.0, 0.25):
        beta, grad, out = torch.tensor([b], device="cuda"), old.clone(), d.clone()
        api.embedding(handle, mat(api, table), api.DnVec(tokens), mat(api, out), alpha, beta)
        want = ref.embedding(table, tokens, 1.5, b, d)
        ref.close(out, want, 4 * F32 * (want.abs() + d.cpu().double().abs()))
        api.embedding_grad(handle, mat(api, d), api.DnVec(tokens), mat(api, grad), alpha, beta)
        want, size, many = ref.embedding_grad(d, tokens, 30, 1.5, b, old)
        ref.close(grad, want, (many + 4) * F32 * size)
    api.embedding(handle, mat(api, table), api.DnVec(tokens), mat(api, out), None, None)
    assert torch.equal(out, table[tokens])
    offsets, columns = ragged(g, 40, 3, 2)
    nnz = len(columns)
    x, w, y, dw = (matrix(g, *s)[0] for s in ((40, 48, "bf16"), (3 * 72, 48, "bf16"), (nnz, 72, "bf16"), (3 * 72, 48, "f32")))
    R = api.CsrMatrix(offsets, columns, torch.empty(nnz, device="cuda"), 40, 3)
    X, W, Y, DW = mat(api, x), mat(api, w), mat(api, y), mat(api, dw)
    buffer = torch.empty(max(api.experts_buffer_size(handle, R, X, W, Y), api.experts_grad_buffer_size(handle, R, Y, X, DW)), dtype=torch.uint8, device="cuda")
    api.experts_preprocess(handle, R, buffer)
    for b in (0.0, 0.5):
        beta = torch.tensor([b], device="cuda")
        want, size, many = ref.experts_grad(offsets, columns, y, x, 3, False, 1.5, b, dw.view(3, 72, 48))
        api.experts_grad(handle, R, Y, X, DW, alpha, beta, buffer=buffer)
        ref.close(dw.view(3, 72, 48), want, ref.rounding(dw.dtype, want) + size * (many + 4) * 2 * F32)
        want, size = ref.experts_mm(offsets, columns, x, w.view(3, 72, 48), 3, True, False, 1.5, b, y)
        api.experts_mm(handle, R, X, W, Y, alpha, beta, buffer=buffer)
        ref.close(y, want, ref.rounding(y.dtype, want) + size * 52 * 2 * F32)
    handle.set_pointer_mode_device(False)


def test_experts_wait_that_runs_out(pkg, handle):
    """Every barrier expects 16 bytes that nobody sends, and the limit is short: the product ends, says so, and the next works."""
    import ctypes
    from ops_sparse_b200 import api
    L = pkg.lib()
    L.b200sp_experts_wait_test.argtypes, L.b200sp_experts_wait_test.restype = [ctypes.c_longlong, ctypes.c_uint], None
    g = gen(4)
    offsets, columns = ragged(g, 50, 4, 2, wild=0)
    nnz = len(columns)
    x, w = matrix(g, 50, 64, "bf16")[0], matrix(g, 4 * 128, 64, "bf16")[0]
    y, dw = torch.full((nnz, 128), 5.0, dtype=torch.bfloat16, device="cuda"), torch.full((512, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    R = api.CsrMatrix(offsets, columns, torch.empty(nnz, device="cuda"), 50, 4)
    X, W, Y, DW = mat(api, x), mat(api, w), mat(api, y), mat(api, dw)
    buffer = torch.empty(max(api.experts_buffer_size(handle, R, X, W, Y), api.experts_grad_buffer_size(handle, R, Y, X, DW)), dtype=torch.uint8, device="cuda")
    api.experts_preprocess(handle, R, buffer)
    torch.cuda.synchronize()
    assert L.b200sp_experts_error() == 0
    for call, out in ((lambda: api.experts_mm(handle, R, X, W, Y, buffer=buffer), y), (lambda: api.experts_grad(handle, R, Y, X, DW, buffer=buffer), dw)):
        try:
            L.b200sp_experts_wait_test(2_000_000, 16)
            call()
            torch.cuda.synchronize()
        finally:
            L.b200sp_experts_wait_test(0, 0)
        assert L.b200sp_experts_error() == 1 and L.b200sp_experts_error_clear() == 0
        assert (out == 5).all()
    api.experts_mm(handle, R, X, W, Y, buffer=buffer)
    torch.cuda.synchronize()
    assert L.b200sp_experts_error() == 0
    want, size = ref.experts_mm(offsets, columns, x, w.view(4, 128, 64), 4, True, False, 1.0, 0.0, y)
    ref.close(y, want, ref.rounding(y.dtype, want) + size * 68 * 2 * F32)


def test_tables_and_weights_beyond_32_bits(pkg, handle):
    """More than 2^31 elements and 2^32 bytes: the last rows of a table, its gradient, the last of the experts."""
    from ops_sparse_b200 import api
    g = gen(9)
    vocab, width = 270001, 8192
    table = torch.empty(vocab, width, dtype=torch.float16, device="cuda")
    assert table.numel() > 2 ** 31
    tokens = torch.tensor([vocab - 1, 0, vocab - 2, vocab - 1, 262145], device="cuda")
    table[tokens] = torch.randn(5, width, generator=g, device="cuda").half()
    out = torch.empty(5, width, dtype=torch.float16, device="cuda")
    api.embedding(handle, mat(api, table), api.DnVec(tokens), mat(api, out))
    assert torch.equal(out, table[tokens])
    table.fill_(3.0)
    api.embedding_grad(handle, mat(api, out), api.DnVec(tokens), mat(api, table))
    want = torch.zeros(vocab, dtype=torch.bool, device="cuda")
    want[tokens] = True
    assert torch.equal((table != 0).any(1), want)
    assert torch.equal(table[vocab - 1], (out[0].float() + out[3].float()).half()) and torch.equal(table[262145], out[4])
    del table
    experts, n, d = 34, 8192, 8192
    w = torch.empty(experts * n, d, dtype=torch.bfloat16, device="cuda")
    assert w.numel() > 2 ** 31
    w[-n:] = torch.randn(n, d, generator=g, device="cuda").bfloat16() / 64
    x = torch.randn(3, d, generator=g, device="cuda").bfloat16()
    R = api.CsrMatrix(torch.arange(4, dtype=torch.int32, device="cuda"), torch.full((3,), experts - 1, dtype=torch.int32, device="cuda"),
                      torch.empty(3, device="cuda"), 3, experts)
    y = torch.empty(3, n, dtype=torch.float32, device="cuda")
    X, W, Y = mat(api, x), mat(api, w), mat(api, y)
    buffer = torch.empty(api.experts_buffer_size(handle, R, X, W, Y), dtype=torch.uint8, device="cuda")
    api.experts_preprocess(handle, R, buffer)
    api.experts_mm(handle, R, X, W, Y, buffer=buffer)
    last = w[-n:].double()
    ref.close(y, x.double() @ last.T, (x.double().abs() @ last.abs().T) * (d + 4) * 2 * F32)
    dy = torch.randn(3, n, generator=g, device="cuda").bfloat16()
    w.fill_(2.0)
    api.experts_grad(handle, R, mat(api, dy), X, W, buffer=buffer)
    assert (w[:-n] == 0).all()
    want = dy.double().T @ x.double()
    ref.close(w[-n:], want, ref.rounding(w.dtype, want) + 14 * F32 * (dy.double().abs().T @ x.double().abs()))
