"""GPU: operators of include/b200sp_rows.h at their borders -- beside other streams, in each form of a product, at far addresses."""
from __future__ import annotations

import pytest
import torch

import rows_reference as rows
import token_reference as ref
from test_rows_gpu import eights, no_error, ordered, routed
from test_tokens_gpu import gen, mat
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
