"""CPU: calls of the token operators that have to be refused before anything is launched, at the borders of what is taken."""
from __future__ import annotations

import types

import pytest
import torch


def test_route_refuses_a_closed_bias(pkg):
    from ops_sparse_b200 import api
    bias = api.DnVec(torch.zeros(4))
    bias.close()
    x = api.DnMat.row_major(torch.zeros(2, 4))
    R = api.CsrMatrix(torch.zeros(3, dtype=torch.int32), torch.zeros(4, dtype=torch.int32), torch.zeros(4), 2, 4)
    nobody = types.SimpleNamespace(_h=None)  # a call that gets as far is refused for it
    with pytest.raises(ValueError, match="closed"):
        api.route(nobody, api.RouteRule(), x, bias, R)
    with pytest.raises(pkg.AclSparseError, match="HANDLE_IS_NULLPTR"):
        api.route(nobody, api.RouteRule(), x, None, R)
