"""CPU: what the token operators (include/b200sp_tokens.h) refuse, before anything is launched, and that they are exported."""
from __future__ import annotations

import re
import subprocess
from ctypes import addressof, byref, c_float, c_int, c_size_t, c_void_p, create_string_buffer
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
FAKE = 0x10000  # descriptors only store pointers; a refused call dereferences none
HANDLE = create_string_buffer(1024)  # stands for a handle: a refused call looks at nothing but whether there is one


def _h():
    return c_void_p(addressof(HANDLE))


def _mat(pkg, rows, cols, kind=None, ld=None, order=0, at=FAKE):
    d = c_void_p()
    kind = pkg.ACL_BF16 if kind is None else kind
    assert pkg.lib().aclsparseCreateDnMat(byref(d), rows, cols, ld or max(cols if order == 0 else rows, 1), c_void_p(at), kind, order) == 0
    return d


def _vec(pkg, size, kind, at=FAKE):
    d = c_void_p()
    assert pkg.lib().aclsparseCreateDnVec(byref(d), size, c_void_p(at), kind) == 0
    return d


def _csr(pkg, rows, cols, nnz, kind=None, offsets=0, base=0, at=FAKE):
    d = c_void_p()
    kind = pkg.ACL_FLOAT if kind is None else kind
    assert pkg.lib().aclsparseCreateCsr(byref(d), rows, cols, nnz, c_void_p(at), c_void_p(at), c_void_p(at), offsets, offsets, base, kind) == 0
    return d


def test_exported_and_mirrored(pkg):
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "b200sp_tokens.h").read_text(), flags=re.S)
    declared = set(re.findall(r"\b(b200sp\w+)\s*\(", text))
    out = subprocess.run(["nm", "-D", "--defined-only", str(pkg.LIB_PATH)], capture_output=True, text=True, check=True)
    exported = {line.split()[-1] for line in out.stdout.splitlines() if " T " in line}
    assert len(declared) == 13 and declared <= exported
    assert {n for n in declared if not n.startswith("b200sp_")} <= set(pkg._SIGNATURES)


def test_header_is_c(tmp_path):
    source = tmp_path / "caller.c"
    source.write_text('#include <stddef.h>\n#include "b200sp_tokens.h"\n'
                      "_Static_assert(sizeof(b200spRouteRule) == 24 && offsetof(b200spRouteRule, scale) == 20, \"layout\");\n")
    built = subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", str(ROOT / "include"), "-c", str(source), "-o",
                            str(tmp_path / "caller.o")], capture_output=True, text=True)
    assert built.returncode == 0, built.stderr


def test_embedding_refusals(pkg):
    S, f = pkg, pkg.lib().b200spEmbedding
    table, tokens, out = _mat(pkg, 100, 64), _vec(pkg, 7, S.ACL_INT64), _mat(pkg, 7, 64)
    call = lambda t=table, k=tokens, o=out, h=None: f(_h() if h is None else h, None, t, k, None, o)  # noqa: E731
    assert f(None, None, table, tokens, None, out) == S.ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR
    bad, no = S.ACL_SPARSE_STATUS_INVALID_VALUE, S.ACL_SPARSE_STATUS_NOT_SUPPORTED
    assert [call(t=None), call(k=None), call(o=None)] == [bad] * 3
    assert call(t=_mat(pkg, 100, 64, S.ACL_INT32)) == no
    assert call(t=_mat(pkg, 100, 64, order=1)) == no
    assert call(o=_mat(pkg, 7, 64, S.ACL_INT8)) == no
    assert call(o=_mat(pkg, 8, 64)) == bad and call(o=_mat(pkg, 7, 63)) == bad
    assert call(k=_vec(pkg, 7, S.ACL_FLOAT)) == no
    assert call(k=_vec(pkg, 7, S.ACL_INT64, FAKE + 4)) == bad  # not on the type's boundary
    assert call(t=_mat(pkg, 100, 64, at=FAKE + 1)) == bad
    assert call(t=_mat(pkg, (1 << 31) - 1, 64)) == no
    many = (1 << 31) - (1 << 20) + 1
    assert call(k=_vec(pkg, many, S.ACL_INT32), o=_mat(pkg, many, 64)) == no
    assert call(t=_mat(pkg, 100, 64, ld=1 << 31)) == no and call(t=_mat(pkg, 1, many)) == no
    size = c_size_t()
    g = pkg.lib().b200spEmbeddingGradBufferSize
    assert g(_h(), out, tokens, table, None) == bad
    assert g(_h(), out, tokens, table, byref(size)) == 0 and size.value > 0
    assert g(_h(), _mat(pkg, 6, 64), tokens, table, byref(size)) == bad
    assert pkg.lib().b200spEmbeddingGrad(_h(), None, out, tokens, None, table, None) == S.ACL_SPARSE_STATUS_INSUFFICIENT_RESOURCES
    assert pkg.lib().b200spEmbeddingGrad(None, None, out, tokens, None, table, None) == S.ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR


def _rule(pkg, **change):
    rule = pkg.RouteRule()
    for name, value in change.items():
        setattr(rule, name, value)
    return rule


@pytest.mark.parametrize("change", [
    {"score": 2}, {"group_score": 2}, {"renormalise": 2}, {"scale": float("nan")}, {"scale": float("inf")}, {"groups": 0},
    {"groups_kept": 0}, {"groups": 4, "groups_kept": 5}, {"groups": 7, "groups_kept": 7},  # 64 experts are no seven groups
    {"groups": 32, "groups_kept": 3},  # six experts for eight entries
])
def test_route_rule_refusals(pkg, change):
    x, R = _mat(pkg, 10, 64), _csr(pkg, 10, 64, 80)
    rule = _rule(pkg, **change)
    assert pkg.lib().b200spRoute(_h(), rule.address, x, None, R) == pkg.ACL_SPARSE_STATUS_INVALID_VALUE
    assert pkg.lib().b200spRouteGrad(_h(), rule.address, x, R, _vec(pkg, 80, pkg.ACL_FLOAT), x) == pkg.ACL_SPARSE_STATUS_INVALID_VALUE


def test_route_refusals(pkg):
    S, f = pkg, pkg.lib().b200spRoute
    rule = pkg.RouteRule()
    x, R = _mat(pkg, 10, 64), _csr(pkg, 10, 64, 80)
    bad, no = S.ACL_SPARSE_STATUS_INVALID_VALUE, S.ACL_SPARSE_STATUS_NOT_SUPPORTED
    assert f(None, rule.address, x, None, R) == S.ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR
    call = lambda x=x, b=None, R=R, r=rule.address: f(_h(), r, x, b, R)  # noqa: E731
    assert [call(x=None), call(R=None), call(r=None)] == [bad] * 3
    assert call(R=_csr(pkg, 10, 64, 81)) == bad  # not the same number in every row
    assert call(R=_csr(pkg, 10, 64, 0)) == bad
    assert call(R=_csr(pkg, 10, 64, 650)) == no and call(R=_csr(pkg, 10, 64, 330)) == no  # more than 32 a row
    assert call(x=_mat(pkg, 10, 8), R=_csr(pkg, 10, 8, 90)) == bad  # nine of eight experts
    assert call(x=_mat(pkg, 11, 64)) == bad and call(x=_mat(pkg, 10, 65)) == bad
    assert call(x=_mat(pkg, 10, 64, order=1)) == no and call(x=_mat(pkg, 10, 64, S.ACL_INT32)) == no
    assert call(R=_csr(pkg, 10, 64, 80, S.ACL_INT32)) == no and call(R=_csr(pkg, 10, 64, 80, offsets=1)) == no
    assert call(R=_csr(pkg, 10, 64, 80, base=1)) == no
    assert call(x=_mat(pkg, 10, 1025), R=_csr(pkg, 10, 1025, 80)) == no
    assert call(b=_vec(pkg, 64, S.ACL_FLOAT, FAKE + 2)) == bad and call(R=_csr(pkg, 10, 64, 80, at=FAKE + 2)) == bad  # not on the types' boundaries
    assert call(b=_vec(pkg, 63, S.ACL_FLOAT)) == bad and call(b=_vec(pkg, 64, S.ACL_BF16)) == no
    many = _rule(pkg, groups=64, groups_kept=64)
    assert f(_h(), many.address, x, None, R) == no
    g = pkg.lib().b200spRouteGrad
    d = _vec(pkg, 80, S.ACL_FLOAT)
    assert g(None, rule.address, x, R, d, x) == S.ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR
    assert g(_h(), rule.address, x, R, None, x) == bad and g(_h(), rule.address, x, R, d, None) == bad
    assert g(_h(), rule.address, x, R, _vec(pkg, 79, S.ACL_FLOAT), x) == bad and g(_h(), rule.address, x, R, _vec(pkg, 80, S.ACL_FLOAT, FAKE + 2), x) == bad
    assert g(_h(), rule.address, x, R, _vec(pkg, 80, S.ACL_INT32), x) == no
    assert g(_h(), rule.address, x, R, d, _mat(pkg, 10, 64, S.ACL_FLOAT)) == no
    assert g(_h(), rule.address, x, R, d, _mat(pkg, 9, 64)) == bad


def test_experts_refusals(pkg):
    S, L = pkg, pkg.lib()
    size = c_size_t()
    bad, no = S.ACL_SPARSE_STATUS_INVALID_VALUE, S.ACL_SPARSE_STATUS_NOT_SUPPORTED
    R, X, W, Y = _csr(pkg, 10, 4, 20), _mat(pkg, 10, 32), _mat(pkg, 4 * 48, 32), _mat(pkg, 20, 48)

    def mm(op=1, rows=0, R=R, X=X, W=W, Y=Y):
        sized = L.b200spExpertsMMBufferSize(_h(), op, rows, R, X, W, Y, byref(size))
        run = L.b200spExpertsMM(_h(), op, rows, None, R, X, W, None, Y, c_void_p(FAKE))
        assert sized == run or (sized == 0 and run == bad)  # no order in the buffer
        return sized

    assert mm() == 0 and size.value >= 4 * (4 + 2) + 4 * 20
    assert mm(op=2) == no and mm(rows=2) == bad
    assert mm(R=None) == bad and mm(X=None) == bad and mm(W=None) == bad and mm(Y=None) == bad
    assert mm(rows=1) == bad  # X has a row per token
    assert mm(rows=1, X=_mat(pkg, 20, 32)) == 0
    assert mm(op=0) == bad and mm(op=0, X=_mat(pkg, 10, 48), Y=_mat(pkg, 20, 32)) == 0
    assert mm(W=_mat(pkg, 4 * 48 + 1, 32)) == bad and mm(W=_mat(pkg, 4 * 48, 33)) == bad
    assert mm(Y=_mat(pkg, 19, 48)) == bad and mm(Y=_mat(pkg, 20, 47)) == bad
    assert mm(Y=_mat(pkg, 20, 48, S.ACL_FLOAT)) == 0 and mm(Y=_mat(pkg, 20, 48, S.ACL_FLOAT16)) == no
    assert mm(X=_mat(pkg, 10, 32, S.ACL_FLOAT)) == no and mm(W=_mat(pkg, 4 * 48, 32, S.ACL_FLOAT16)) == no
    assert mm(X=_mat(pkg, 10, 32, order=1)) == no
    assert mm(R=_csr(pkg, 10, 4, 20, offsets=1)) == no and mm(R=_csr(pkg, 10, 4, 20, base=1)) == no
    assert mm(R=_csr(pkg, 10, 4, 20, at=FAKE + 1)) == bad
    assert mm(R=_csr(pkg, 10, 1025, 20), W=_mat(pkg, 1025, 32), Y=_mat(pkg, 20, 1)) == no
    assert L.b200spExpertsMM(None, 1, 0, None, R, X, W, None, Y, None) == S.ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR
    assert L.b200spExpertsMM(_h(), 1, 0, None, R, X, W, None, Y, None) == S.ACL_SPARSE_STATUS_INSUFFICIENT_RESOURCES
    assert L.b200spExpertsMMBufferSize(_h(), 1, 0, R, X, W, Y, None) == bad
    assert L.b200spExpertsPreprocess(None, R, None) == S.ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR
    assert L.b200spExpertsPreprocess(_h(), R, None) == S.ACL_SPARSE_STATUS_INSUFFICIENT_RESOURCES
    assert L.b200spExpertsPreprocess(_h(), None, c_void_p(FAKE)) == bad
    dY, dW = Y, W

    def grad(rows=0, R=R, dY=dY, X=X, dW=dW):
        return L.b200spExpertsGradBufferSize(_h(), rows, R, dY, X, dW, byref(size))

    assert grad() == 0 and grad(dW=_mat(pkg, 4 * 48, 32, S.ACL_FLOAT)) == 0
    assert grad(dY=_mat(pkg, 20, 47)) == bad and grad(dY=_mat(pkg, 21, 48)) == bad and grad(X=_mat(pkg, 10, 31)) == bad
    assert grad(dY=_mat(pkg, 20, 48, S.ACL_FLOAT)) == no and grad(rows=3) == bad
    assert L.b200spExpertsGrad(_h(), 0, None, R, dY, X, None, dW, c_void_p(FAKE)) == bad  # no order in the buffer
    assert L.b200spExpertsGrad(_h(), 0, None, R, dY, X, None, dW, None) == S.ACL_SPARSE_STATUS_INSUFFICIENT_RESOURCES
    assert c_float(1).value == 1 and c_int(1).value == 1
