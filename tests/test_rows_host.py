"""CPU: what the operators of include/b200sp_rows.h refuse, before anything is launched, and that they are exported."""
from __future__ import annotations

import re
import subprocess
from ctypes import byref, c_size_t, c_void_p
from pathlib import Path

import pytest
import torch

import rows_reference as rows
from test_tokens_host import FAKE, _csr, _h, _mat, _vec

ROOT = Path(__file__).resolve().parents[1]
BUFFER = c_void_p(FAKE)


def test_exported_and_mirrored(pkg):
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "b200sp_rows.h").read_text(), flags=re.S)
    declared = set(re.findall(r"\b(b200sp\w+)\s*\(", text))
    out = subprocess.run(["nm", "-D", "--defined-only", str(pkg.LIB_PATH)], capture_output=True, text=True, check=True)
    exported = {line.split()[-1] for line in out.stdout.splitlines() if " T " in line}
    assert len(declared) == 13 and declared <= exported
    assert {n for n in declared if not n.startswith("b200sp_")} <= set(pkg._SIGNATURES)


def test_header_is_c(tmp_path):
    source = tmp_path / "caller.c"
    source.write_text('#include "b200sp_rows.h"\nint main(void) { return B200SP_WEIGHTS_NONE; }\n')
    built = subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", str(ROOT / "include"), "-c", str(source), "-o",
                            str(tmp_path / "caller.o")], capture_output=True, text=True)
    assert built.returncode == 0, built.stderr


def _routing(pkg):
    """Ten tokens of twenty entries, four experts."""
    return _csr(pkg, 10, 4, 20)


def _bad_routings(pkg):
    S = pkg
    return [(None, S.ACL_SPARSE_STATUS_INVALID_VALUE), (_csr(pkg, 10, 4, 20, offsets=1), S.ACL_SPARSE_STATUS_NOT_SUPPORTED),
            (_csr(pkg, 10, 4, 20, base=1), S.ACL_SPARSE_STATUS_NOT_SUPPORTED),
            (_csr(pkg, 10, 4, 20, at=FAKE + 2), S.ACL_SPARSE_STATUS_INVALID_VALUE),
            (_csr(pkg, 10, 1025, 20), S.ACL_SPARSE_STATUS_NOT_SUPPORTED), (_csr(pkg, 10, 4, 0), S.ACL_SPARSE_STATUS_INVALID_VALUE)]


def test_order_buffer_size(pkg):
    f, size = pkg.lib().b200spExpertsOrderBufferSize, c_size_t()
    assert f(_h(), _routing(pkg), byref(size)) == 0 and size.value >= 4 * (4 + 2) + 3 * 4 * 20
    assert f(_h(), _routing(pkg), None) == pkg.ACL_SPARSE_STATUS_INVALID_VALUE
    assert f(None, _routing(pkg), byref(size)) == pkg.ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR
    for R, status in _bad_routings(pkg):
        assert f(_h(), R, byref(size)) == status


def test_dispatch_refusals(pkg):
    S, f = pkg, pkg.lib().b200spExpertsDispatch
    bad, no = S.ACL_SPARSE_STATUS_INVALID_VALUE, S.ACL_SPARSE_STATUS_NOT_SUPPORTED
    R, X, Y = _routing(pkg), _mat(pkg, 10, 32), _mat(pkg, 20, 32)
    call = lambda R=R, X=X, Y=Y, o=None, b=BUFFER: f(_h(), None, R, X, None, Y, o, b)  # noqa: E731
    assert f(None, None, R, X, None, Y, None, BUFFER) == S.ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR
    assert call() == bad  # no order in the buffer
    assert call(b=None) == S.ACL_SPARSE_STATUS_INSUFFICIENT_RESOURCES
    for M, status in _bad_routings(pkg):
        assert call(R=M) == status
    assert [call(X=None), call(Y=None), call(X=_mat(pkg, 9, 32)), call(Y=_mat(pkg, 21, 32)), call(Y=_mat(pkg, 20, 31)),
            call(X=_mat(pkg, 10, 32, at=FAKE + 1))] == [bad] * 6
    assert [call(X=_mat(pkg, 10, 32, order=1)), call(Y=_mat(pkg, 20, 32, S.ACL_FLOAT16)), call(X=_mat(pkg, 10, 32, S.ACL_FLOAT)),
            call(X=_mat(pkg, 10, 32, S.ACL_INT8), Y=_mat(pkg, 20, 32, S.ACL_INT8))] == [no] * 4
    sized = dict(b=None)
    ok = S.ACL_SPARSE_STATUS_INSUFFICIENT_RESOURCES  # the last thing that is looked at
    assert call(Y=_mat(pkg, 20, 32, S.ACL_FLOAT), **sized) == ok and call(o=_vec(pkg, 5, S.ACL_INT32), **sized) == ok
    assert call(o=_vec(pkg, 4, S.ACL_INT32), **sized) == bad and call(o=_vec(pkg, 5, S.ACL_INT32, FAKE + 2), **sized) == bad
    assert call(o=_vec(pkg, 5, S.ACL_INT64), **sized) == no


def test_combine_refusals(pkg):
    S, f = pkg, pkg.lib().b200spExpertsCombine
    bad, no, ok = S.ACL_SPARSE_STATUS_INVALID_VALUE, S.ACL_SPARSE_STATUS_NOT_SUPPORTED, S.ACL_SPARSE_STATUS_INSUFFICIENT_RESOURCES
    R, X, Y = _routing(pkg), _mat(pkg, 20, 32), _mat(pkg, 10, 32)
    call = lambda w=1, R=R, X=X, Y=Y, b=None: f(_h(), w, None, R, X, None, Y, b)  # noqa: E731
    assert f(None, 1, None, R, X, None, Y, BUFFER) == S.ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR
    assert call() == ok and call(b=BUFFER) == bad
    for M, status in _bad_routings(pkg):
        assert call(R=M) == status
    assert [call(w=2), call(w=-1), call(X=None), call(Y=None), call(X=_mat(pkg, 19, 32)), call(Y=_mat(pkg, 11, 32)),
            call(Y=_mat(pkg, 10, 33))] == [bad] * 7
    whole = _csr(pkg, 10, 4, 20, S.ACL_INT32)
    assert call(R=whole) == no and call(w=0, R=whole) == ok
    F, H = S.ACL_FLOAT, S.ACL_FLOAT16
    assert call(Y=_mat(pkg, 10, 32, H)) == no and call(Y=_mat(pkg, 10, 32, F)) == ok
    assert call(X=_mat(pkg, 20, 32, F), Y=_mat(pkg, 10, 32, H)) == ok and call(X=_mat(pkg, 20, 32, order=1)) == no


def test_combine_gradient_refusals(pkg):
    S, f = pkg, pkg.lib().b200spExpertsCombineGrad
    bad, no, ok = S.ACL_SPARSE_STATUS_INVALID_VALUE, S.ACL_SPARSE_STATUS_NOT_SUPPORTED, S.ACL_SPARSE_STATUS_INSUFFICIENT_RESOURCES
    R, G, X, D, V = _routing(pkg), _mat(pkg, 10, 32), _mat(pkg, 20, 32), _mat(pkg, 20, 32), _vec(pkg, 20, S.ACL_FLOAT)
    call = lambda R=R, G=G, X=X, D=D, V=V, b=None: f(_h(), None, R, G, X, None, D, V, b)  # noqa: E731
    assert f(None, None, R, G, X, None, D, V, BUFFER) == S.ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR
    assert call() == ok and call(b=BUFFER) == bad and call(X=None, V=None) == ok
    for M, status in _bad_routings(pkg):
        assert call(R=M) == status
    assert [call(X=None), call(V=None), call(G=None), call(D=None), call(G=_mat(pkg, 9, 32)), call(X=_mat(pkg, 20, 31)),
            call(D=_mat(pkg, 19, 32)), call(V=_vec(pkg, 19, S.ACL_FLOAT)), call(V=_vec(pkg, 20, S.ACL_BF16, FAKE + 1))] == [bad] * 9
    assert [call(R=_csr(pkg, 10, 4, 20, S.ACL_INT8)), call(V=_vec(pkg, 20, S.ACL_INT32)), call(X=_mat(pkg, 20, 32, S.ACL_FLOAT)),
            call(G=_mat(pkg, 10, 32, S.ACL_FLOAT16))] == [no] * 4
    assert call(V=_vec(pkg, 20, S.ACL_BF16)) == ok and call(G=_mat(pkg, 10, 32, S.ACL_FLOAT)) == ok


def test_quantise_refusals(pkg):
    S, f, g = pkg, pkg.lib().b200spQuantiseRows, pkg.lib().b200spExpertsQuantise
    bad, no, ok = S.ACL_SPARSE_STATUS_INVALID_VALUE, S.ACL_SPARSE_STATUS_NOT_SUPPORTED, S.ACL_SPARSE_STATUS_INSUFFICIENT_RESOURCES
    R, X, Q, V = _routing(pkg), _mat(pkg, 10, 32), _mat(pkg, 20, 32, S.ACL_INT8), _vec(pkg, 20, S.ACL_FLOAT)
    rows_ = lambda X=_mat(pkg, 20, 32), Q=Q, V=V: f(_h(), X, Q, V)  # noqa: E731
    experts = lambda R=R, X=X, Q=Q, V=V, o=None, b=None: g(_h(), R, X, Q, V, o, b)  # noqa: E731
    assert f(None, X, Q, V) == g(None, R, X, Q, V, None, BUFFER) == S.ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR
    assert experts() == ok and experts(b=BUFFER) == bad and experts(o=_vec(pkg, 5, S.ACL_INT32)) == ok
    assert experts(o=_vec(pkg, 6, S.ACL_INT32)) == bad
    for M, status in _bad_routings(pkg):
        assert experts(R=M) == status
    for call in (rows_, experts):
        assert [call(X=None), call(Q=None), call(V=None), call(X=_mat(pkg, 11, 32)), call(Q=_mat(pkg, 20, 31, S.ACL_INT8)),
                call(V=_vec(pkg, 19, S.ACL_FLOAT)), call(V=_vec(pkg, 20, S.ACL_FLOAT, FAKE + 2))] == [bad] * 7
        assert [call(X=_mat(pkg, 10, 32, S.ACL_INT8)), call(Q=_mat(pkg, 20, 32)), call(V=_vec(pkg, 20, S.ACL_FLOAT16)),
                call(Q=_mat(pkg, 20, 32, S.ACL_INT8, order=1))] == [no] * 4


def test_scaled_refusals(pkg):
    S, L = pkg, pkg.lib()
    bad, no, short = S.ACL_SPARSE_STATUS_INVALID_VALUE, S.ACL_SPARSE_STATUS_NOT_SUPPORTED, S.ACL_SPARSE_STATUS_INSUFFICIENT_RESOURCES
    size, I8 = c_size_t(), S.ACL_INT8
    X, W, Y = _mat(pkg, 10, 64, I8), _mat(pkg, 48, 64, I8), _mat(pkg, 10, 48)
    sx, sw = _vec(pkg, 10, S.ACL_FLOAT), _vec(pkg, 48, S.ACL_FLOAT)
    sized = lambda X=X, W=W, Y=Y: L.b200spScaledMMBufferSize(_h(), X, W, Y, byref(size))  # noqa: E731
    assert sized() == 0 and size.value == 0
    assert sized(X=_mat(pkg, 10, 64, I8, ld=65)) == 0 and size.value >= 640
    assert sized(W=_mat(pkg, 48, 64, I8, at=FAKE + 1)) == 0 and size.value >= 48 * 64
    assert L.b200spScaledMMBufferSize(_h(), X, W, Y, None) == bad
    assert L.b200spScaledMMBufferSize(None, X, W, Y, byref(size)) == S.ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR
    assert [sized(X=None), sized(W=None), sized(Y=None), sized(W=_mat(pkg, 48, 63, I8)), sized(Y=_mat(pkg, 11, 48)),
            sized(Y=_mat(pkg, 10, 47))] == [bad] * 6
    deep = 131072
    assert [sized(X=_mat(pkg, 10, 64)), sized(W=_mat(pkg, 48, 64, S.ACL_INT32)), sized(Y=_mat(pkg, 10, 48, I8)),
            sized(X=_mat(pkg, 10, 64, I8, order=1)), sized(Y=_mat(pkg, 10, 48, order=1)),
            sized(X=_mat(pkg, 10, deep, I8), W=_mat(pkg, 48, deep, I8))] == [no] * 6
    assert sized(X=_mat(pkg, 10, deep - 1, I8), W=_mat(pkg, 48, deep - 1, I8)) == 0
    f = L.b200spScaledMM
    assert f(None, None, X, sx, W, sw, None, Y, None) == S.ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR
    odd = _mat(pkg, 10, 64, I8, ld=65)
    assert f(_h(), None, odd, sx, W, sw, None, Y, None) == short
    for wrong, status in ((None, bad), (_vec(pkg, 11, S.ACL_FLOAT), bad), (_vec(pkg, 10, S.ACL_FLOAT, FAKE + 1), bad),
                          (_vec(pkg, 10, S.ACL_BF16), no)):
        assert f(_h(), None, odd, wrong, W, sw, None, Y, None) == status
    assert f(_h(), None, odd, sx, W, sx, None, Y, None) == bad

    R, X, W, Y = _routing(pkg), _mat(pkg, 20, 64, I8), _mat(pkg, 4 * 48, 64, I8), _mat(pkg, 20, 48)
    sx, sw = _vec(pkg, 20, S.ACL_FLOAT), _vec(pkg, 192, S.ACL_FLOAT)
    experts = lambda R=R, X=X, W=W, Y=Y: L.b200spExpertsScaledMMBufferSize(_h(), R, X, W, Y, byref(size))  # noqa: E731
    assert experts() == 0
    plain = size.value
    assert experts(X=_mat(pkg, 20, 64, I8, ld=72)) == 0 and size.value >= plain + 20 * 64
    for M, status in _bad_routings(pkg):
        assert experts(R=M, W=_mat(pkg, 1025, 64, I8) if M is not None else W) == status
    assert [experts(W=_mat(pkg, 191, 64, I8)), experts(X=_mat(pkg, 10, 64, I8), Y=_mat(pkg, 10, 48)), experts(Y=_mat(pkg, 20, 47))] == [bad] * 3
    f = L.b200spExpertsScaledMM
    assert f(None, None, R, X, sx, W, sw, None, Y, BUFFER) == S.ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR
    assert f(_h(), None, R, X, sx, W, sw, None, Y, None) == short
    assert f(_h(), None, R, X, sx, W, sw, None, Y, BUFFER) == bad  # no order in the buffer
    assert f(_h(), None, R, X, sw, W, sw, None, Y, None) == bad and f(_h(), None, R, X, sx, W, sx, None, Y, None) == bad


def test_closed_descriptors_are_refused(pkg):
    """A closed optional argument is no absent one."""
    from ops_sparse_b200 import api

    class Closed:
        _d = c_void_p()

    for call in (lambda c: api.experts_dispatch(None, None, None, None, offsets=c),
                 lambda c: api.experts_quantise(None, None, None, None, None, offsets=c)):
        with pytest.raises((ValueError, AttributeError)):
            call(Closed())
    with pytest.raises(ValueError):
        api._optional(Closed(), "S")
    assert api._optional(None, "S") is None


def test_reference_rounding():
    """The definition that the kernels are held to, by arithmetic of fractions."""
    from fractions import Fraction
    g = torch.Generator().manual_seed(3)
    x = torch.randn(20, 50, generator=g).bfloat16().float()
    x[0] = torch.arange(50) / 2.0 - 12.25
    x[0, 0] = 127.0  # halves
    q, scale = rows.quantise(x)
    for r in range(20):
        top = max(abs(Fraction(v)) for v in x[r].tolist())
        assert q[r].tolist() == [round(Fraction(v) * 127 / top) for v in x[r].tolist()]  # Python's halves go to the even one, too
        assert abs(Fraction(scale[r].item()) - top / 127) <= top / 127 * Fraction(1, 2 ** 24)
