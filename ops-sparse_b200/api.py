"""Object wrappers over the aclsparse C API for callers that hold torch CUDA tensors.

Each class owns one C descriptor (created in __init__, destroyed in close()/__del__) and
keeps a reference to the tensors whose device pointers the descriptor borrows.  The call
sequence is the reference's own (test/spmv/arch22/spmv_test.cpp:415-479,
test/spmm/arch35/spmm_test.cpp:460-516): handle -> descriptors -> GetBufferSize ->
Preprocess -> compute.  All arithmetic happens inside libops_sparse.so.
"""
from __future__ import annotations

from ctypes import Structure, addressof, byref, c_float, c_int, c_int32, c_size_t, c_void_p

import torch

from . import (
    ACL_BF16, ACL_FLOAT, ACL_FLOAT16, ACL_INT8, ACL_INT32, ACL_INT64, ACL_SPARSE_INDEX_32I, ACL_SPARSE_INDEX_64I,
    ACL_SPARSE_INDEX_BASE_ZERO, ACL_SPARSE_SPMVOP_ALG_DEFAULT, ACL_SPARSE_SPMVOP_ALG2,
    ACL_SPARSE_OP_NON_TRANSPOSE, ACL_SPARSE_ORDER_COL, ACL_SPARSE_ORDER_ROW, ACL_SPARSE_POINTER_MODE_DEVICE,
    ACL_SPARSE_OP_TRANSPOSE, ACL_SPARSE_SPMM_ALG_DEFAULT, ACL_SPARSE_SPMV_ALG_DEFAULT, B200SP_GROUP_MAX, B200SP_GROUP_TOP2,
    B200SP_ROUTE_SIGMOID, B200SP_ROUTE_SOFTMAX, B200SP_ROWS_OF_ENTRIES, B200SP_ROWS_OF_TOKENS, B200SP_WEIGHTS_NONE,
    B200SP_WEIGHTS_OF_R, check, lib,
)

_ACL_OF = {
    torch.float32: ACL_FLOAT, torch.float16: ACL_FLOAT16, torch.bfloat16: ACL_BF16,
    torch.int32: ACL_INT32, torch.int8: ACL_INT8, torch.int64: ACL_INT64,
}


def acl_type_of(dtype: torch.dtype) -> int:
    try:
        return _ACL_OF[dtype]
    except KeyError:
        raise TypeError(f"no aclDataType for {dtype}") from None


def _ptr(t: torch.Tensor | None) -> c_void_p | None:
    """Device pointer of a tensor as a C void* (None -> NULL)."""
    return None if t is None else c_void_p(t.data_ptr())


class _PackedCall(Structure):
    """b200spPackedCall (include/b200sp_packed.h)."""

    _fields_ = [("handle", c_void_p), ("a", c_void_p), ("x", c_void_p), ("y", c_void_p), ("out", c_void_p),
                ("buffer", c_void_p), ("opA", c_int), ("opB", c_int), ("alg", c_int)]


class _PackedCalls(dict):
    """Packed argument structs of the products a matrix (or plan) was used in, by the very values they hold: an entry
    can not go stale, it is found only by a call with the same arguments.  Converting ten arguments costs an
    interpreter more than launching a small product; with these a repeated call converts three."""

    MOST = 64

    def pack(self, key, **fields) -> tuple:
        if len(self) >= self.MOST:
            self.clear()
        struct = _PackedCall(**fields)
        call = self[key] = struct, addressof(struct)
        return call  # not looked up again: another thread may have emptied the table


class Handle:
    """aclsparseHandle_t bound to a CUDA stream (default: torch's current stream)."""

    def __init__(self, stream: torch.cuda.Stream | None = None):
        self._h = c_void_p()
        check(lib().aclsparseCreate(byref(self._h)), "aclsparseCreate")
        s = stream if stream is not None else torch.cuda.current_stream()
        self.stream = s
        check(lib().aclsparseSetStream(self._h, c_void_p(s.cuda_stream)), "aclsparseSetStream")
        self.device_scalars = False

    @property
    def raw(self) -> c_void_p:
        return self._h

    def set_pointer_mode_device(self, on: bool) -> None:
        check(lib().aclsparseSetPointerMode(self._h, ACL_SPARSE_POINTER_MODE_DEVICE if on else 0),
              "aclsparseSetPointerMode")
        self.device_scalars = on

    def close(self) -> None:
        if self._h:
            lib().aclsparseDestroy(self._h)
            self._h = c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class DnVec:
    def __init__(self, values: torch.Tensor, size: int | None = None):
        self.values = values
        self.is_i32 = values.dtype == torch.int32
        self._d = c_void_p()
        n = values.numel() if size is None else size
        check(lib().aclsparseCreateDnVec(byref(self._d), n, _ptr(values), acl_type_of(values.dtype)),
              "aclsparseCreateDnVec")

    @property
    def raw(self) -> c_void_p:
        return self._d

    def close(self) -> None:
        if self._d:
            lib().aclsparseDestroyDnVec(self._d)
            self._d = c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class DnMat:
    """Dense matrix descriptor over a 2-D tensor.  order 'row': ld = stride(0); 'col': the
    tensor holds the column-major storage, i.e. it has shape (cols, ld-ish) transposed."""

    def __init__(self, values: torch.Tensor, rows: int, cols: int, ld: int, order: str = "row"):
        self.values = values
        self.is_i32 = values.dtype == torch.int32
        self.rows, self.cols, self.ld, self.order = rows, cols, ld, order
        self._d = c_void_p()
        check(lib().aclsparseCreateDnMat(byref(self._d), rows, cols, ld, _ptr(values), acl_type_of(values.dtype),
                                         ACL_SPARSE_ORDER_ROW if order == "row" else ACL_SPARSE_ORDER_COL),
              "aclsparseCreateDnMat")

    @classmethod
    def row_major(cls, t: torch.Tensor) -> "DnMat":
        assert t.dim() == 2 and t.stride(1) == 1
        return cls(t, t.shape[0], t.shape[1], t.stride(0), "row")

    @property
    def raw(self) -> c_void_p:
        return self._d

    def close(self) -> None:
        if self._d:
            lib().aclsparseDestroyDnMat(self._d)
            self._d = c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class CsrMatrix:
    def __init__(self, row_ptr: torch.Tensor, col_ind: torch.Tensor, values: torch.Tensor, rows: int, cols: int,
                 nnz: int | None = None, index_base: int = ACL_SPARSE_INDEX_BASE_ZERO):
        """row_ptr is int32, or int64 for the SpMVOp plan API; index_base 1 likewise is SpMVOp only."""
        assert row_ptr.dtype in (torch.int32, torch.int64) and col_ind.dtype == torch.int32
        self.row_ptr, self.col_ind, self.values = row_ptr, col_ind, values
        self.is_whole = values.dtype in (torch.int32, torch.int8)
        self.rows, self.cols = rows, cols
        self.nnz = col_ind.numel() if nnz is None else nnz
        self._d = c_void_p()
        off_type = ACL_SPARSE_INDEX_64I if row_ptr.dtype == torch.int64 else ACL_SPARSE_INDEX_32I
        check(lib().aclsparseCreateCsr(byref(self._d), rows, cols, self.nnz, _ptr(row_ptr), _ptr(col_ind),
                                       _ptr(values), off_type, ACL_SPARSE_INDEX_32I, index_base,
                                       acl_type_of(values.dtype)),
              "aclsparseCreateCsr")
        self.buffer: torch.Tensor | None = None  # workspace recorded by preprocess_*()
        self._calls = _PackedCalls()

    @property
    def raw(self) -> c_void_p:
        return self._d

    def close(self) -> None:
        if self._d:
            self._calls.clear()
            lib().aclsparseDestroySpMat(self._d)
            self._d = c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def _scalars(handle: Handle, alpha, beta, compute_type: int):
    """The scalar arguments of the C call: pointers to host copies that live as long as the arguments do, or the
    device pointers themselves.  (byref of a fresh object: a cast to c_void_p costs as much as the rest of a call.)"""
    if handle.device_scalars:
        return _ptr(alpha), _ptr(beta)
    if compute_type == ACL_INT32:
        return byref(c_int32(alpha)), byref(c_int32(beta))
    return byref(c_float(alpha)), byref(c_float(beta))


def _compute_type(values: torch.Tensor, out: torch.Tensor) -> int:
    return ACL_INT32 if (values.dtype in (torch.int32, torch.int8) and out.dtype == torch.int32) else ACL_FLOAT


def _product_type(A: CsrMatrix, out: DnVec | DnMat) -> int:
    """The same from what the descriptors were created with."""
    return ACL_INT32 if A.is_whole and out.is_i32 else ACL_FLOAT


def spmv_buffer_size(handle: Handle, A: CsrMatrix, x: DnVec, y: DnVec, op: int = ACL_SPARSE_OP_NON_TRANSPOSE) -> int:
    size = c_size_t()
    ct = _product_type(A, y)
    check(lib().aclsparseSpMVGetBufferSize(handle.raw, op, None, A.raw, x.raw, None, y.raw, ct,
                                           ACL_SPARSE_SPMV_ALG_DEFAULT, byref(size)), "aclsparseSpMVGetBufferSize")
    return size.value


def spmv_preprocess(handle: Handle, A: CsrMatrix, x: DnVec, y: DnVec, op: int = ACL_SPARSE_OP_NON_TRANSPOSE):
    """GetBufferSize + device allocation + Preprocess; the buffer is kept on A.buffer."""
    nbytes = spmv_buffer_size(handle, A, x, y, op)
    A.buffer = torch.empty(nbytes, dtype=torch.uint8, device=A.row_ptr.device)
    ct = _product_type(A, y)
    check(lib().aclsparseSpMVPreprocess(handle.raw, op, None, A.raw, x.raw, None, y.raw, ct,
                                        ACL_SPARSE_SPMV_ALG_DEFAULT, _ptr(A.buffer)), "aclsparseSpMVPreprocess")
    return A.buffer


def spmv(handle: Handle, A: CsrMatrix, x: DnVec, y: DnVec, alpha=1.0, beta=0.0,
         op: int = ACL_SPARSE_OP_NON_TRANSPOSE, buffer: torch.Tensor | None = None) -> None:
    """y = alpha * op(A) x + beta * y, enqueued on the handle's stream."""
    ct = _product_type(A, y)
    buf = buffer.data_ptr() if buffer is not None else None
    if ct == ACL_FLOAT and not handle.device_scalars:
        h, xd, yd = handle._h.value, x._d.value, y._d.value
        key = (h, xd, yd, buf, op)
        call = A._calls.get(key) or A._calls.pack(key, handle=h, a=A._d.value, x=xd, out=yd, buffer=buf, opA=op,
                                                  alg=ACL_SPARSE_SPMV_ALG_DEFAULT)
        status = lib().b200spPackedSpMV(call[1], alpha, beta)
        if status:
            check(status, "aclsparseSpMV")
        return
    a, b = _scalars(handle, alpha, beta, ct)
    status = lib().aclsparseSpMV(handle._h, op, a, A._d, x._d, b, y._d, ct, ACL_SPARSE_SPMV_ALG_DEFAULT, buf)
    if status:
        check(status, "aclsparseSpMV")


def spmm_buffer_size(handle: Handle, A: CsrMatrix, B: DnMat, C: DnMat, op_b: int = ACL_SPARSE_OP_NON_TRANSPOSE,
                     alg: int = ACL_SPARSE_SPMM_ALG_DEFAULT) -> int:
    size = c_size_t()
    ct = _product_type(A, C)
    check(lib().aclsparseSpMMGetBufferSize(handle.raw, ACL_SPARSE_OP_NON_TRANSPOSE, op_b, None, A.raw, B.raw, None,
                                           C.raw, ct, alg, byref(size)), "aclsparseSpMMGetBufferSize")
    return size.value


def spmm_preprocess(handle: Handle, A: CsrMatrix, B: DnMat, C: DnMat, op_b: int = ACL_SPARSE_OP_NON_TRANSPOSE,
                    alg: int = ACL_SPARSE_SPMM_ALG_DEFAULT):
    nbytes = spmm_buffer_size(handle, A, B, C, op_b, alg)
    A.buffer = torch.empty(nbytes, dtype=torch.uint8, device=A.row_ptr.device)
    ct = _product_type(A, C)
    check(lib().aclsparseSpMMPreprocess(handle.raw, ACL_SPARSE_OP_NON_TRANSPOSE, op_b, None, A.raw, B.raw, None,
                                        C.raw, ct, alg, _ptr(A.buffer)), "aclsparseSpMMPreprocess")
    return A.buffer


def spmm(handle: Handle, A: CsrMatrix, B: DnMat, C: DnMat, alpha=1.0, beta=0.0,
         op_b: int = ACL_SPARSE_OP_NON_TRANSPOSE, alg: int = ACL_SPARSE_SPMM_ALG_DEFAULT,
         buffer: torch.Tensor | None = None) -> None:
    """C = alpha * A op(B) + beta * C, enqueued on the handle's stream."""
    ct = _product_type(A, C)
    buf = buffer if buffer is not None else A.buffer
    if buf is None:
        buf = spmm_preprocess(handle, A, B, C, op_b, alg)
    if ct == ACL_FLOAT and not handle.device_scalars:
        h, bd, cd, ptr = handle._h.value, B._d.value, C._d.value, buf.data_ptr()
        key = (h, bd, cd, ptr, op_b, alg)
        call = A._calls.get(key) or A._calls.pack(key, handle=h, a=A._d.value, x=bd, out=cd, buffer=ptr,
                                                  opA=ACL_SPARSE_OP_NON_TRANSPOSE, opB=op_b, alg=alg)
        status = lib().b200spPackedSpMM(call[1], alpha, beta)
        if status:
            check(status, "aclsparseSpMM")
        return
    a, b = _scalars(handle, alpha, beta, ct)
    status = lib().aclsparseSpMM(handle._h, ACL_SPARSE_OP_NON_TRANSPOSE, op_b, a, A._d, B._d, b, C._d, ct, alg,
                                 buf.data_ptr())
    if status:
        check(status, "aclsparseSpMM")


class SpMVOpPlan:
    """aclsparseSpMVOp_bufferSize -> createDescr -> createPlan for one matrix; `run` is aclsparseSpMVOp.

    Z = alpha * A * X + beta * Y in fp32 with compensated row sums; Z may be Y.  The workspace of ALG2
    is owned by this object and lives as long as it does.
    """

    def __init__(self, handle: Handle, A: CsrMatrix, x: DnVec, y: DnVec, z: DnVec,
                 alg: int = ACL_SPARSE_SPMVOP_ALG_DEFAULT):
        self.handle, self.A = handle, A
        size = c_size_t()
        check(lib().aclsparseSpMVOp_bufferSize(handle.raw, ACL_SPARSE_OP_NON_TRANSPOSE, A.raw, x.raw, y.raw, z.raw,
                                               ACL_FLOAT, alg, byref(size)), "aclsparseSpMVOp_bufferSize")
        self.buffer_bytes = size.value
        self.buffer = (torch.empty(max(size.value, 1), dtype=torch.uint8, device=A.col_ind.device)
                       if alg == ACL_SPARSE_SPMVOP_ALG2 else None)
        self._descr, self._plan = c_void_p(), c_void_p()
        self._calls = _PackedCalls()
        check(lib().aclsparseSpMVOp_createDescr(handle.raw, byref(self._descr), ACL_SPARSE_OP_NON_TRANSPOSE, A.raw,
                                                x.raw, y.raw, z.raw, ACL_FLOAT, alg,
                                                _ptr(self.buffer) if self.buffer is not None else None),
              "aclsparseSpMVOp_createDescr")
        check(lib().aclsparseSpMVOp_createPlan(handle.raw, self._descr, byref(self._plan), None, 0),
              "aclsparseSpMVOp_createPlan")

    def run(self, x: DnVec, y: DnVec, z: DnVec, alpha=1.0, beta=0.0) -> None:
        if not self.handle.device_scalars:
            h, xd, yd, zd = self.handle._h.value, x._d.value, y._d.value, z._d.value
            key = (h, xd, yd, zd)
            call = self._calls.get(key) or self._calls.pack(key, handle=h, a=self._plan.value, x=xd, y=yd, out=zd)
            status = lib().b200spPackedSpMVOp(call[1], alpha, beta)
            if status:
                check(status, "aclsparseSpMVOp")
            return
        a, b = _scalars(self.handle, alpha, beta, ACL_FLOAT)
        status = lib().aclsparseSpMVOp(self.handle._h, self._plan, a, b, x._d, y._d, z._d)
        if status:
            check(status, "aclsparseSpMVOp")

    def close(self) -> None:
        self._calls.clear()
        if self._plan:
            lib().aclsparseSpMVOp_destroyPlan(self._plan)
            self._plan = c_void_p()
        if self._descr:
            lib().aclsparseSpMVOp_destroyDescr(self._descr)
            self._descr = c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ---- token operators (include/b200sp_tokens.h) ----

class RouteRule(Structure):
    """b200spRouteRule: how experts are scored and chosen.  score 'softmax' or 'sigmoid'; experts in `groups` of which the
    `kept` best take part, by their best value ('max') or the sum of their two best ('top2')."""

    _fields_ = [("score", c_int32), ("groups", c_int32), ("groups_kept", c_int32), ("group_score", c_int32),
                ("renormalise", c_int32), ("scale", c_float)]

    def __init__(self, score: str = "softmax", groups: int = 1, kept: int = 1, group_score: str = "max",
                 renormalise: bool = True, scale: float = 1.0):
        super().__init__({"softmax": B200SP_ROUTE_SOFTMAX, "sigmoid": B200SP_ROUTE_SIGMOID}[score], groups, kept,
                         {"max": B200SP_GROUP_MAX, "top2": B200SP_GROUP_TOP2}[group_score], int(renormalise), scale)
        self.address = addressof(self)


def _float_scalars(handle: Handle, alpha, beta):
    """alpha and beta of a token operator; their defaults need no memory (NULL is 1 and 0)."""
    if handle.device_scalars:
        return (alpha if alpha is None else _ptr(alpha)), (beta if beta is None else _ptr(beta))
    return None if alpha == 1.0 else byref(c_float(alpha)), None if beta == 0.0 else byref(c_float(beta))


def embedding(handle: Handle, table: DnMat, tokens: DnVec, out: DnMat, alpha=1.0, beta=0.0) -> None:
    """out[i] = alpha * table[tokens[i]] + beta * out[i]; tokens int32 or int64, those outside the table are padding.
    (With device scalars, here and below: tensors, or None for the defaults.)"""
    a, b = _float_scalars(handle, alpha, beta)
    status = lib().b200spEmbedding(handle._h, a, table._d, tokens._d, b, out._d)
    if status:
        check(status, "b200spEmbedding")


def embedding_grad_buffer_size(handle: Handle, grad: DnMat, tokens: DnVec, d_table: DnMat) -> int:
    size = c_size_t()
    check(lib().b200spEmbeddingGradBufferSize(handle.raw, grad.raw, tokens.raw, d_table.raw, byref(size)),
          "b200spEmbeddingGradBufferSize")
    return size.value


def embedding_grad(handle: Handle, grad: DnMat, tokens: DnVec, d_table: DnMat, alpha=1.0, beta=0.0,
                   buffer: torch.Tensor | None = None) -> None:
    """d_table[v] = alpha * sum of grad[i] over tokens[i] == v + beta * d_table[v].  Without a buffer one is allocated."""
    if buffer is None:
        with torch.cuda.stream(handle.stream):  # memory that is this stream's, also when it is freed below
            buffer = torch.empty(embedding_grad_buffer_size(handle, grad, tokens, d_table), dtype=torch.uint8,
                                 device=d_table.values.device)
    a, b = _float_scalars(handle, alpha, beta)
    status = lib().b200spEmbeddingGrad(handle._h, a, grad._d, tokens._d, b, d_table._d, buffer.data_ptr())
    if status:
        check(status, "b200spEmbeddingGrad")


def route(handle: Handle, rule: RouteRule, logits: DnMat, bias: DnVec | None, R: CsrMatrix) -> None:
    """Writes R (tokens x experts, the same number of entries in every row): offsets, ascending columns and values."""
    if bias is not None and not bias._d:
        raise ValueError("route: the bias has been closed")  # its NULL would say that there is none
    status = lib().b200spRoute(handle._h, rule.address, logits._d, None if bias is None else bias._d, R._d)
    if status:
        check(status, "b200spRoute")


def route_grad(handle: Handle, rule: RouteRule, logits: DnMat, R: CsrMatrix, d_values: DnVec, d_logits: DnMat) -> None:
    """Gradient of the logits (whole) from that of R's values."""
    status = lib().b200spRouteGrad(handle._h, rule.address, logits._d, R._d, d_values._d, d_logits._d)
    if status:
        check(status, "b200spRouteGrad")


_ROWS = {"tokens": B200SP_ROWS_OF_TOKENS, "entries": B200SP_ROWS_OF_ENTRIES}


def experts_buffer_size(handle: Handle, R: CsrMatrix, X: DnMat, W: DnMat, Y: DnMat, transpose: bool = True,
                        rows: str = "tokens") -> int:
    size = c_size_t()
    check(lib().b200spExpertsMMBufferSize(handle.raw, ACL_SPARSE_OP_TRANSPOSE if transpose else ACL_SPARSE_OP_NON_TRANSPOSE,
                                          _ROWS[rows], R.raw, X.raw, W.raw, Y.raw, byref(size)), "b200spExpertsMMBufferSize")
    return size.value


def experts_grad_buffer_size(handle: Handle, R: CsrMatrix, dY: DnMat, X: DnMat, dW: DnMat, rows: str = "tokens") -> int:
    size = c_size_t()
    check(lib().b200spExpertsGradBufferSize(handle.raw, _ROWS[rows], R.raw, dY.raw, X.raw, dW.raw, byref(size)),
          "b200spExpertsGradBufferSize")
    return size.value


def experts_preprocess(handle: Handle, R: CsrMatrix, buffer: torch.Tensor) -> None:
    """Orders R's entries by expert in the buffer, for the products that follow with it."""
    status = lib().b200spExpertsPreprocess(handle._h, R._d, buffer.data_ptr())
    if status:
        check(status, "b200spExpertsPreprocess")


def experts_mm(handle: Handle, R: CsrMatrix, X: DnMat, W: DnMat, Y: DnMat, alpha=1.0, beta=0.0, transpose: bool = True,
               rows: str = "tokens", buffer: torch.Tensor | None = None) -> None:
    """Y[i] = alpha * X[row of entry i] * op(W of its expert) + beta * Y[i]; W: the experts' matrices stacked."""
    a, b = _float_scalars(handle, alpha, beta)
    status = lib().b200spExpertsMM(handle._h, ACL_SPARSE_OP_TRANSPOSE if transpose else ACL_SPARSE_OP_NON_TRANSPOSE,
                                   _ROWS[rows], a, R._d, X._d, W._d, b, Y._d, None if buffer is None else buffer.data_ptr())
    if status:
        check(status, "b200spExpertsMM")


def experts_grad(handle: Handle, R: CsrMatrix, dY: DnMat, X: DnMat, dW: DnMat, alpha=1.0, beta=0.0, rows: str = "tokens",
                 buffer: torch.Tensor | None = None) -> None:
    """dW of every expert = alpha * sum over its entries of dY[i]^T X[row of entry i] + beta * dW."""
    a, b = _float_scalars(handle, alpha, beta)
    status = lib().b200spExpertsGrad(handle._h, _ROWS[rows], a, R._d, dY._d, X._d, b, dW._d,
                                     None if buffer is None else buffer.data_ptr())
    if status:
        check(status, "b200spExpertsGrad")


# ---- rows in the order of the experts and in 8 bits (include/b200sp_rows.h) ----

def _optional(what, name: str):
    """The descriptor of an argument that may be None.  (A closed one is refused: its NULL would say that there is none.)"""
    if what is None:
        return None
    if not what._d:
        raise ValueError(f"{name} has been closed")
    return what._d


def _address(buffer: torch.Tensor | None):
    return None if buffer is None else buffer.data_ptr()


def experts_order_buffer_size(handle: Handle, R: CsrMatrix) -> int:
    """For experts_preprocess and the calls below but experts_scaled_mm."""
    size = c_size_t()
    check(lib().b200spExpertsOrderBufferSize(handle.raw, R.raw, byref(size)), "b200spExpertsOrderBufferSize")
    return size.value


def experts_dispatch(handle: Handle, R: CsrMatrix, X: DnMat, S: DnMat, alpha=1.0, beta=0.0, offsets: DnVec | None = None,
                     buffer: torch.Tensor | None = None) -> None:
    """S[place of entry i] = alpha * X[token of entry i] + beta * S[place]: the tokens' rows in the order of the experts.
    offsets: takes the first row of every expert and the end of the last one's, int32."""
    a, b = _float_scalars(handle, alpha, beta)
    status = lib().b200spExpertsDispatch(handle._h, a, R._d, X._d, b, S._d, _optional(offsets, "experts_dispatch: offsets"),
                                         _address(buffer))
    if status:
        check(status, "b200spExpertsDispatch")


def experts_combine(handle: Handle, R: CsrMatrix, S: DnMat, out: DnMat, alpha=1.0, beta=0.0, weighted: bool = True,
                    buffer: torch.Tensor | None = None) -> None:
    """out[t] = alpha * sum over the entries i of token t of (R's value i if weighted, else 1) * S[place of i] + beta * out[t].
    Without weights it is the gradient of experts_dispatch."""
    a, b = _float_scalars(handle, alpha, beta)
    status = lib().b200spExpertsCombine(handle._h, B200SP_WEIGHTS_OF_R if weighted else B200SP_WEIGHTS_NONE, a, R._d, S._d,
                                        b, out._d, _address(buffer))
    if status:
        check(status, "b200spExpertsCombine")


def experts_combine_grad(handle: Handle, R: CsrMatrix, d_out: DnMat, S: DnMat | None, d_S: DnMat,
                         d_values: DnVec | None = None, alpha=1.0, beta=0.0, buffer: torch.Tensor | None = None) -> None:
    """Gradients of the weighted experts_combine: of the rows, and with S and d_values of R's values."""
    a, b = _float_scalars(handle, alpha, beta)
    status = lib().b200spExpertsCombineGrad(handle._h, a, R._d, d_out._d, _optional(S, "experts_combine_grad: S"), b, d_S._d,
                                            _optional(d_values, "experts_combine_grad: d_values"), _address(buffer))
    if status:
        check(status, "b200spExpertsCombineGrad")


def quantise_rows(handle: Handle, X: DnMat, Q: DnMat, scales: DnVec) -> None:
    """Q = X in whole numbers of up to 127 (int8), every row by its largest absolute value, and the rows' scales."""
    status = lib().b200spQuantiseRows(handle._h, X._d, Q._d, scales._d)
    if status:
        check(status, "b200spQuantiseRows")


def experts_quantise(handle: Handle, R: CsrMatrix, X: DnMat, Q: DnMat, scales: DnVec, offsets: DnVec | None = None,
                     buffer: torch.Tensor | None = None) -> None:
    """quantise_rows of every token's row into the rows of its entries in the order of the experts."""
    status = lib().b200spExpertsQuantise(handle._h, R._d, X._d, Q._d, scales._d, _optional(offsets, "experts_quantise: offsets"),
                                         _address(buffer))
    if status:
        check(status, "b200spExpertsQuantise")


def scaled_mm_buffer_size(handle: Handle, X: DnMat, W: DnMat, Y: DnMat) -> int:
    """0 where the rows of X and W start on 16 bytes: no buffer is needed then."""
    size = c_size_t()
    check(lib().b200spScaledMMBufferSize(handle.raw, X.raw, W.raw, Y.raw, byref(size)), "b200spScaledMMBufferSize")
    return size.value


def scaled_mm(handle: Handle, X: DnMat, x_scales: DnVec, W: DnMat, w_scales: DnVec, Y: DnMat, alpha=1.0, beta=0.0,
              buffer: torch.Tensor | None = None) -> None:
    """Y[i][j] = alpha * x_scales[i] * w_scales[j] * <X[i], W[j]> + beta * Y[i][j]; X and W int8."""
    a, b = _float_scalars(handle, alpha, beta)
    status = lib().b200spScaledMM(handle._h, a, X._d, x_scales._d, W._d, w_scales._d, b, Y._d, _address(buffer))
    if status:
        check(status, "b200spScaledMM")


def experts_scaled_mm_buffer_size(handle: Handle, R: CsrMatrix, X: DnMat, W: DnMat, Y: DnMat) -> int:
    size = c_size_t()
    check(lib().b200spExpertsScaledMMBufferSize(handle.raw, R.raw, X.raw, W.raw, Y.raw, byref(size)),
          "b200spExpertsScaledMMBufferSize")
    return size.value


def experts_scaled_mm(handle: Handle, R: CsrMatrix, X: DnMat, x_scales: DnVec, W: DnMat, w_scales: DnVec, Y: DnMat, alpha=1.0,
                      beta=0.0, buffer: torch.Tensor | None = None) -> None:
    """scaled_mm of every expert's rows, in the order of the experts, by its own matrix; W: the experts' matrices stacked."""
    a, b = _float_scalars(handle, alpha, beta)
    status = lib().b200spExpertsScaledMM(handle._h, a, R._d, X._d, x_scales._d, W._d, w_scales._d, b, Y._d, _address(buffer))
    if status:
        check(status, "b200spExpertsScaledMM")
