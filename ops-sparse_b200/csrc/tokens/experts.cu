// The calls around a routing to experts but those in 8-bit products: the order of its entries (b200spExpertsPreprocess), products of the rows of tokens with the
// experts' matrices and their gradients (b200spExpertsMM, b200spExpertsGrad; experts_tensor.cuh), rows in the order of the experts, back, and in 8 bits
// (b200spExpertsDispatch, b200spExpertsCombine, b200spExpertsCombineGrad, b200spExpertsQuantise, b200spQuantiseRows; experts_rows.cuh).
//
// The entries of R, in CSR order, are sorted by expert once (b200spExpertsPreprocess); a product then takes the entries of one
// expert after the other.  Its rows are gathered from X as they lie and its results stored in the rows of their
// entries: nothing is laid out in between.
#include <algorithm>
#include <type_traits>

#include "b200sp_rows.h"
#include "b200sp_tokens.h"
#include "tokens/common.cuh"
#include "tokens/experts_plan.cuh"
#include "tokens/rows.cuh"
#include "tokens/sort.cuh"
#include "tokens/tensor.cuh"

namespace {

using namespace b200sp_tokens;

// ---------------------------------------------------------------- the order of the entries

__global__ void __launch_bounds__(kSortThreads, 1) ExpertsOrderKernel(const SortArgs s, const int *__restrict__ rowPtr, int rows,
                                                                     int *__restrict__ rowOf, int *__restrict__ placeOf,
                                                                     int *__restrict__ offsets, int4 *header, const int4 mark,
                                                                     const uint64_t number)
{
    extern __shared__ unsigned char sSort[];
    b200sp::WaitForPrevious();
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        header[0] = mark;
        *reinterpret_cast<uint64_t *>(header + 1) = number;
    }
    ClusterSort<int>(s, sSort, [&](int, int entry, int to) {
        // rows are of about the same length: the first guess is nearly always right
        int r = (int)((long long)entry * rows / s.count);
        if (__ldg(rowPtr + r) > entry || __ldg(rowPtr + r + 1) <= entry) {
            int lo = 0, hi = rows;  // the last row that starts at or before the entry
            while (hi - lo > 1) {
                const int mid = lo + ((hi - lo) >> 1);
                if (__ldg(rowPtr + mid) <= entry) lo = mid;
                else hi = mid;
            }
            r = lo;
        }
        rowOf[to] = r;
        placeOf[entry] = to;
    });
    if (s.passes > 1 && blockIdx.x == 0) {
        for (int e = threadIdx.x; e <= s.limit + 1; e += kSortThreads) {
            int lo = 0, hi = s.count;
            while (lo < hi) {
                const int mid = lo + ((hi - lo) >> 1);
                if (__ldcg(s.keyA + mid) < e) lo = mid + 1;
                else hi = mid;
            }
            offsets[e] = lo;
        }
    }
}

// ---------------------------------------------------------------- operands that do not start on 16 bytes

// Rows of 16-bit elements into rows of a multiple of eight, zeros behind the last: what the copies of the products need.  A thread writes 16
// bytes, read two at a time, which is what bounds it: 2048 tokens, four of 64 experts, 1001 x 777 take 127 us, 1008 x 784 without copies 35.
// offsets: with rowsEach > 0 the rows are those of experts, as many each, and one without entries is left out.
__global__ void __launch_bounds__(256) ExpertsAlignKernel(const uint16_t *__restrict__ from, long long rows, int cols, long long ld,
                                                          uint4 *__restrict__ to, const int *__restrict__ offsets, int rowsEach)
{
    b200sp::WaitForPrevious();
    const int pieces = (cols + 7) / 8;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < rows * pieces; i += (long long)gridDim.x * 256) {
        const long long r = i / pieces;
        if (rowsEach > 0) {
            const int e = (int)(r / rowsEach);
            if (__ldg(offsets + e) == __ldg(offsets + e + 1)) continue;
        }
        const int c = (int)(i - r * pieces) * 8;
        const uint16_t *const row = from + r * ld + c;
        __align__(16) uint16_t v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = c + u < cols ? __ldg(row + u) : 0;
        to[i] = *reinterpret_cast<const uint4 *>(v);
    }
}

// ---------------------------------------------------------------- products

#include "tokens/experts_tensor.cuh"

// ---------------------------------------------------------------- rows in the order of the experts

#include "tokens/experts_rows.cuh"

// ---------------------------------------------------------------- host

bool Is16(aclDataType t) { return t == ACL_FLOAT16 || t == ACL_BF16; }

// rows of entries (Y or dY), X, and the stacked matrices (W or dW); `in`, `out`: of which the one is read and the other written.
aclsparseStatus_t CheckProduct(const aclsparseSpMatDescr *R, b200spExpertRows_t rowsOfX, const aclsparseDnMatDescr *X,
                               const aclsparseDnMatDescr *perEntry, const aclsparseDnMatDescr *stacked, const aclsparseDnMatDescr *in,
                               const aclsparseDnMatDescr *out)
{
    const aclsparseStatus_t st = CheckRouted(R);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (rowsOfX != B200SP_ROWS_OF_TOKENS && rowsOfX != B200SP_ROWS_OF_ENTRIES) return ACL_SPARSE_STATUS_INVALID_VALUE;
    for (const aclsparseDnMatDescr *m : {X, perEntry, stacked}) {
        const aclsparseStatus_t s = CheckDense(m);
        if (s != ACL_SPARSE_STATUS_SUCCESS) return s;
    }
    if (!Is16(X->valueType) || in->valueType != X->valueType) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (out->valueType != X->valueType && out->valueType != ACL_FLOAT) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (X->rows != (rowsOfX == B200SP_ROWS_OF_TOKENS ? R->rows : R->nnz) || perEntry->rows != R->nnz) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (stacked->rows % R->cols != 0) return ACL_SPARSE_STATUS_INVALID_VALUE;
    return ACL_SPARSE_STATUS_SUCCESS;
}

aclsparseStatus_t CheckMM(aclsparseOperation_t opW, b200spExpertRows_t rowsOfX, const aclsparseSpMatDescr *R, const aclsparseDnMatDescr *X,
                          const aclsparseDnMatDescr *W, const aclsparseDnMatDescr *Y)
{
    if (opW != ACL_SPARSE_OP_NON_TRANSPOSE && opW != ACL_SPARSE_OP_TRANSPOSE) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    const aclsparseStatus_t st = CheckProduct(R, rowsOfX, X, Y, W, W, Y);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    const int64_t n = W->rows / R->cols, d = W->cols;
    const bool t = opW == ACL_SPARSE_OP_TRANSPOSE;
    if (X->cols != (t ? d : n) || Y->cols != (t ? n : d)) return ACL_SPARSE_STATUS_INVALID_VALUE;
    return ACL_SPARSE_STATUS_SUCCESS;
}

aclsparseStatus_t CheckGrad(b200spExpertRows_t rowsOfX, const aclsparseSpMatDescr *R, const aclsparseDnMatDescr *dY,
                            const aclsparseDnMatDescr *X, const aclsparseDnMatDescr *dW)
{
    const aclsparseStatus_t st = CheckProduct(R, rowsOfX, X, dY, dW, dY, dW);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (dY->cols != dW->rows / R->cols || X->cols != dW->cols) return ACL_SPARSE_STATUS_INVALID_VALUE;
    return ACL_SPARSE_STATUS_SUCCESS;
}

MmaArgs ArgsOf(const aclsparseSpMatDescr *R, b200spExpertRows_t rowsOfX, const void *buffer, uint64_t number, const aclsparseDnMatDescr *stacked,
               const aclsparseDnMatDescr *out, const Scalars &sc)
{
    const PlanLayout L = PlanLayoutFor(R->nnz, R->cols);
    const char *p = BufferStart(buffer);
    MmaArgs a{};
    a.header = reinterpret_cast<const int4 *>(p);
    a.mark = HeaderOf(R->nnz, R->cols, R->rows);
    a.number = number;
    a.offsets = reinterpret_cast<const int *>(p + L.offsets);
    a.entries = reinterpret_cast<const int *>(p + L.entries);
    a.rows = reinterpret_cast<const int *>(p + L.rows);
    a.out = out->values;
    a.ldo = out->ld;
    a.vectors = RowsAligned(out);
    a.experts = (int)R->cols;
    a.n = (int)(stacked->rows / R->cols);
    a.d = (int)stacked->cols;
    a.byEntry = rowsOfX == B200SP_ROWS_OF_ENTRIES;
    a.sc = sc;
    return a;
}

// Bytes for a copy of an operand whose rows do not start on multiples of 16 bytes.
size_t AlignedBytes(const aclsparseDnMatDescr *m)
{
    return RowsAligned(m) ? 0 : AlignUp((size_t)m->rows * AlignUp((size_t)m->cols, 8) * 2, 256);
}
size_t BufferBytes(const aclsparseSpMatDescr *R, const aclsparseDnMatDescr *first, const aclsparseDnMatDescr *second)
{
    return PlanLayoutFor(R->nnz, R->cols).total + AlignedBytes(first) + AlignedBytes(second);
}
// An operand as the kernels read it: where it lies, or its copy at `room`, which moves on.
struct Operand {
    const void *values;
    long long ld;
    cudaError_t error;
};
Operand Aligned(const aclsparseDnMatDescr *m, char **room, cudaStream_t stream, const int *offsets = nullptr, int rowsEach = 0)
{
    const size_t bytes = AlignedBytes(m);
    if (bytes == 0) return {m->values, m->ld, cudaSuccess};
    char *const to = *room;
    *room += bytes;
    const long long pieces = m->rows * ((m->cols + 7) / 8);
    const unsigned blocks = (unsigned)std::min<long long>((pieces + 255) / 256, (long long)b200sp_sm_count() * 32);
    b200sp_note_launches(1);
    const cudaError_t e = b200sp::LaunchChained(ExpertsAlignKernel, blocks, 256, 0, stream, static_cast<const uint16_t *>(m->values),
                                                m->rows, (int)m->cols, m->ld, reinterpret_cast<uint4 *>(to), offsets, rowsEach);
    return {to, (long long)AlignUp((size_t)m->cols, 8), e};
}

}  // namespace

extern "C" {

int b200sp_experts_error(void)
{
    int flag = 0;
    if (cudaDeviceSynchronize() != cudaSuccess) return -1;  // the copy alone waits for no stream that the default one does not wait for
    return cudaMemcpyFromSymbol(&flag, gExpertsError, sizeof(flag)) == cudaSuccess ? flag : -1;
}

int b200sp_experts_error_clear(void)
{
    const int zero = 0;
    const cudaError_t e = cudaDeviceSynchronize();
    if (e != cudaSuccess) return (int)e;
    return (int)cudaMemcpyToSymbol(gExpertsError, &zero, sizeof(zero));
}

void b200sp_experts_wait_test(long long wait_cycles, unsigned extra_tx)
{
    gExpertsWaitCycles = wait_cycles > 0 ? wait_cycles : kMmaWaitCycles;
    gExpertsExtraTx = extra_tx;
}

aclsparseStatus_t b200spExpertsPreprocess(aclsparseHandle_t handle, aclsparseConstSpMatDescr_t matR, void *buffer)
{
    if (handle == nullptr) return ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR;
    const aclsparseStatus_t st = CheckRouted(matR);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (buffer == nullptr) return ACL_SPARSE_STATUS_INSUFFICIENT_RESOURCES;
    const OnDevice device(handle);
    std::lock_guard<std::mutex> lock(matR->expertsMutex);
    const uint64_t before = SameBuffer(matR, buffer) ? matR->experts.number : 0;
    const uint64_t generation = NoteWrite(buffer), number = before != 0 ? before : generation;  // generations are given once
    if (generation == 0) return ACL_SPARSE_STATUS_ALLOC_FAILED;
    const PlanLayout L = PlanLayoutFor(matR->nnz, matR->cols);
    char *const p = BufferStart(buffer);
    int *const offsets = reinterpret_cast<int *>(p + L.offsets);
    SortArgs s{};
    s.keys = matR->indices;
    s.count = (int)matR->nnz;
    s.limit = (int)matR->cols;
    SortPasses(s.limit, s.count, &s);
    s.keyA = reinterpret_cast<int *>(p + L.keyA);
    s.posA = reinterpret_cast<int *>(p + L.entries);
    s.keyB = reinterpret_cast<int *>(p + L.keyB);
    s.posB = reinterpret_cast<int *>(p + L.posB);
    s.offsets = s.passes == 1 ? offsets : nullptr;
    cudaError_t e = AllowShared<ExpertsOrderKernel>(kSortSharedMost);
    if (e == cudaSuccess) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)SortCtas(s.count));
        cfg.blockDim = dim3(kSortThreads);
        cfg.dynamicSmemBytes = (size_t)SortShared(s.digitBits, s.count <= kSortTile && s.passes > 1);
        cfg.stream = handle->stream;
        cudaLaunchAttribute attr[2] = {};
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = cfg.gridDim.x;
        attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 2;
        b200sp_note_launches(1);
        e = cudaLaunchKernelEx(&cfg, ExpertsOrderKernel, s, static_cast<const int *>(matR->offsets), (int)matR->rows,
                               reinterpret_cast<int *>(p + L.rows), reinterpret_cast<int *>(p + L.places), offsets,
                               reinterpret_cast<int4 *>(p), HeaderOf(matR->nnz, matR->cols, matR->rows), number);
    }
    matR->experts = {};
    if (e == cudaSuccess)
        matR->experts = {buffer, matR->offsets, matR->indices, matR->rows, matR->cols, matR->nnz, generation, number, Captures(handle->stream), false};
    return Finished(e, "b200spExpertsPreprocess");
}

aclsparseStatus_t b200spExpertsMMBufferSize(aclsparseHandle_t handle, aclsparseOperation_t opW, b200spExpertRows_t rowsOfX,
                                            aclsparseConstSpMatDescr_t matR, aclsparseConstDnMatDescr_t matX,
                                            aclsparseConstDnMatDescr_t matW, aclsparseConstDnMatDescr_t matY, size_t *bufferSize)
{
    if (handle == nullptr) return ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR;
    if (bufferSize == nullptr) return ACL_SPARSE_STATUS_INVALID_VALUE;
    const aclsparseStatus_t st = CheckMM(opW, rowsOfX, matR, matX, matW, matY);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    *bufferSize = NoteSize(matR, BufferBytes(matR, matX, matW));
    return ACL_SPARSE_STATUS_SUCCESS;
}

aclsparseStatus_t b200spExpertsMM(aclsparseHandle_t handle, aclsparseOperation_t opW, b200spExpertRows_t rowsOfX, const void *alpha,
                                  aclsparseConstSpMatDescr_t matR, aclsparseConstDnMatDescr_t matX, aclsparseConstDnMatDescr_t matW,
                                  const void *beta, aclsparseDnMatDescr_t matY, void *buffer)
{
    if (handle == nullptr) return ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR;
    const aclsparseStatus_t st = CheckMM(opW, rowsOfX, matR, matX, matW, matY);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (buffer == nullptr) return ACL_SPARSE_STATUS_INSUFFICIENT_RESOURCES;
    uint64_t number;
    if (!HoldsOrder(matR, buffer, handle->stream, &number) || !HasRoomFor(matR, AlignedBytes(matX) + AlignedBytes(matW))) return ACL_SPARSE_STATUS_INVALID_VALUE;
    const OnDevice device(handle);
    MmaArgs a = ArgsOf(matR, rowsOfX, buffer, number, matW, matY, ScalarsOf(handle, alpha, beta));
    char *room = BufferStart(buffer) + PlanLayoutFor(matR->nnz, matR->cols).total - 256;
    const Operand x = Aligned(matX, &room, handle->stream), w = Aligned(matW, &room, handle->stream, a.offsets, a.n);
    if (x.error != cudaSuccess || w.error != cudaSuccess) return Finished(x.error != cudaSuccess ? x.error : w.error, "b200spExpertsMM");
    a.x = x.values;
    a.ldx = x.ld;
    a.colsMost = TileColumns(matR->nnz, matR->cols);
    const bool transposed = opW == ACL_SPARSE_OP_TRANSPOSE;
    CUtensorMap mapW;
    if (!MapOf(&mapW, matW->valueType, w.values, a.d, a.n, w.ld, a.experts, transposed ? kMmaRows : kMmaDepth))
        return ACL_SPARSE_STATUS_INTERNAL_ERROR;
    const cudaError_t e = WithType(matX->valueType, [&](auto in) {
        return WithType(matY->valueType, [&](auto out) {
            using T = decltype(in);
            using Out = decltype(out);
            if constexpr (sizeof(T) == 2 && (sizeof(Out) == 4 || std::is_same_v<T, Out>))
                return transposed ? LaunchTensor<T, Out, Mode::kProductT>(a, mapW, handle->stream)
                                  : LaunchTensor<T, Out, Mode::kProductN>(a, mapW, handle->stream);
            else
                return cudaErrorInvalidValue;  // refused above
        });
    });
    return Finished(e, "b200spExpertsMM");
}

aclsparseStatus_t b200spExpertsGradBufferSize(aclsparseHandle_t handle, b200spExpertRows_t rowsOfX, aclsparseConstSpMatDescr_t matR,
                                              aclsparseConstDnMatDescr_t dY, aclsparseConstDnMatDescr_t matX,
                                              aclsparseConstDnMatDescr_t dW, size_t *bufferSize)
{
    if (handle == nullptr) return ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR;
    if (bufferSize == nullptr) return ACL_SPARSE_STATUS_INVALID_VALUE;
    const aclsparseStatus_t st = CheckGrad(rowsOfX, matR, dY, matX, dW);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    *bufferSize = NoteSize(matR, BufferBytes(matR, matX, dY));
    return ACL_SPARSE_STATUS_SUCCESS;
}

aclsparseStatus_t b200spExpertsGrad(aclsparseHandle_t handle, b200spExpertRows_t rowsOfX, const void *alpha,
                                    aclsparseConstSpMatDescr_t matR, aclsparseConstDnMatDescr_t dY, aclsparseConstDnMatDescr_t matX,
                                    const void *beta, aclsparseDnMatDescr_t dW, void *buffer)
{
    if (handle == nullptr) return ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR;
    const aclsparseStatus_t st = CheckGrad(rowsOfX, matR, dY, matX, dW);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (buffer == nullptr) return ACL_SPARSE_STATUS_INSUFFICIENT_RESOURCES;
    uint64_t number;
    if (!HoldsOrder(matR, buffer, handle->stream, &number) || !HasRoomFor(matR, AlignedBytes(matX) + AlignedBytes(dY))) return ACL_SPARSE_STATUS_INVALID_VALUE;
    const OnDevice device(handle);
    MmaArgs a = ArgsOf(matR, rowsOfX, buffer, number, dW, dW, ScalarsOf(handle, alpha, beta));
    char *room = BufferStart(buffer) + PlanLayoutFor(matR->nnz, matR->cols).total - 256;
    const Operand x = Aligned(matX, &room, handle->stream), y = Aligned(dY, &room, handle->stream);
    if (x.error != cudaSuccess || y.error != cudaSuccess) return Finished(x.error != cudaSuccess ? x.error : y.error, "b200spExpertsGrad");
    a.x = x.values;
    a.ldx = x.ld;
    a.dy = y.values;
    a.ldy = y.ld;
    a.colsMost = kMmaColsMost;
    const CUtensorMap none{};
    const cudaError_t e = WithType(matX->valueType, [&](auto in) {
        return WithType(dW->valueType, [&](auto out) {
            using T = decltype(in);
            using Out = decltype(out);
            if constexpr (sizeof(T) == 2 && (sizeof(Out) == 4 || std::is_same_v<T, Out>))
                return LaunchTensor<T, Out, Mode::kGrad>(a, none, handle->stream);
            else
                return cudaErrorInvalidValue;  // refused above
        });
    });
    return Finished(e, "b200spExpertsGrad");
}

// ---------------------------------------------------------------- rows in the order of the experts, and in 8 bits

aclsparseStatus_t b200spExpertsOrderBufferSize(aclsparseHandle_t handle, aclsparseConstSpMatDescr_t matR, size_t *bufferSize)
{
    if (handle == nullptr) return ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR;
    if (bufferSize == nullptr) return ACL_SPARSE_STATUS_INVALID_VALUE;
    const aclsparseStatus_t st = CheckRouted(matR);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    *bufferSize = NoteSize(matR, PlanLayoutFor(matR->nnz, matR->cols).total);
    return ACL_SPARSE_STATUS_SUCCESS;
}

aclsparseStatus_t b200spExpertsDispatch(aclsparseHandle_t handle, const void *alpha, aclsparseConstSpMatDescr_t matR,
                                        aclsparseConstDnMatDescr_t matX, const void *beta, aclsparseDnMatDescr_t matS,
                                        aclsparseDnVecDescr_t offsets, const void *buffer)
{
    if (handle == nullptr) return ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR;
    aclsparseStatus_t st = CheckRouted(matR);
    if (st == ACL_SPARSE_STATUS_SUCCESS) st = CheckDense(matX);
    if (st == ACL_SPARSE_STATUS_SUCCESS) st = CheckDense(matS);
    if (st == ACL_SPARSE_STATUS_SUCCESS) st = CheckStarts(matR, offsets);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (matS->valueType != matX->valueType && matS->valueType != ACL_FLOAT) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (matX->rows != matR->rows || matS->rows != matR->nnz || matX->cols != matS->cols) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (buffer == nullptr) return ACL_SPARSE_STATUS_INSUFFICIENT_RESOURCES;
    uint64_t number;
    if (!HoldsOrder(matR, buffer, handle->stream, &number)) return ACL_SPARSE_STATUS_INVALID_VALUE;
    const OnDevice device(handle);
    RowsArgs a = RowsOf(matR, buffer, number);
    a.width = (int)matX->cols;
    a.perToken = matX->values;
    a.ldToken = matX->ld;
    a.out = matS->values;
    a.ldOut = matS->ld;
    a.starts = offsets == nullptr ? nullptr : static_cast<int *>(offsets->values);
    a.sc = ScalarsOf(handle, alpha, beta);
    const bool vectors = RowsAligned(matX) && RowsAligned(matS);
    const cudaError_t e = WithTypes(matX->valueType, matS->valueType, [&](auto in, auto out) {
        using In = decltype(in);
        using Out = decltype(out);
        if constexpr (std::is_same_v<In, Out> || sizeof(Out) == 4) {
            const unsigned blocks = RowsBlocks(a.tokens * ((a.width + kStretch - 1) / kStretch), kDispatchCtas);
            b200sp_note_launches(1);
            return vectors ? b200sp::LaunchChained(ExpertsDispatchKernel<In, Out, true>, blocks, kRowsThreads, 0, handle->stream, a)
                           : b200sp::LaunchChained(ExpertsDispatchKernel<In, Out, false>, blocks, kRowsThreads, 0, handle->stream, a);
        } else {
            return cudaErrorInvalidValue;  // refused above
        }
    });
    return Finished(e, "b200spExpertsDispatch");
}

aclsparseStatus_t b200spExpertsCombine(aclsparseHandle_t handle, b200spExpertWeights_t weights, const void *alpha,
                                       aclsparseConstSpMatDescr_t matR, aclsparseConstDnMatDescr_t matS, const void *beta,
                                       aclsparseDnMatDescr_t matOut, const void *buffer)
{
    if (handle == nullptr) return ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR;
    if (weights != B200SP_WEIGHTS_NONE && weights != B200SP_WEIGHTS_OF_R) return ACL_SPARSE_STATUS_INVALID_VALUE;
    const bool weighted = weights == B200SP_WEIGHTS_OF_R;
    aclsparseStatus_t st = CheckRouted(matR);
    if (st == ACL_SPARSE_STATUS_SUCCESS) st = CheckDense(matS);
    if (st == ACL_SPARSE_STATUS_SUCCESS) st = CheckDense(matOut);
    if (st == ACL_SPARSE_STATUS_SUCCESS && weighted) st = CheckWeights(matR);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (UnlikeHalves(matS->valueType, matOut->valueType)) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (matOut->rows != matR->rows || matS->rows != matR->nnz || matOut->cols != matS->cols) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (buffer == nullptr) return ACL_SPARSE_STATUS_INSUFFICIENT_RESOURCES;
    uint64_t number;
    if (!HoldsOrder(matR, buffer, handle->stream, &number)) return ACL_SPARSE_STATUS_INVALID_VALUE;
    const OnDevice device(handle);
    RowsArgs a = RowsOf(matR, buffer, number);
    a.width = (int)matS->cols;
    a.perEntry = matS->values;
    a.ldEntry = matS->ld;
    a.out = matOut->values;
    a.ldOut = matOut->ld;
    a.weights = weighted ? matR->values : nullptr;
    a.weightType = matR->valueType;
    a.sc = ScalarsOf(handle, alpha, beta);
    const bool vectors = RowsAligned(matS) && RowsAligned(matOut);
    const cudaError_t e = WithTypes(matS->valueType, matOut->valueType, [&](auto in, auto out) {
        using In = decltype(in);
        using Out = decltype(out);
        const unsigned blocks = RowsBlocks(a.tokens * ((a.width + kStretch - 1) / kStretch), kCombineCtas);
        b200sp_note_launches(1);
        return vectors ? b200sp::LaunchChained(ExpertsCombineKernel<In, Out, true>, blocks, kRowsThreads, 0, handle->stream, a)
                       : b200sp::LaunchChained(ExpertsCombineKernel<In, Out, false>, blocks, kRowsThreads, 0, handle->stream, a);
    });
    return Finished(e, "b200spExpertsCombine");
}

aclsparseStatus_t b200spExpertsCombineGrad(aclsparseHandle_t handle, const void *alpha, aclsparseConstSpMatDescr_t matR,
                                           aclsparseConstDnMatDescr_t dOut, aclsparseConstDnMatDescr_t matS, const void *beta,
                                           aclsparseDnMatDescr_t dS, aclsparseDnVecDescr_t dValues, const void *buffer)
{
    if (handle == nullptr) return ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR;
    aclsparseStatus_t st = CheckRouted(matR);
    if (st == ACL_SPARSE_STATUS_SUCCESS) st = CheckDense(dOut);
    if (st == ACL_SPARSE_STATUS_SUCCESS) st = CheckDense(dS);
    if (st == ACL_SPARSE_STATUS_SUCCESS) st = CheckWeights(matR);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if ((matS == nullptr) != (dValues == nullptr)) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (UnlikeHalves(dOut->valueType, dS->valueType)) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (dOut->rows != matR->rows || dS->rows != matR->nnz || dOut->cols != dS->cols) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (matS != nullptr) {
        st = CheckDense(matS);
        if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
        if (matS->valueType != dS->valueType) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
        if (matS->rows != dS->rows || matS->cols != dS->cols) return ACL_SPARSE_STATUS_INVALID_VALUE;
        if (dValues->magic != b200sp::kDnVecMagic) return ACL_SPARSE_STATUS_INVALID_VALUE;
        if (!IsFloatType(dValues->valueType)) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
        st = CheckNumbers(dValues, matR->nnz, dValues->valueType, BytesOf(dValues->valueType));
        if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    }
    if (buffer == nullptr) return ACL_SPARSE_STATUS_INSUFFICIENT_RESOURCES;
    uint64_t number;
    if (!HoldsOrder(matR, buffer, handle->stream, &number)) return ACL_SPARSE_STATUS_INVALID_VALUE;
    const OnDevice device(handle);
    RowsArgs a = RowsOf(matR, buffer, number);
    a.width = (int)dOut->cols;
    a.perToken = dOut->values;
    a.ldToken = dOut->ld;
    a.out = dS->values;
    a.ldOut = dS->ld;
    if (matS != nullptr) {
        a.perEntry = matS->values;
        a.ldEntry = matS->ld;
        a.dValues = dValues->values;
        a.dValuesType = dValues->valueType;
    }
    a.weights = matR->values;
    a.weightType = matR->valueType;
    a.sc = ScalarsOf(handle, alpha, beta);
    const bool vectors = RowsAligned(dOut) && RowsAligned(dS) && (matS == nullptr || RowsAligned(matS));
    const cudaError_t e = WithTypes(dS->valueType, dOut->valueType, [&](auto s, auto g) {
        using T = decltype(s);
        using G = decltype(g);
        const bool cta = a.tokens < (long long)b200sp_sm_count() * kRowsWarps;
        const unsigned blocks = RowsBlocks(cta ? a.tokens * kRowsWarps : a.tokens, kGradCtas);
        b200sp_note_launches(1);
        if (cta)
            return vectors ? b200sp::LaunchChained(ExpertsCombineGradKernel<T, G, true, kRowsWarps>, blocks, kRowsThreads, 0, handle->stream, a)
                           : b200sp::LaunchChained(ExpertsCombineGradKernel<T, G, false, kRowsWarps>, blocks, kRowsThreads, 0, handle->stream, a);
        return vectors ? b200sp::LaunchChained(ExpertsCombineGradKernel<T, G, true, 1>, blocks, kRowsThreads, 0, handle->stream, a)
                       : b200sp::LaunchChained(ExpertsCombineGradKernel<T, G, false, 1>, blocks, kRowsThreads, 0, handle->stream, a);
    });
    return Finished(e, "b200spExpertsCombineGrad");
}

aclsparseStatus_t b200spQuantiseRows(aclsparseHandle_t handle, aclsparseConstDnMatDescr_t matX, aclsparseDnMatDescr_t matQ,
                                     aclsparseDnVecDescr_t scales)
{
    if (handle == nullptr) return ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR;
    aclsparseStatus_t st = CheckDense(matX);
    if (st == ACL_SPARSE_STATUS_SUCCESS) st = CheckBytes(matQ);
    if (st == ACL_SPARSE_STATUS_SUCCESS) st = CheckNumbers(scales, matQ->rows, ACL_FLOAT, 4);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (matX->rows != matQ->rows || matX->cols != matQ->cols) return ACL_SPARSE_STATUS_INVALID_VALUE;
    const OnDevice device(handle);
    RowsArgs a{};
    a.tokens = matX->rows;
    a.width = (int)matX->cols;
    a.perToken = matX->values;
    a.ldToken = matX->ld;
    a.out = matQ->values;
    a.ldOut = matQ->ld;
    a.scales = static_cast<float *>(scales->values);
    const cudaError_t e = WithType(matX->valueType, [&](auto x) {
        return LaunchQuantise<decltype(x), false>(a, QuantiseVectors(matX, matQ), handle->stream);
    });
    return Finished(e, "b200spQuantiseRows");
}

aclsparseStatus_t b200spExpertsQuantise(aclsparseHandle_t handle, aclsparseConstSpMatDescr_t matR, aclsparseConstDnMatDescr_t matX,
                                        aclsparseDnMatDescr_t matQ, aclsparseDnVecDescr_t scales, aclsparseDnVecDescr_t offsets,
                                        const void *buffer)
{
    if (handle == nullptr) return ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR;
    aclsparseStatus_t st = CheckRouted(matR);
    if (st == ACL_SPARSE_STATUS_SUCCESS) st = CheckDense(matX);
    if (st == ACL_SPARSE_STATUS_SUCCESS) st = CheckBytes(matQ);
    if (st == ACL_SPARSE_STATUS_SUCCESS) st = CheckNumbers(scales, matQ->rows, ACL_FLOAT, 4);
    if (st == ACL_SPARSE_STATUS_SUCCESS) st = CheckStarts(matR, offsets);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (matX->rows != matR->rows || matQ->rows != matR->nnz || matX->cols != matQ->cols) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (buffer == nullptr) return ACL_SPARSE_STATUS_INSUFFICIENT_RESOURCES;
    uint64_t number;
    if (!HoldsOrder(matR, buffer, handle->stream, &number)) return ACL_SPARSE_STATUS_INVALID_VALUE;
    const OnDevice device(handle);
    RowsArgs a = RowsOf(matR, buffer, number);
    a.width = (int)matX->cols;
    a.perToken = matX->values;
    a.ldToken = matX->ld;
    a.out = matQ->values;
    a.ldOut = matQ->ld;
    a.scales = static_cast<float *>(scales->values);
    a.starts = offsets == nullptr ? nullptr : static_cast<int *>(offsets->values);
    const cudaError_t e = WithType(matX->valueType, [&](auto x) {
        return LaunchQuantise<decltype(x), true>(a, QuantiseVectors(matX, matQ), handle->stream);
    });
    return Finished(e, "b200spExpertsQuantise");
}

}  // extern "C"
