// b200spExpertsMM, b200spExpertsGrad: products of the rows of tokens with the matrices of the experts that they are routed to.
//
// The entries of R, in CSR order, are sorted by expert once (b200spExpertsPreprocess); a product then takes the entries of one
// expert after the other.  Its rows are gathered from X as they lie and its results stored in the rows of their
// entries: nothing is laid out in between.
#include <algorithm>
#include <type_traits>

#include "b200sp_tokens.h"
#include "tokens/common.cuh"
#include "tokens/sort.cuh"

namespace {

using namespace b200sp_tokens;

constexpr int kMaxExperts = 1024;

// The buffer: what R it is the order of; where every expert's entries begin (one more group: entries of no expert), the entries by
// expert and the rows of R that they lie in; and the sort's own arrays.
struct PlanLayout {
    size_t offsets, entries, rows, keyA, keyB, posB, total;
};
PlanLayout PlanLayoutFor(long long nnz, long long experts)
{
    PlanLayout L;
    const size_t words = AlignUp(sizeof(int) * (size_t)nnz, 256);
    L.offsets = 256;  // the header lies before
    L.entries = L.offsets + AlignUp(sizeof(int) * (size_t)(experts + 2), 256);
    L.rows = L.entries + words;
    L.keyA = L.rows + words;
    L.keyB = L.keyA + words;
    L.posB = L.keyB + words;
    L.total = L.posB + words + 256;  // any address is accepted
    return L;
}

// A product follows the order only if the buffer starts with this: the sizes that its entries and rows are below, then a number of the order.
// A Preprocess that was captured and has not been replayed yet has written nothing: an eager product after it wants its number.  (Others do
// not: a graph's products follow the order that is there when they are replayed, whoever made it last.)  All that order the entries of one R
// in one buffer write the same number, so that any of them may have been the last to run, until an eager b200spRoute gives R other columns.
constexpr int kOrderMark = 0x45585031;
inline int4 HeaderOf(long long nnz, long long experts, long long rows) { return make_int4(kOrderMark, (int)nnz, (int)experts, (int)rows); }

// ---------------------------------------------------------------- the order of the entries

__global__ void __launch_bounds__(kSortThreads, 1) ExpertsOrderKernel(const SortArgs s, const int *__restrict__ rowPtr, int rows,
                                                                     int *__restrict__ rowOf, int *__restrict__ offsets, int4 *header,
                                                                     const int4 mark, const uint64_t number)
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

// ---------------------------------------------------------------- host

aclsparseStatus_t CheckRouted(const aclsparseSpMatDescr *R)
{
    if (R == nullptr) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (R->format != ACL_SPARSE_FORMAT_CSR) return ACL_SPARSE_STATUS_MATRIX_TYPE_NOT_SUPPORTED;
    const aclsparseStatus_t idx = b200sp::CheckExecIndexTypes(R->offsetType, R->indexType);
    if (idx != ACL_SPARSE_STATUS_SUCCESS) return idx;
    if (R->base != ACL_SPARSE_INDEX_BASE_ZERO) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (R->cols > kMaxExperts || R->rows >= INT32_MAX || R->nnz > kMostCounted) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (R->rows == 0 || R->cols == 0 || R->nnz == 0) return ACL_SPARSE_STATUS_INVALID_VALUE;  // no dense operand has as few rows
    if (R->offsets == nullptr || R->indices == nullptr) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (!OnBoundary(R->offsets, 4) || !OnBoundary(R->indices, 4)) return ACL_SPARSE_STATUS_INVALID_VALUE;
    return ACL_SPARSE_STATUS_SUCCESS;
}

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

char *BufferStart(const void *buffer) { return reinterpret_cast<char *>(AlignUp(reinterpret_cast<uintptr_t>(buffer), 256)); }

// Whether the buffer is the one that R's entries were ordered in last, and no other call has written it since.
bool SameBuffer(const aclsparseSpMatDescr *R, const void *buffer)
{
    const b200sp::ExpertsPlan &p = R->experts;
    return buffer != nullptr && p.buffer == buffer && p.offsets == R->offsets && p.indices == R->indices && p.rows == R->rows &&
           p.cols == R->cols && p.nnz == R->nnz && p.generation != 0 && p.generation == b200sp::BufferGeneration(buffer);
}
// Whether the buffer still holds the order of R's entries; the number that it has to have, 0: any.
bool HoldsOrder(const aclsparseSpMatDescr *R, const void *buffer, cudaStream_t stream, uint64_t *number)
{
    std::lock_guard<std::mutex> lock(R->expertsMutex);
    *number = R->experts.captured && !Captures(stream) ? R->experts.number : 0;
    return SameBuffer(R, buffer) && !R->experts.stale;
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
// What the BufferSize calls for this matrix have said at most.
size_t NoteSize(const aclsparseSpMatDescr *R, size_t bytes)
{
    std::lock_guard<std::mutex> lock(R->expertsMutex);
    R->expertsSized = std::max(R->expertsSized, (int64_t)bytes);
    return bytes;
}
// Whether the buffer may be taken to have room for copies of the operands, if any: what Preprocess writes it has.
bool HasRoom(const aclsparseSpMatDescr *R, const aclsparseDnMatDescr *first, const aclsparseDnMatDescr *second)
{
    if (AlignedBytes(first) + AlignedBytes(second) == 0) return true;
    std::lock_guard<std::mutex> lock(R->expertsMutex);
    return (int64_t)BufferBytes(R, first, second) <= R->expertsSized;
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
                               reinterpret_cast<int *>(p + L.rows), offsets, reinterpret_cast<int4 *>(p),
                               HeaderOf(matR->nnz, matR->cols, matR->rows), number);
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
    if (!HoldsOrder(matR, buffer, handle->stream, &number) || !HasRoom(matR, matX, matW)) return ACL_SPARSE_STATUS_INVALID_VALUE;
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
    if (!HoldsOrder(matR, buffer, handle->stream, &number) || !HasRoom(matR, matX, dY)) return ACL_SPARSE_STATUS_INVALID_VALUE;
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

}  // extern "C"
