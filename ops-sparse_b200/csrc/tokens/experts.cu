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

// The buffer: where every expert's entries begin (one more group: entries of no expert), the entries by expert and the
// rows of R that they lie in; and the sort's own arrays.
struct PlanLayout {
    size_t offsets, entries, rows, keyA, keyB, posB, total;
};
PlanLayout PlanLayoutFor(long long nnz, long long experts)
{
    PlanLayout L;
    const size_t words = AlignUp(sizeof(int) * (size_t)nnz, 256);
    L.offsets = 0;
    L.entries = AlignUp(sizeof(int) * (size_t)(experts + 2), 256);
    L.rows = L.entries + words;
    L.keyA = L.rows + words;
    L.keyB = L.keyA + words;
    L.posB = L.keyB + words;
    L.total = L.posB + words + 256;  // any address is accepted
    return L;
}

// ---------------------------------------------------------------- the order of the entries

__global__ void __launch_bounds__(kSortThreads, 1) ExpertsOrderKernel(const SortArgs s, const int *__restrict__ rowPtr, int rows,
                                                                     int *__restrict__ rowOf, int *__restrict__ offsets)
{
    extern __shared__ unsigned char sSort[];
    b200sp::WaitForPrevious();
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
                const int mid = (lo + hi) >> 1;
                if (__ldcg(s.keyA + mid) < e) lo = mid + 1;
                else hi = mid;
            }
            offsets[e] = lo;
        }
    }
}

// ---------------------------------------------------------------- products

struct ProductArgs {
    const int *offsets, *entries, *rows;
    const void *x, *w, *dy;
    void *out;
    long long ldx, ldw, ldy, ldo;
    int experts, nnz;
    int n, d;          // rows and columns of an expert's matrix
    int byEntry;       // X has a row per entry
    int transposed;    // opW = T
    Scalars sc;
};

constexpr int kTile = 64, kDepth = 16;

// Which expert's which tile of 64 entries.  Group `experts` has the entries of no expert.
__device__ __forceinline__ bool TileOf(const int *offsets, int groups, int tile, int *expert, int *first, int *end)
{
    for (int e = 0; e < groups; ++e) {
        const int lo = __ldg(offsets + e), hi = __ldg(offsets + e + 1), tiles = (hi - lo + kTile - 1) / kTile;
        if (tile < tiles) {
            *expert = e;
            *first = lo + tile * kTile;
            *end = hi;
            return true;
        }
        tile -= tiles;
    }
    return false;
}

template <typename T, typename Out> __global__ void __launch_bounds__(256) ExpertsSimpleKernel(const ProductArgs a)
{
    __shared__ float sX[kDepth][kTile + 4], sW[kDepth][kTile + 4];
    b200sp::WaitForPrevious();
    int expert, first, end;
    if (!TileOf(a.offsets, a.experts + 1, blockIdx.y, &expert, &first, &end)) return;
    const int cols = a.transposed ? a.n : a.d, depth = a.transposed ? a.d : a.n, c0 = blockIdx.x * kTile;
    const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
    float acc[4][4] = {};
    if (expert < a.experts) {
        const T *const w = static_cast<const T *>(a.w) + (long long)expert * a.n * a.ldw;
        for (int k0 = 0; k0 < depth; k0 += kDepth) {
            for (int i = tid; i < kTile * kDepth; i += 256) {
                const int r = i / kDepth, k = k0 + i % kDepth;
                float v = 0.0f;
                if (first + r < end && k < depth) {
                    const long long row = a.byEntry ? __ldg(a.entries + first + r) : __ldg(a.rows + first + r);
                    v = ToFloat(static_cast<const T *>(a.x)[row * a.ldx + k]);
                }
                sX[i % kDepth][r] = v;
                const int c = a.transposed ? i / kDepth : i % kTile, kw = a.transposed ? i % kDepth : i / kTile;
                float u = 0.0f;
                if (c0 + c < cols && k0 + kw < depth)
                    u = ToFloat(a.transposed ? w[(long long)(c0 + c) * a.ldw + k0 + kw] : w[(long long)(k0 + kw) * a.ldw + c0 + c]);
                sW[kw][c] = u;
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < kDepth; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sX[k][ty * 4 + i], sW[k][tx + 16 * j], acc[i][j]);
            __syncthreads();
        }
    }
    const float alpha = a.sc.Alpha(), beta = a.sc.Beta();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int at = first + ty * 4 + i;
        if (at >= end) continue;
        Out *const out = static_cast<Out *>(a.out) + __ldg(a.entries + at) * a.ldo;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = c0 + tx + 16 * j;
            if (c >= cols) continue;
            float v = alpha * acc[i][j];
            if (expert == a.experts) v = 0.0f;
            if (beta != 0.0f) v = fmaf(beta, ToFloat(out[c]), v);
            out[c] = FromFloat<Out>(v);
        }
    }
}

template <typename T, typename Out> __global__ void __launch_bounds__(256) ExpertsSimpleGradKernel(const ProductArgs a)
{
    __shared__ float sY[kDepth][kTile + 4], sX[kDepth][kTile + 4];
    b200sp::WaitForPrevious();
    const int expert = blockIdx.z, d0 = blockIdx.x * kTile, n0 = blockIdx.y * kTile;
    const int lo = __ldg(a.offsets + expert), hi = __ldg(a.offsets + expert + 1);
    const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
    float acc[4][4] = {};
    for (int k0 = lo; k0 < hi; k0 += kDepth) {
        for (int i = tid; i < kTile * kDepth; i += 256) {
            const int k = i / kTile, c = i % kTile;
            float y = 0.0f, x = 0.0f;
            if (k0 + k < hi) {
                const long long entry = __ldg(a.entries + k0 + k), row = a.byEntry ? entry : __ldg(a.rows + k0 + k);
                if (n0 + c < a.n) y = ToFloat(static_cast<const T *>(a.dy)[entry * a.ldy + n0 + c]);
                if (d0 + c < a.d) x = ToFloat(static_cast<const T *>(a.x)[row * a.ldx + d0 + c]);
            }
            sY[k][c] = y;
            sX[k][c] = x;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kDepth; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sY[k][ty * 4 + i], sX[k][tx + 16 * j], acc[i][j]);
        __syncthreads();
    }
    const float alpha = a.sc.Alpha(), beta = a.sc.Beta();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (n0 + ty * 4 + i >= a.n) continue;
        Out *const out = static_cast<Out *>(a.out) + ((long long)expert * a.n + n0 + ty * 4 + i) * a.ldo;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = d0 + tx + 16 * j;
            if (c >= a.d) continue;
            float v = lo < hi ? alpha * acc[i][j] : 0.0f;
            if (beta != 0.0f) v = fmaf(beta, ToFloat(out[c]), v);
            out[c] = FromFloat<Out>(v);
        }
    }
}

#include "tokens/experts_tensor.cuh"

// ---------------------------------------------------------------- host

aclsparseStatus_t CheckRouted(const aclsparseSpMatDescr *R)
{
    if (R == nullptr) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (R->format != ACL_SPARSE_FORMAT_CSR) return ACL_SPARSE_STATUS_MATRIX_TYPE_NOT_SUPPORTED;
    const aclsparseStatus_t idx = b200sp::CheckExecIndexTypes(R->offsetType, R->indexType);
    if (idx != ACL_SPARSE_STATUS_SUCCESS) return idx;
    if (R->base != ACL_SPARSE_INDEX_BASE_ZERO) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (R->cols > kMaxExperts || R->rows >= INT32_MAX || R->nnz >= INT32_MAX) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (R->rows == 0 || R->cols == 0 || R->nnz == 0) return ACL_SPARSE_STATUS_INVALID_VALUE;  // no dense operand has as few rows
    if (R->offsets == nullptr || R->indices == nullptr) return ACL_SPARSE_STATUS_INVALID_VALUE;
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

// Whether the buffer still holds the order of R's entries.
bool HoldsOrder(const aclsparseSpMatDescr *R, const void *buffer)
{
    std::lock_guard<std::mutex> lock(R->expertsMutex);
    const b200sp::ExpertsPlan &p = R->experts;
    return buffer != nullptr && p.buffer == buffer && p.offsets == R->offsets && p.indices == R->indices && p.rows == R->rows &&
           p.cols == R->cols && p.nnz == R->nnz && p.generation != 0 && p.generation == b200sp::BufferGeneration(buffer);
}

ProductArgs ArgsOf(const aclsparseSpMatDescr *R, b200spExpertRows_t rowsOfX, void *buffer, const Scalars &sc)
{
    const PlanLayout L = PlanLayoutFor(R->nnz, R->cols);
    const char *p = BufferStart(buffer);
    ProductArgs a{};
    a.offsets = reinterpret_cast<const int *>(p + L.offsets);
    a.entries = reinterpret_cast<const int *>(p + L.entries);
    a.rows = reinterpret_cast<const int *>(p + L.rows);
    a.experts = (int)R->cols;
    a.nnz = (int)R->nnz;
    a.byEntry = rowsOfX == B200SP_ROWS_OF_ENTRIES;
    a.sc = sc;
    return a;
}

MmaArgs TensorArgsOf(const ProductArgs &a, const aclsparseSpMatDescr *R)
{
    MmaArgs t{};
    t.offsets = a.offsets;
    t.entries = a.entries;
    t.rows = a.rows;
    t.out = a.out;
    t.dy = a.dy;
    t.x = a.x;
    t.ldy = a.ldy;
    t.ldx = a.ldx;
    t.ldo = a.ldo;
    t.experts = (int)R->cols;
    t.n = a.n;
    t.d = a.d;
    t.byEntry = a.byEntry;
    t.sc = a.sc;
    return t;
}

}  // namespace

extern "C" {

int b200sp_experts_error(void)
{
    int flag = 0;
    return cudaMemcpyFromSymbol(&flag, gExpertsError, sizeof(flag)) == cudaSuccess ? flag : -1;
}

int b200sp_experts_error_clear(void)
{
    const int zero = 0;
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
    const uint64_t generation = NoteWrite(buffer);
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
    cudaError_t e = cudaFuncSetAttribute(ExpertsOrderKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSortSharedMost);
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
                               reinterpret_cast<int *>(p + L.rows), offsets);
    }
    std::lock_guard<std::mutex> lock(matR->expertsMutex);
    matR->experts = {};
    if (e == cudaSuccess) matR->experts = {buffer, matR->offsets, matR->indices, matR->rows, matR->cols, matR->nnz, generation};
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
    *bufferSize = PlanLayoutFor(matR->nnz, matR->cols).total;
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
    if (!HoldsOrder(matR, buffer)) return ACL_SPARSE_STATUS_INVALID_VALUE;
    const OnDevice device(handle);
    ProductArgs a = ArgsOf(matR, rowsOfX, buffer, ScalarsOf(handle, alpha, beta));
    a.x = matX->values;
    a.w = matW->values;
    a.out = matY->values;
    a.ldx = matX->ld;
    a.ldw = matW->ld;
    a.ldo = matY->ld;
    a.n = (int)(matW->rows / matR->cols);
    a.d = (int)matW->cols;
    a.transposed = opW == ACL_SPARSE_OP_TRANSPOSE;
    if (RowsAligned(matX) && RowsAligned(matW)) {
        MmaArgs t = TensorArgsOf(a, matR);
        t.colsMost = TileColumns(matR->nnz, matR->cols);
        t.vectors = RowsAligned(matY);
        CUtensorMap mapW;
        if (!MapOf(&mapW, matW->valueType, matW->values, a.d, a.n, matW->ld, (int)matR->cols, a.transposed ? kMmaRows : kMmaDepth))
            return ACL_SPARSE_STATUS_INTERNAL_ERROR;
        const cudaError_t e = WithType(matX->valueType, [&](auto in) {
            return WithType(matY->valueType, [&](auto out) {
                using T = decltype(in);
                using Out = decltype(out);
                if constexpr (sizeof(T) == 2 && (sizeof(Out) == 4 || std::is_same_v<T, Out>))
                    return a.transposed ? LaunchTensor<T, Out, Mode::kProductT>(t, mapW, handle->stream)
                                        : LaunchTensor<T, Out, Mode::kProductN>(t, mapW, handle->stream);
                else
                    return cudaErrorInvalidValue;  // refused above
            });
        });
        return Finished(e, "b200spExpertsMM");
    }
    const dim3 grid((unsigned)((matY->cols + kTile - 1) / kTile), (unsigned)((a.nnz + kTile - 1) / kTile + a.experts + 1));
    b200sp_note_launches(1);
    WithType(matX->valueType, [&](auto in) {
        WithType(matY->valueType, [&](auto out) {
            if constexpr (sizeof(in) == 2) ExpertsSimpleKernel<decltype(in), decltype(out)><<<grid, 256, 0, handle->stream>>>(a);
        });
    });
    return Finished(cudaGetLastError(), "b200spExpertsMM");
}

aclsparseStatus_t b200spExpertsGradBufferSize(aclsparseHandle_t handle, b200spExpertRows_t rowsOfX, aclsparseConstSpMatDescr_t matR,
                                              aclsparseConstDnMatDescr_t dY, aclsparseConstDnMatDescr_t matX,
                                              aclsparseConstDnMatDescr_t dW, size_t *bufferSize)
{
    if (handle == nullptr) return ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR;
    if (bufferSize == nullptr) return ACL_SPARSE_STATUS_INVALID_VALUE;
    const aclsparseStatus_t st = CheckGrad(rowsOfX, matR, dY, matX, dW);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    *bufferSize = PlanLayoutFor(matR->nnz, matR->cols).total;
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
    if (!HoldsOrder(matR, buffer)) return ACL_SPARSE_STATUS_INVALID_VALUE;
    const OnDevice device(handle);
    ProductArgs a = ArgsOf(matR, rowsOfX, buffer, ScalarsOf(handle, alpha, beta));
    a.x = matX->values;
    a.dy = dY->values;
    a.out = dW->values;
    a.ldx = matX->ld;
    a.ldy = dY->ld;
    a.ldo = dW->ld;
    a.n = (int)(dW->rows / matR->cols);
    a.d = (int)dW->cols;
    if (RowsAligned(matX) && RowsAligned(dY)) {
        MmaArgs t = TensorArgsOf(a, matR);
        t.colsMost = kMmaColsMost;
        t.vectors = RowsAligned(dW);
        const CUtensorMap none{};
        const cudaError_t e = WithType(matX->valueType, [&](auto in) {
            return WithType(dW->valueType, [&](auto out) {
                using T = decltype(in);
                using Out = decltype(out);
                if constexpr (sizeof(T) == 2 && (sizeof(Out) == 4 || std::is_same_v<T, Out>))
                    return LaunchTensor<T, Out, Mode::kGrad>(t, none, handle->stream);
                else
                    return cudaErrorInvalidValue;  // refused above
            });
        });
        return Finished(e, "b200spExpertsGrad");
    }
    const dim3 grid((unsigned)((a.d + kTile - 1) / kTile), (unsigned)((a.n + kTile - 1) / kTile), (unsigned)a.experts);
    b200sp_note_launches(1);
    WithType(matX->valueType, [&](auto in) {
        WithType(dW->valueType, [&](auto out) {
            if constexpr (sizeof(in) == 2) ExpertsSimpleGradKernel<decltype(in), decltype(out)><<<grid, 256, 0, handle->stream>>>(a);
        });
    });
    return Finished(cudaGetLastError(), "b200spExpertsGrad");
}

}  // extern "C"
