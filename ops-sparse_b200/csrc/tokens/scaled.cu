// b200spScaledMM, b200spExpertsScaledMM: products in 8-bit integers with a scale for each row and channel.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "b200sp_bench.h"
#include "b200sp_rows.h"
#include "tokens/common.cuh"
#include "tokens/experts_plan.cuh"
#include "tokens/tensor.cuh"

namespace {

using namespace b200sp_tokens;

constexpr long long kMostDepth = 131071;  // sums of so many products of 8 bits are less than 2^31

// ---------------------------------------------------------------- operands that do not start on 16 bytes

// Rows of bytes into rows of a multiple of 16, zeros behind the last: what the copies of the products need.  A thread writes 16 bytes, from five words
// of four; only the first and last bytes of the matrix, whose words may reach beyond it, are read one by one.
__global__ void __launch_bounds__(256) ScaledAlignKernel(const uint8_t *__restrict__ from, long long rows, int cols, long long ld,
                                                         uint4 *__restrict__ to, const int4 *header, const int4 mark, const uint64_t number,
                                                         const int *__restrict__ offsets, int rowsEach)
{
    b200sp::WaitForPrevious();
    if (header != nullptr && !StartsWith(header, mark, number)) return;  // the product raises the flag
    const int pieces = (cols + 15) / 16;
    const uint8_t *const last = from + (rows - 1) * ld + cols;  // the end of what may be read
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < rows * pieces; i += (long long)gridDim.x * 256) {
        const long long r = i / pieces;
        if (rowsEach > 0) {  // an expert's without entries are left out
            const int e = (int)(r / rowsEach);
            if (__ldg(offsets + e) == __ldg(offsets + e + 1)) continue;
        }
        const int c = (int)(i - r * pieces) * 16, many = min(16, cols - c);
        const uint8_t *const at = from + r * ld + c;
        const uint8_t *const word = reinterpret_cast<const uint8_t *>(reinterpret_cast<uintptr_t>(at) & ~(uintptr_t)3);
        __align__(16) uint32_t v[4];
        if (word >= from && word + 20 <= last) {
            uint32_t w[5];
#pragma unroll
            for (int u = 0; u < 5; ++u) w[u] = __ldg(reinterpret_cast<const uint32_t *>(word) + u);
            const uint32_t shift = 8 * (uint32_t)(at - word);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                v[u] = __funnelshift_r(w[u], w[u + 1], shift);
                const int left = many - 4 * u;  // bytes that exist
                if (left < 4) v[u] = left <= 0 ? 0 : v[u] & ((1u << 8 * left) - 1);
            }
        } else {
            uint8_t *const bytes = reinterpret_cast<uint8_t *>(v);
#pragma unroll
            for (int u = 0; u < 16; ++u) bytes[u] = u < many ? at[u] : 0;
        }
        to[i] = *reinterpret_cast<const uint4 *>(v);
    }
}

// ---------------------------------------------------------------- products

#include "tokens/scaled_tensor.cuh"

// ---------------------------------------------------------------- host

aclsparseStatus_t CheckBytes(const aclsparseDnMatDescr *m)
{
    if (m == nullptr) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (m->order != ACL_SPARSE_ORDER_ROW || m->valueType != ACL_INT8) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (m->rows > INT32_MAX || m->cols > kMostDepth || m->ld > INT32_MAX) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    return m->values == nullptr ? ACL_SPARSE_STATUS_INVALID_VALUE : ACL_SPARSE_STATUS_SUCCESS;
}
aclsparseStatus_t CheckScales(const aclsparseDnVecDescr *v, int64_t size)
{
    if (v == nullptr || v->magic != b200sp::kDnVecMagic) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (v->valueType != ACL_FLOAT) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (v->size != size || v->values == nullptr || !OnBoundary(v->values, 4)) return ACL_SPARSE_STATUS_INVALID_VALUE;
    return ACL_SPARSE_STATUS_SUCCESS;
}

// experts: 1 without a routing.
aclsparseStatus_t CheckOperands(const aclsparseDnMatDescr *X, const aclsparseDnMatDescr *W, const aclsparseDnMatDescr *Y, int64_t experts)
{
    aclsparseStatus_t st = CheckBytes(X);
    if (st == ACL_SPARSE_STATUS_SUCCESS) st = CheckBytes(W);
    if (st == ACL_SPARSE_STATUS_SUCCESS) st = CheckDense(Y);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (X->rows > kMostCounted || W->rows > kMostCounted) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (X->cols != W->cols || X->rows != Y->rows || W->rows % experts != 0 || W->rows / experts != Y->cols) return ACL_SPARSE_STATUS_INVALID_VALUE;
    return ACL_SPARSE_STATUS_SUCCESS;
}

// Bytes for a copy of an operand whose rows do not start on multiples of 16 bytes.
bool BytesAligned(const aclsparseDnMatDescr *m) { return Aligned16(m->values) && m->ld % 16 == 0; }
size_t CopyBytes(const aclsparseDnMatDescr *m)
{
    return BytesAligned(m) ? 0 : AlignUp((size_t)m->rows * AlignUp((size_t)m->cols, 16), 256);
}

struct Operand {
    const void *values;
    long long ld;
    cudaError_t error;
};
// An operand as the kernels read it: where it lies, or its copy at `room`, which moves on.
Operand Aligned(const aclsparseDnMatDescr *m, char **room, cudaStream_t stream, const ScaledArgs &a, int rowsEach)
{
    const size_t bytes = CopyBytes(m);
    if (bytes == 0) return {m->values, m->ld, cudaSuccess};
    char *const to = *room;
    *room += bytes;
    const long long pieces = m->rows * ((m->cols + 15) / 16);
    const unsigned blocks = (unsigned)std::min<long long>((pieces + 255) / 256, (long long)b200sp_sm_count() * 32);
    b200sp_note_launches(1);
    const cudaError_t e = b200sp::LaunchChained(ScaledAlignKernel, blocks, 256, 0, stream, static_cast<const uint8_t *>(m->values), m->rows,
                                                (int)m->cols, m->ld, reinterpret_cast<uint4 *>(to), a.header, a.mark, a.number, a.offsets, rowsEach);
    return {to, (long long)AlignUp((size_t)m->cols, 16), e};
}

// Rows of X of a tile: of as many as the matrix (or an expert, on average, and half as much again for the uneven ones) has.
int TileColumns(long long rows, long long experts)
{
    const long long want = experts > 1 ? (rows * 3 + 2 * experts - 1) / (2 * experts) : rows;
    int cols = 16;
    while (cols < kTileColsMost && cols < want) cols *= 2;
    return cols;
}

// How a product without experts is computed: by tiles, of a CTA, a pair of them, or a cluster that shares a tile's steps, or without tiles.  An estimate of the
// time of every way, us, fitted to 620 timings of 48 products, 1 to 2048 rows by six matrices of 128 KB to 17 MB, in the ways and widths of tiles that each allows.  On
// 70 other products (1 to 2048 rows, 128 to 8192 channels, 256 to 8192 columns) it takes one 1.7 % slower than the fastest on average; eight lose 5 % or more, one
// 21 %: 16 rows of 672 by 2392, without tiles 7.4, by tiles of 32 6.1.  (512 rows of 4096 by 4096: pairs 17, clusters of two 37; 16 rows: clusters of four 10, whole
// tiles 15; one row: clusters 10, without tiles 6.6; four rows 10 and 12.6; 8 rows of 1024 by 1024: 6.4 and 3.7.)
enum FormKind { kWhole, kPairs, kShared, kFew };
struct Form {
    FormKind kind;
    int cols, split;
};
Form FormOf(long long rows, long long n, long long depth)
{
    const double steps = (double)((depth + kTileDepth - 1) / kTileDepth);
    const int sms = b200sp_sm_count();
    Form best{kWhole, 16, 1};
    const double bytes = (double)n * (double)depth;
    // W from DRAM, and the products of four bytes
    const bool few = rows <= 16 && n < 1 << 26;  // its items are counted in 31 bits
    double least = few ? 2.6 + bytes * (1.4e-7 + 1.2e-7 * (double)rows) : 1e300;
    if (few) best.kind = kFew;
    const auto offer = [&](double us, FormKind kind, int cols, int split) {
        us += 1e-7 * bytes;
        if (us < least) least = us, best = {kind, cols, split};
    };
    for (int cols = 16; cols <= kTileColsMost; cols *= 2) {
        const long long across = (rows + cols - 1) / cols, tiles = (n + kTileRows - 1) / kTileRows * across;
        const auto wide = [&](int unit) { return (double)(((rows + across - 1) / across + unit - 1) / unit * unit); };
        const auto whole = [&](double start, double step, double perRow, double store, double waves, double columns) {
            return start + waves * std::max(steps * (step + perRow * columns), store + 0.0078 * columns) + 0.0078 * columns;
        };
        offer(whole(4.3, 0.309, 0.0004, 1.47, (double)((tiles + sms - 1) / sms), wide(16)), kWhole, cols, 1);
        const long long pairs = (n + 2 * kTileRows - 1) / (2 * kTileRows) * across;
        if (cols >= 64 && n > kTileRows)
            offer(whole(4.7, 0.319, 0.0003, 1.35, (double)((pairs + sms / 2 - 1) / (sms / 2)), wide(32)), kPairs, cols, 1);
        for (int split = 2; split <= kSplitMost && split <= steps; split *= 2) {
            // one CTA an SM, and clusters that the SMs' groups hold side by side
            if (tiles * split > (split == 2 ? sms : split == 4 ? 136 : 112)) break;
            const double columns = (double)std::min<long long>(cols, (rows + 15) / 16 * 16);
            offer(4.46 + std::ceil(steps / split) * (0.309 + 0.0004 * columns) + (0.0074 + 0.1685 / split) * columns, kShared, cols, split);
        }
    }
    return best;
}

// With experts, of whose rows the host knows the average only.  us for 32 experts of 2048 x 2048, four a token, by CTAs on 32 and 64 rows, by pairs on 128 and 256: 64
// tokens 29, 29, 30, 31; 256 tokens 37, 30, 31, 32; 1024 tokens 96, 58, 43, 35; 4096 tokens 332, 180, 105, 73.  Single CTAs on as many rows as the pairs: 1024 tokens
// 44 and 37, 4096 107 and 77.  Without tiles, and by tiles of 16: 64 experts of 2048 x 2048, eight a token, one token 8.4 and 10.5, two 15.7 and 16.8, four 27.3
// and 23.9.  (The border is right for such; it goes by entries alone: of few experts more would be faster without tiles -- two tokens to two of eight of 4096 x 4096
// 8.6, and 14.7 as it is -- and of many fewer: eight tokens to eight of 256 of 2048 x 2048 42 by tiles, and 55 as it is.)
Form FormOfExperts(long long rows, long long n, long long experts)
{
    Form form{kWhole, TileColumns(rows, experts), 1};
    if (form.cols >= 128 && n > kTileRows) form.kind = kPairs;
    // hardly an expert has more than one
    if (4 * rows <= experts) form.kind = kFew;
    return form;
}

aclsparseStatus_t Product(const char *call, const aclsparseContext *handle, ScaledArgs a, const aclsparseDnMatDescr *X,
                          const aclsparseDnVecDescr *scalesX, const aclsparseDnMatDescr *W, const aclsparseDnVecDescr *scalesW,
                          const aclsparseDnMatDescr *Y, char *room)
{
    a.rows = (int)X->rows;
    a.n = (int)Y->cols;
    a.steps = (int)((X->cols + kTileDepth - 1) / kTileDepth);
    a.scalesX = static_cast<const float *>(scalesX->values);
    a.scalesW = static_cast<const float *>(scalesW->values);
    a.y = Y->values;
    a.ldy = Y->ld;
    a.vectors = RowsAligned(Y);
    const Operand x = Aligned(X, &room, handle->stream, a, 0);
    const Operand w = Aligned(W, &room, handle->stream, a, a.header != nullptr ? a.n : 0);
    if (x.error != cudaSuccess || w.error != cudaSuccess) return Finished(x.error != cudaSuccess ? x.error : w.error, call);
    const Form form = a.header == nullptr ? FormOf(a.rows, a.n, X->cols) : FormOfExperts(a.rows, a.n, a.experts);
    if (form.kind == kFew) {
        const long long chunks = a.header == nullptr ? (a.rows + kFewRowsX - 1) / kFewRowsX : a.rows;
        const cudaError_t e = WithType(Y->valueType, [&](auto out) {
            return LaunchFew<decltype(out)>(a, x.values, x.ld, w.values, w.ld, (int)X->cols, chunks, handle->stream);
        });
        return Finished(e, call);
    }
    a.colsMost = form.cols;
    a.split = form.split;
    a.box = form.kind == kPairs ? a.colsMost / 2 : a.colsMost;
    CUtensorMap mapW, mapX;
    if (!MapOfBytes(&mapW, w.values, W->cols, W->rows, w.ld, kTileRows) || !MapOfBytes(&mapX, x.values, X->cols, X->rows, x.ld, a.box))
        return ACL_SPARSE_STATUS_INTERNAL_ERROR;
    const cudaError_t e = WithType(Y->valueType, [&](auto out) {
        using Out = decltype(out);
        if (form.kind == kShared) return LaunchSplit<Out>(a, mapW, mapX, handle->stream);
        return form.kind == kPairs ? LaunchScaled<Out, true>(a, mapW, mapX, handle->stream) : LaunchScaled<Out, false>(a, mapW, mapX, handle->stream);
    });
    return Finished(e, call);
}

size_t BufferBytes(const aclsparseSpMatDescr *R, const aclsparseDnMatDescr *X, const aclsparseDnMatDescr *W)
{
    return (R != nullptr ? PlanLayoutFor(R->nnz, R->cols).total : 0) + CopyBytes(X) + CopyBytes(W);
}

aclsparseStatus_t CheckExperts(const aclsparseSpMatDescr *R, const aclsparseDnMatDescr *X, const aclsparseDnMatDescr *W,
                               const aclsparseDnMatDescr *Y)
{
    const aclsparseStatus_t st = CheckRouted(R);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    const aclsparseStatus_t s = CheckOperands(X, W, Y, R->cols);
    if (s != ACL_SPARSE_STATUS_SUCCESS) return s;
    return X->rows == R->nnz ? ACL_SPARSE_STATUS_SUCCESS : ACL_SPARSE_STATUS_INVALID_VALUE;
}

}  // namespace

extern "C" {

int b200sp_scaled_error(void)
{
    int flag = 0;
    if (cudaDeviceSynchronize() != cudaSuccess) return -1;
    return cudaMemcpyFromSymbol(&flag, gScaledError, sizeof(flag)) == cudaSuccess ? flag : -1;
}

int b200sp_scaled_error_clear(void)
{
    const int zero = 0;
    const cudaError_t e = cudaDeviceSynchronize();
    if (e != cudaSuccess) return (int)e;
    return (int)cudaMemcpyToSymbol(gScaledError, &zero, sizeof(zero));
}

void b200sp_scaled_wait_test(long long wait_cycles, unsigned extra_tx)
{
    gScaledWaitCycles = wait_cycles > 0 ? wait_cycles : kTileWaitCycles;
    gScaledExtraTx = extra_tx;
}

aclsparseStatus_t b200spScaledMMBufferSize(aclsparseHandle_t handle, aclsparseConstDnMatDescr_t matX, aclsparseConstDnMatDescr_t matW,
                                           aclsparseConstDnMatDescr_t matY, size_t *bufferSize)
{
    if (handle == nullptr) return ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR;
    if (bufferSize == nullptr) return ACL_SPARSE_STATUS_INVALID_VALUE;
    const aclsparseStatus_t st = CheckOperands(matX, matW, matY, 1);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    const size_t bytes = BufferBytes(nullptr, matX, matW);
    *bufferSize = bytes + (bytes > 0 ? 256 : 0);  // any address is accepted
    return ACL_SPARSE_STATUS_SUCCESS;
}

aclsparseStatus_t b200spScaledMM(aclsparseHandle_t handle, const void *alpha, aclsparseConstDnMatDescr_t matX,
                                 aclsparseConstDnVecDescr_t scalesX, aclsparseConstDnMatDescr_t matW, aclsparseConstDnVecDescr_t scalesW,
                                 const void *beta, aclsparseDnMatDescr_t matY, void *buffer)
{
    if (handle == nullptr) return ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR;
    aclsparseStatus_t st = CheckOperands(matX, matW, matY, 1);
    if (st == ACL_SPARSE_STATUS_SUCCESS) st = CheckScales(scalesX, matX->rows);
    if (st == ACL_SPARSE_STATUS_SUCCESS) st = CheckScales(scalesW, matW->rows);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    const bool copies = BufferBytes(nullptr, matX, matW) > 0;
    if (copies && buffer == nullptr) return ACL_SPARSE_STATUS_INSUFFICIENT_RESOURCES;
    const OnDevice device(handle);
    if (copies && NoteWrite(buffer) == 0) return ACL_SPARSE_STATUS_ALLOC_FAILED;
    ScaledArgs a{};
    a.experts = 1;
    a.sc = ScalarsOf(handle, alpha, beta);
    return Product("b200spScaledMM", handle, a, matX, scalesX, matW, scalesW, matY, copies ? BufferStart(buffer) : nullptr);
}

aclsparseStatus_t b200spExpertsScaledMMBufferSize(aclsparseHandle_t handle, aclsparseConstSpMatDescr_t matR, aclsparseConstDnMatDescr_t matX,
                                                  aclsparseConstDnMatDescr_t matW, aclsparseConstDnMatDescr_t matY, size_t *bufferSize)
{
    if (handle == nullptr) return ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR;
    if (bufferSize == nullptr) return ACL_SPARSE_STATUS_INVALID_VALUE;
    const aclsparseStatus_t st = CheckExperts(matR, matX, matW, matY);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    *bufferSize = NoteSize(matR, BufferBytes(matR, matX, matW));
    return ACL_SPARSE_STATUS_SUCCESS;
}

aclsparseStatus_t b200spExpertsScaledMM(aclsparseHandle_t handle, const void *alpha, aclsparseConstSpMatDescr_t matR,
                                        aclsparseConstDnMatDescr_t matX, aclsparseConstDnVecDescr_t scalesX, aclsparseConstDnMatDescr_t matW,
                                        aclsparseConstDnVecDescr_t scalesW, const void *beta, aclsparseDnMatDescr_t matY, void *buffer)
{
    if (handle == nullptr) return ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR;
    aclsparseStatus_t st = CheckExperts(matR, matX, matW, matY);
    if (st == ACL_SPARSE_STATUS_SUCCESS) st = CheckScales(scalesX, matX->rows);
    if (st == ACL_SPARSE_STATUS_SUCCESS) st = CheckScales(scalesW, matW->rows);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (buffer == nullptr) return ACL_SPARSE_STATUS_INSUFFICIENT_RESOURCES;
    uint64_t number;
    if (!HoldsOrder(matR, buffer, handle->stream, &number) || !HasRoomFor(matR, CopyBytes(matX) + CopyBytes(matW)))
        return ACL_SPARSE_STATUS_INVALID_VALUE;
    const OnDevice device(handle);
    const PlanLayout L = PlanLayoutFor(matR->nnz, matR->cols);
    char *const p = BufferStart(buffer);
    ScaledArgs a{};
    a.header = reinterpret_cast<const int4 *>(p);
    a.mark = HeaderOf(matR->nnz, matR->cols, matR->rows);
    a.number = number;
    a.offsets = reinterpret_cast<const int *>(p + L.offsets);
    a.experts = (int)matR->cols;
    a.sc = ScalarsOf(handle, alpha, beta);
    return Product("b200spExpertsScaledMM", handle, a, matX, scalesX, matW, scalesW, matY, p + L.total - 256);
}

aclsparseStatus_t b200spScaledMMInfo(aclsparseConstSpMatDescr_t matR, aclsparseConstDnMatDescr_t matX, aclsparseConstDnMatDescr_t matW,
                                     aclsparseConstDnMatDescr_t matY, int32_t info[3])
{
    if (info == nullptr) return ACL_SPARSE_STATUS_INVALID_VALUE;
    const aclsparseStatus_t st = matR == nullptr ? CheckOperands(matX, matW, matY, 1) : CheckExperts(matR, matX, matW, matY);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    const Form form = matR == nullptr ? FormOf(matX->rows, matY->cols, matX->cols) : FormOfExperts(matX->rows, matY->cols, matR->cols);
    info[0] = form.kind;
    info[1] = form.kind == kFew ? 0 : form.cols;
    info[2] = form.kind == kShared ? form.split : 1;
    return ACL_SPARSE_STATUS_SUCCESS;
}

}  // extern "C"
