// The order of a routing's entries by expert: what a buffer holds of it, and what the calls that follow it check.
#pragma once

#include <algorithm>
#include <mutex>

#include "tokens/common.cuh"

namespace b200sp_tokens {

constexpr int kMaxExperts = 1024;

// The buffer: what R it is the order of; where every expert's entries begin (one more group: entries of no expert), the entries by
// expert, the rows of R that they lie in, and every entry's place among them; and the sort's own arrays.
struct PlanLayout {
    size_t offsets, entries, rows, places, keyA, keyB, posB, total;
};
inline PlanLayout PlanLayoutFor(long long nnz, long long experts)
{
    PlanLayout L;
    const size_t words = AlignUp(sizeof(int) * (size_t)nnz, 256);
    L.offsets = 256;  // the header lies before
    L.entries = L.offsets + AlignUp(sizeof(int) * (size_t)(experts + 2), 256);
    L.rows = L.entries + words;
    L.places = L.rows + words;
    L.keyA = L.places + words;
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

// Whether a buffer starts with what a call expects; number 0: any.
__device__ __forceinline__ bool StartsWith(const int4 *header, const int4 &mark, uint64_t number)
{
    const int4 found = __ldg(header);
    return found.x == mark.x && found.y == mark.y && found.z == mark.z && found.w == mark.w &&
           (number == 0 || __ldg(reinterpret_cast<const unsigned long long *>(header + 1)) == number);
}

// ---------------------------------------------------------------- host

inline aclsparseStatus_t CheckRouted(const aclsparseSpMatDescr *R)
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

inline char *BufferStart(const void *buffer) { return reinterpret_cast<char *>(AlignUp(reinterpret_cast<uintptr_t>(buffer), 256)); }

// Whether the buffer is the one that R's entries were ordered in last, and no other call has written it since.
inline bool SameBuffer(const aclsparseSpMatDescr *R, const void *buffer)
{
    const b200sp::ExpertsPlan &p = R->experts;
    return buffer != nullptr && p.buffer == buffer && p.offsets == R->offsets && p.indices == R->indices && p.rows == R->rows &&
           p.cols == R->cols && p.nnz == R->nnz && p.generation != 0 && p.generation == b200sp::BufferGeneration(buffer);
}
// Whether the buffer still holds the order of R's entries; the number that it has to have, 0: any.
inline bool HoldsOrder(const aclsparseSpMatDescr *R, const void *buffer, cudaStream_t stream, uint64_t *number)
{
    std::lock_guard<std::mutex> lock(R->expertsMutex);
    *number = R->experts.captured && !Captures(stream) ? R->experts.number : 0;
    return SameBuffer(R, buffer) && !R->experts.stale;
}

// What the BufferSize calls for this matrix have said at most.
inline size_t NoteSize(const aclsparseSpMatDescr *R, size_t bytes)
{
    std::lock_guard<std::mutex> lock(R->expertsMutex);
    R->expertsSized = std::max(R->expertsSized, (int64_t)bytes);
    return bytes;
}
// Whether the buffer may be taken to have room for copies of so many bytes behind the order, if any: what Preprocess writes it has.
inline bool HasRoomFor(const aclsparseSpMatDescr *R, size_t copies)
{
    if (copies == 0) return true;
    std::lock_guard<std::mutex> lock(R->expertsMutex);
    return (int64_t)(PlanLayoutFor(R->nnz, R->cols).total + copies) <= R->expertsSized;
}

}  // namespace b200sp_tokens
